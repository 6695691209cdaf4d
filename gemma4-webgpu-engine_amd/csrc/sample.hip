// Sampling with temperature, top-k, top-p and min-p from given random numbers (include/g4serve.h).
//
// All filters keep a prefix of the row ordered by (logit down, id up), so a row's kept set is one cut in that
// order, and min-p a bound on the logit beside it. The order is never made: (1) the maximum of every unit of 1024 tokens
// and part of the row; (2) weights, and for a row with top-k or top-p a histogram of them over bins of the capped
// logit; (3) the bins where the cuts lie, from the histogram, the units' weights above them, and a list of what lies in
// them, for which only units that reach up to them are read again; (4) a block per row finds the cuts within its list,
// the unit and then the token where the running sum passes u of the total. A row without top-k and top-p has its
// units' weights from (2).
//
// Weights are integers, steps of 2^-shift of the row's largest: sums are exact, and additions in any order, atomic ones
// too, give the same. A bin never falls as a logit falls, so that bins and logits have one order.
#include "g4_logits.h"
#include "../../include/g4serve.h"
#include <cmath>

namespace g4 {

typedef unsigned long long u64;

constexpr int kSampleThreads = 256, kSampleWaves = kSampleThreads / 64;
constexpr int kSampleUnit = 1024, kSamplePer = kSampleUnit / 64;  // a wave's range, and a lane's part of it
constexpr int kSamplePart = kSampleWaves * kSampleUnit;
constexpr int kBins = 1024, kBinsPer = kBins / 64;
constexpr int kList = 4096;  // entries; a row with more is read again
constexpr int kFew = 64;     // entries that a wave orders by itself
constexpr int kSub = 1024, kSubPer = kSub / kSampleThreads;  // ranges of one refinement step
constexpr int kUnitPer = kSampleUnit / kSampleThreads;
constexpr int kLineWords = 32;
constexpr int kWideRow = 128;  // units
constexpr int kMaxVocab = 1 << 22;

struct PartMax {
    float max, min;  // of the logits above -infinity
    int index;       // of the first maximum (-1: no logit)
    int pad;
};

// Where a filtered row's cuts lie (bins from the top; kBins: nowhere).
struct Cuts {
    int k_bin, p_low, p_high, k_rest;  // the k-th token is the k_rest-th of k_bin
    u64 k_before, p_before;            // weight of the bins above k_bin and above p_low
    float least, pad;                  // no logit below this is in one of these bins, or above
};

// What a row's weights are made with.
struct Row {
    double top, slope, d_min, bins;  // weight 2^((y - top) slope), kept from d_min on, bin (top - y) bins
    double d_low;                    // here a weight is 2^-1000 of the largest, none
    double inv_t, p;
    int index, k;                // the first maximum (-1: no logit)
    int greedy, filtered, inf, pad;  // inf: the maximum is +infinity, whose like share all weight
};

// (half_cap: a little less than half the cap)
struct CapArgs {
    double cap, inv_cap, inv_cap2;
    float half_cap;
};

struct SampleArgs {
    const float *logits;
    int64_t stride;
    const int32_t *row_index;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    CapArgs cap;
    int logit_rows, vocab, parts, units, shift, vec, cuts;  // cuts: top-k or top-p given
    int wide, share, spans, many;  // waves of a block of (2) and (3), those of a unit, blocks a row, whether there are many
    PartMax *stats;              // [rows][parts]
    Row *row;                    // [rows]
    Cuts *cut;                   // [rows]
    u64 *span_sums, *unit_sums;  // [rows][spans], [rows][units]
    u64 *bin_mass;               // [rows][kBins]
    u64 *list;                   // [rows][kList]
    uint32_t *bin_count;         // [rows][kBins]
    uint32_t *listed;            // [rows], kLineWords apart: rows' counters on lines of their own
    float *unit_max;             // [rows][units]
    int32_t *tokens;
    float *logprobs;
};

// The logits of request `row`, null where it names none.
__device__ __forceinline__ const float *row_of(const SampleArgs &A, int row) {
    const int r = A.row_index ? A.row_index[row] : row;
    return (unsigned)r < (unsigned)A.logit_rows ? A.logits + r * A.stride : nullptr;
}

// The place in its unit of a lane's value j: groups of 4 where rows are read 16 bytes at a time.
__device__ __forceinline__ int unit_place(int j, int lane, int vec) {
    return vec ? (j / 4) * 256 + 4 * lane + j % 4 : j * 64 + lane;
}

// The lane's values of the wave's unit, or quarter of one, at x, `n` of which exist; a NaN is one.
template <int PER>
__device__ __forceinline__ void load_unit(const float *x, int n, int lane, int vec, float (&v)[PER]) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            const int i = unit_place(j, lane, 1);
            if (i + 4 <= n) {
                const float4 y = *reinterpret_cast<const float4 *>(x + i);
                v[j] = y.x;
                v[j + 1] = y.y;
                v[j + 2] = y.z;
                v[j + 3] = y.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j + e] = i + e < n ? x[i + e] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = unit_place(j, lane, 0);
            v[j] = i < n ? x[i] : -INFINITY;
        }
    }
}

__device__ __forceinline__ void join_max(PartMax &a, float max, float min, int index) {
    if (max > a.max || (max == a.max && (unsigned)index < (unsigned)a.index)) {
        a.max = max;
        a.index = index;
    }
    a.min = fminf(a.min, min);
}
__device__ __forceinline__ PartMax wave_join(PartMax m) {
#pragma unroll
    for (int s = 32; s; s >>= 1) join_max(m, __shfl_xor(m.max, s), __shfl_xor(m.min, s), __shfl_xor(m.index, s));
    return m;
}

// Grid (parts, rows). Also clears the row's histogram and list for the kernels behind. Bound by reads: 256 rows of 262144 in
// 40 us, 6.7 TB/s; one row 4.1.
__global__ __launch_bounds__(kSampleThreads) void sample_max_kernel(SampleArgs A) {
    __shared__ PartMax ms[kSampleWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, part = blockIdx.x, row = blockIdx.y;
    const float *x = row_of(A, row);
    const int base = part * kSamplePart + wave * kSampleUnit;
    PartMax m{-INFINITY, INFINITY, -1, 0};
    if (x && base < A.vocab) {
        float v[kSamplePer];
        load_unit(x + base, A.vocab - base, lane, A.vec, v);
#pragma unroll
        for (int j = 0; j < kSamplePer; ++j) {
            v[j] = clean(v[j]);
            m.max = fmaxf(m.max, v[j]);
            m.min = fminf(m.min, v[j] > -INFINITY ? v[j] : INFINITY);
        }
        if (m.max > -INFINITY) {
#pragma unroll
            for (int j = kSamplePer - 1; j >= 0; --j) m.index = v[j] == m.max ? base + unit_place(j, lane, A.vec) : m.index;
        }
    }
    m = wave_join(m);
    if (lane == 0) ms[wave] = m;
    if (A.cuts) {
        if (lane == 0 && base < A.vocab) A.unit_max[(int64_t)row * A.units + part * kSampleWaves + wave] = m.max;
        for (int i = part * kSampleThreads + t; i < kBins; i += A.parts * kSampleThreads) {
            A.bin_mass[(int64_t)row * kBins + i] = 0;
            A.bin_count[(int64_t)row * kBins + i] = 0;
        }
        if (part == 0 && t == 0) A.listed[(int64_t)row * kLineWords] = 0;
    }
    __syncthreads();
    if (t) return;
#pragma unroll
    for (int w = 1; w < kSampleWaves; ++w) join_max(m, ms[w].max, ms[w].min, ms[w].index);
    A.stats[(int64_t)row * A.parts + part] = m;
}

// The softcap past half the cap, cap - 2 cap / (e^(2 |x| / cap) + 1), 1e-14 of the cap off, where the library's exponential
// would hold twenty registers through the loops around it: 2^z as n + f, |f| <= 1/2, by the series to f^11.
__device__ __forceinline__ double far_logit(float x, const CapArgs &A) {
    const double z = fmin(fabs((double)x) * A.inv_cap * (2 * 1.4426950408889634074), 1000.0);
    const double r = z + 0x1.8p52, f = z - (r - 0x1.8p52);
    double e = 4.44553827187081e-10;
    e = fma_k(e, f, 7.054911620801121e-09);
    e = fma_k(e, f, 1.0178086009239696e-07);
    e = fma_k(e, f, 1.3215486790144305e-06);
    e = fma_k(e, f, 1.5252733804059838e-05);
    e = fma_k(e, f, 0.00015403530393381606);
    e = fma_k(e, f, 0.0013333558146428441);
    e = fma_k(e, f, 0.009618129107628477);
    e = fma_k(e, f, 0.055504108664821576);
    e = fma_k(e, f, 0.2402265069591007);
    e = fma_k(e, f, 0.6931471805599453);
    e = fma_k(e, f, 1.0);
    e = __hiloint2double(__double2hiint(e) + (int)((uint32_t)__double2loint(r) << 20), __double2loint(e)) + 1.0;
    double q = __builtin_amdgcn_rcp(e);
    q *= __builtin_fma(-e, q, 2.0);
    q *= __builtin_fma(-e, q, 2.0);
    return copysign(__builtin_fma(-2.0 * A.cap, q, A.cap), (double)x);
}
__device__ __forceinline__ double capped(float x, const CapArgs &A) {
    if (A.cap == 0.0) return x;
    return fabsf(x) > A.half_cap ? far_logit(x, A) : near_cap((double)x, A);
}

// By one wave, the same in every lane.
__device__ __forceinline__ Row row_params(const SampleArgs &A, int row) {
    const int lane = threadIdx.x & 63;
    PartMax m{-INFINITY, INFINITY, -1, 0};
    for (int c = lane; c < A.parts; c += 64) {
        const PartMax s = A.stats[(int64_t)row * A.parts + c];
        join_max(m, s.max, s.min, s.index);
    }
    const float tf = A.temperature ? A.temperature[row] : 1.0f, pf = A.top_p ? A.top_p[row] : 1.0f;
    const float mf = A.min_p ? A.min_p[row] : 0.0f;
    const int k = A.top_k ? A.top_k[row] : 0;
    m = wave_join(m);
    Row R;
    R.index = m.index;
    R.greedy = !(tf > 0.0f);
    const double t = R.greedy ? 1.0 : fmin((double)tf, 0x1p200);  // (past all differences; -infinity / infinity would be NaN)
    R.inv_t = 1.0 / t;
    R.slope = R.inv_t * 1.4426950408889634074;
    R.inf = A.cap.cap == 0.0 && m.max == INFINITY;
    R.top = R.inf || m.index < 0 ? 0.0 : capped(m.max, A.cap);
    R.d_min = -INFINITY;
    if (mf > 0.0f && tf < INFINITY) R.d_min = mf >= 1.0f ? 0.0 : log((double)mf) * t;  // (an infinite one makes all alike)
    R.k = k < A.vocab ? k : 0;
    R.p = pf < 1.0f ? (double)pf : 1.0;  // NaN: off
    R.filtered = !R.greedy && m.index >= 0 && (R.k > 0 || R.p < 1.0);
    R.d_low = -693.0 * t;
    R.bins = 0.0;
    if (R.filtered && !R.inf) {
        // the bins reach from the top to the lowest logit, or to where weights round to no step
        const double range = fmin(R.top - capped(m.min, A.cap), (A.shift + 1) * 0.69314718055994530942 * t);
        if (range > 0.0) R.bins = fmin((kBins - 1) * __builtin_amdgcn_rcp(range), 1e300);
    }
    R.pad = 0;
    return R;
}

// The same value in scalar registers: it is the block's.
template <class T>
__device__ __forceinline__ T uniform(const T &v) {
    static_assert(sizeof(T) % 4 == 0, "words");
    struct Words {
        int w[sizeof(T) / 4];
    };
    Words a = __builtin_bit_cast(Words, v);
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 4; ++i) a.w[i] = __builtin_amdgcn_readfirstlane(a.w[i]);
    return __builtin_bit_cast(T, a);
}

// The same of what an earlier kernel left in memory, by scalar loads.
template <class T>
__device__ __forceinline__ T uniform_at(const T *p) {
    struct Words {
        int w[sizeof(T) / 4];
    };
    const auto *from = (const __attribute__((address_space(4))) int *)(uintptr_t)p;
    Words a;
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 4; ++i) a.w[i] = from[i];
    return __builtin_bit_cast(T, a);
}

// Under an infinite maximum a logit is as good as it, or nothing.
__device__ __forceinline__ float seen(float x, const Row &R) { return R.inf ? (x == INFINITY ? 0.0f : -INFINITY) : x; }

// The polynomials' first coefficients.
constexpr double kPowFirst = 1.3259689002093833e-06;
struct Firsts {
    double cap = kNearCapFirst, pow = kPowFirst;
};
// The same kept in vector registers: a step has a place for one scalar operand, and they would be made for each logit.
__device__ __forceinline__ Firsts firsts() {
    Firsts F;
    asm("" : "+v"(F.cap), "+v"(F.pow));
    return F;
}

// y - top of a logit that is not past half the cap; for a NaN and a -infinity one of these two (no weight).
template <bool CAP>
__device__ __forceinline__ double near_distance(float x, const Row &R, const SampleArgs &A, Firsts F = {}) {
    return (CAP ? near_cap((double)x, A.cap, F.cap) : (double)x) - R.top;
}
// And of any.
template <bool CAP>
__device__ __forceinline__ double distance(float x, const Row &R, const SampleArgs &A) {
    double y = x;
    if (CAP) {
        y = near_cap(y, A.cap);
        if (is_far(x, A.cap)) y = far_logit(x, A.cap);
    }
    return y - R.top;
}
// The weight in steps (at most 2^51 and a little), rounded, above kNoSteps; its bits above kNoStepsBits are the integer.
constexpr double kNoSteps = 0x1p52;
constexpr u64 kNoStepsBits = 0x4330000000000000ull;
// 2^(d slope + shift) as pow2 of g4_logits.h makes it, with fewer steps: the integer part comes from one fused product, and d
// is bounded where that is (a NaN too).
__device__ __forceinline__ double raised_steps(double d, const Row &R, const SampleArgs &A, Firsts F = {}) {
    d = fmax(d, R.d_low);
    const double magic = 0x1.8p52 + A.shift, r = __builtin_fma(d, R.slope, magic);  // n + shift in the low word
    const double f = __builtin_fma(d, R.slope, -(r - magic));
    double e = F.pow;
    e = fma_k(e, f, 1.531008106933654e-05);
    e = fma_k(e, f, 0.00015403433582607232);
    e = fma_k(e, f, 0.0013333450560096254);
    e = fma_k(e, f, 0.009618129194093111);
    e = fma_k(e, f, 0.05550410941217064);
    e = fma_k(e, f, 0.24022650695640319);
    e = fma_k(e, f, 0.6931471805459295);
    e = fma_k(e, f, 1.0000000000000135);
    return __hiloint2double(__double2hiint(e) + (int)((uint32_t)__double2loint(r) << 20), __double2loint(e)) + kNoSteps;
}
__device__ __forceinline__ u64 steps(double d, const Row &R, const SampleArgs &A, Firsts F = {}) {
    return (u64)__double_as_longlong(raised_steps(d, R, A, F)) - kNoStepsBits;
}
// (The conversion takes what is below 0, a rounding, and a NaN to 0, and what is too large to the largest.) A weight above
// no step is more than half of one, its d above -(shift + 1) ln 2 t, and no d is below the lowest logit's: the number is
// below kBins, whose share of the range is a bin more than bins counts on.
__device__ __forceinline__ uint32_t bin_number(double d, const Row &R) {
    uint32_t b;
    asm("v_cvt_u32_f64 %0, %1" : "=v"(b) : "v"(-d * R.bins));
    return b;
}
__device__ __forceinline__ int bin_of(double d, const Row &R) { return (int)min(bin_number(d, R), (uint32_t)kBins - 1); }

// Order of tokens: logit down, then id up, as a number (0: none).
__device__ __forceinline__ u64 order_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
    const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (u64)up << 32 | (uint32_t)~id;
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

// Inclusive sum over the block's threads; *total: of all.
__device__ __forceinline__ u64 block_run(u64 v, u64 *lds, u64 *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const u64 o = __shfl_up(v, s);
        if (lane >= s) v += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
        const u64 s = lds[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return before + v;
}

// The bin that stands at place i of a row's histogram in memory: a lane's 16 consecutive bins lie 64 apart, so that a
// wave's loads of them are of whole lines. (Loads of 128 bytes a lane stalled on each other's lines: 12 us.)
__device__ __forceinline__ int bin_at(int i) { return i % 64 * kBinsPer + i / 64; }

// The sums of units that waves of a block share.
template <int WAVES, int SHARE>
__device__ __forceinline__ void put_unit_sums(const SampleArgs &A, int row, const u64 *sums) {
    const int t = threadIdx.x, unit = blockIdx.x * (WAVES / SHARE) + t;
    if (t >= WAVES / SHARE || unit >= A.units) return;
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < SHARE; ++w) all += sums[t * SHARE + w];
    A.unit_sums[(int64_t)row * A.units + unit] = all;
}

// Four rows a block, a wave each: for calls of many blocks, each of which would do it again (5.4 us).
__global__ __launch_bounds__(kSampleThreads) void sample_row_kernel(SampleArgs A, int rows) {
    const int row = blockIdx.x * kSampleWaves + (threadIdx.x >> 6);
    if (row >= rows) return;
    const Row R = row_params(A, row);
    if ((threadIdx.x & 63) == 0) A.row[row] = R;
}

// Grid (spans, rows). Bound by issue: with a cap 41 vector operations a logit, 27 of them 64-bit, which keep the vector
// units busy for 75% of 105 us (256 rows of 262144); the atomics keep LDS busy for half of it. One row: 7.2 us, a chain.
// With a cap and a wave a unit three of the 64 registers that eight waves a SIMD have are kept in memory over the values of a
// row without cuts: a store and a load a wave, none a logit, and none in rows with cuts.
// SHARE: waves that share a unit, a quarter each.
// READY: the rows' parameters are there (sample_row_kernel).
template <bool CAP, int WAVES, int SHARE, bool READY>
__global__ __launch_bounds__(64 * WAVES, 8) void sample_weights_kernel(SampleArgs A) {
    __shared__ u64 mass[kBins];        // (16 bytes a bin with its count: a wave's atomics in more conflicts, 4 us of 105)
    __shared__ uint32_t count[kBins];  // where there is a top-k
    __shared__ u64 ss[WAVES], ks[WAVES];
    constexpr int kPer = kSamplePer / SHARE;
    __shared__ Row shared_row;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.y;
    const float *x = row_of(A, row);
    const int place = blockIdx.x * WAVES + wave, unit = place / SHARE, base = place * (kSampleUnit / SHARE);
    float v[kPer];
    load_unit(x + base, x ? A.vocab - base : 0, lane, A.vec, v);
    if (!READY && wave == 0) {  // once a block: as many operations as the weights of a unit
        const Row R = row_params(A, row);
        if (lane == 0) {
            shared_row = R;
            if (blockIdx.x == 0) A.row[row] = R;
        }
    }
    if (A.cuts)
        for (int i = t; i < kBins; i += 64 * WAVES) mass[i] = 0, count[i] = 0;
    __syncthreads();
    const Row R = READY ? uniform_at(A.row + row) : uniform(shared_row);
    if (R.index < 0) return;
    const Firsts F = firsts();
    auto each = [&](auto add) {
        float most = 0.0f;
        if (CAP) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) most = fmaxf(most, fabsf(v[j]));
        }
        uint32_t far = 0;  // places where a lane's logit is past half the cap: few, one at a time
        if (CAP && __any(most > A.cap.half_cap)) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const bool f = is_far(v[j], A.cap);
                far |= __ballot(f) ? 1u << j : 0u;
                v[j] = f ? -INFINITY : v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            float xs = v[j];
            asm("" : "+v"(xs));  // one after the other: all at once they would not fit the registers
            add(near_distance<CAP>(xs, R, A, F));
        }
        for (; far; far &= far - 1) {
            const int i = base + unit_place(__ffs(far) - 1, lane, A.vec);
            const float xs = i < A.vocab ? x[i] : -INFINITY;
            if (is_far(xs, A.cap)) add(distance<CAP>(xs, R, A));
        }
    };
    if (R.inf) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = seen(v[j], R);
    }
    u64 all = 0;
    if (R.filtered) {
        uint32_t one = 1;
        asm("" : "+v"(one));  // kept, and not made again for each logit
        each([&](double d) {
            const double w = raised_steps(d, R, A, F);
            if (w > kNoSteps) {  // a weight of no step would be past the last bin, no other is
                const uint32_t b = bin_number(d, R);
                atomicAdd(&mass[b], (u64)__double_as_longlong(w) - kNoStepsBits);
                if (R.k) atomicAdd(&count[b], one);
            }
        });
    } else {
        u64 kept = 0;
        each([&](double d) {
            const u64 w = steps(d, R, A, F);
            all += w;
            kept += d >= R.d_min ? w : 0;
        });
        kept = wave_sum(kept);
        if (SHARE == 1 && lane == 0 && unit < A.units) A.unit_sums[(int64_t)row * A.units + unit] = kept;
        if (SHARE > 1 && lane == 0) ks[wave] = kept;
    }
    if (R.filtered) {
        __syncthreads();
        for (int i = t; i < kBins; i += 64 * WAVES) {
            const u64 m = mass[bin_at(i)];
            if (!m) continue;
            all += m;
            atomicAdd(&A.bin_mass[(int64_t)row * kBins + i], m);
            if (R.k) atomicAdd(&A.bin_count[(int64_t)row * kBins + i], count[bin_at(i)]);
        }
    }
    all = wave_sum(all);
    if (lane == 0) ss[wave] = all;
    __syncthreads();
    if (SHARE > 1 && !R.filtered) put_unit_sums<WAVES, SHARE>(A, row, ks);
    if (t) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) all += ss[w];
    A.span_sums[(int64_t)row * A.spans + blockIdx.x] = all;
}

// A token is kept while the weight before it is under p * total: while it is under this.
__device__ __forceinline__ u64 mass_target(double p, u64 total) {
    const double m = ceil(p * (double)total);
    return m >= 1.0 ? (u64)m : 1;
}

// A logit below which all lie in bins behind `bin`, a little lower than the least such one, so that f32 will do.
__device__ __forceinline__ float least_of(const SampleArgs &A, const Row &R, int bin) {
    if (R.inf || !(R.bins > 0.0) || bin >= kBins - 1) return -INFINITY;
    const float y = (float)(R.top - (bin + 1.5) * __builtin_amdgcn_rcp(R.bins));
    if (A.cap.cap == 0.0) return y - 1e-6f * fabsf(y);
    const float cap = (float)A.cap.cap, r = fminf(y / cap, 0.9999f);
    if (!(r > -0.9999f)) return -INFINITY;
    const float z = 0.5f * cap * __logf((1.0f + r) / (1.0f - r));
    return z - 1e-3f * (fabsf(z) + cap);
}

// Inclusive sum over a wave's lanes.
template <class T>
__device__ __forceinline__ T wave_run(T v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const T o = __shfl_up(v, s);
        if ((int)(threadIdx.x & 63) >= s) v += o;
    }
    return v;
}

// A lane's 16 bins of a row.
struct LaneBins {
    u64 m[kBinsPer];
    uint32_t n[kBinsPer];
    __device__ __forceinline__ void load(const SampleArgs &A, int row) {
        const int64_t at = (int64_t)row * kBins + (threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
            m[i] = A.bin_mass[at + 64 * i];
            n[i] = A.bin_count[at + 64 * i];
        }
    }
};

// The bins of a row's cuts, by one wave, the same in every lane.
__device__ __forceinline__ Cuts find_cuts(const SampleArgs &A, const Row &R, const LaneBins &B) {
    const int lane = threadIdx.x & 63;
    const auto &m = B.m;
    const auto &n = B.n;
    u64 m_sum = 0;
    uint32_t n_sum = 0;
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
        m_sum += m[i];
        n_sum += n[i];
    }
    const u64 m_run = wave_run(m_sum), m_all = __shfl(m_run, 63), m_first = m_run - m_sum;
    const uint32_t n_run = wave_run(n_sum), n_all = __shfl(n_run, 63), n_first = n_run - n_sum;
    Cuts C{kBins, kBins, kBins, 0, 0, 0, 0.0f, 0.0f};
    const bool by_k = R.k > 0 && (uint32_t)R.k < n_all;
    u64 low_total = m_all, high_total = m_all;
    if (by_k) {
        const uint32_t k = R.k;
        const bool mine = n_first < k && k <= n_run;  // one lane
        int bin = 0, rest = 0;
        u64 mb = m_first, before = 0, after = 0;
        uint32_t nb = n_first;
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
            if (nb < k && k <= nb + n[i]) {
                bin = lane * kBinsPer + i;
                rest = (int)(k - nb);
                before = mb;
                after = mb + m[i];
            }
            mb += m[i];
            nb += n[i];
        }
        const int at = __ffsll((long long)__ballot(mine)) - 1;
        C.k_bin = __shfl(bin, at);
        C.k_rest = __shfl(rest, at);
        C.k_before = low_total = __shfl(before, at);
        high_total = __shfl(after, at);
        C.p_low = C.p_high = C.k_bin;
    }
    if (R.p < 1.0) {
        // the weight that top-k leaves lies between that above its bin and that with it
        const u64 low = mass_target(R.p, low_total), high = mass_target(R.p, high_total);
        int low_bin = 0, high_bin = 0;
        u64 mb = m_first, before = 0;
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
            if (mb < low && low <= mb + m[i]) {
                low_bin = lane * kBinsPer + i;
                before = mb;
            }
            if (mb < high && high <= mb + m[i]) high_bin = lane * kBinsPer + i;
            mb += m[i];
        }
        const int low_at = __ffsll((long long)__ballot(m_first < low && low <= m_run)) - 1;
        const int high_at = __ffsll((long long)__ballot(m_first < high && high <= m_run)) - 1;
        C.p_low = __shfl(low_bin, low_at);
        C.p_before = __shfl(before, low_at);
        C.p_high = __shfl(high_bin, high_at);
    }
    C.least = least_of(A, R, max(C.p_high, by_k ? C.k_bin : 0));
    return C;
}

// Four rows a block, a wave each: for calls of many blocks, each of which would do it again (5.2 us).
__global__ __launch_bounds__(kSampleThreads) void sample_find_kernel(SampleArgs A, int rows) {
    const int row = blockIdx.x * kSampleWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= rows) return;
    LaneBins B;
    B.load(A, row);
    const Row R = uniform_at(A.row + row);
    if (!R.filtered) return;
    const Cuts C = find_cuts(A, R, B);
    if ((threadIdx.x & 63) == 0) A.cut[row] = C;
}

// A wave's unit of a row with cuts: the weight above them, and what lies in their bins to the list. v: its logits, at x.
template <bool CAP, int PER>
__device__ __forceinline__ u64 cut_unit(const SampleArgs &A, const Row &R, const Cuts &c, int row, const float *x, int base,
                                        const float (&v)[PER]) {
    const int lane = threadIdx.x & 63;
    u64 sure = 0;
    uint32_t far = 0, in = 0;  // places where a lane's token is past half the cap, and may count; a lane's for the list
    int many = 0;
    const int low = min(c.p_low, c.k_bin), wide = max(c.p_high, c.k_bin < kBins ? c.k_bin : 0) - low;
    auto take = [&](int j, double d, bool real) {
        const int b = bin_of(d, R);
        const u64 w = real ? steps(d, R, A) : 0;
        if (b < c.p_low && d >= R.d_min) sure += w;
        if (__any((uint32_t)(b - low) <= (uint32_t)wide)) {  // few: the cuts' bins are narrow
            const bool mine = w && ((b >= c.p_low && b <= c.p_high) || b == c.k_bin);
            in |= mine ? 1u << j : 0u;
            many += __popcll(__ballot(mine));
        }
    };
    float most = 0.0f;
    if (CAP) {
#pragma unroll
        for (int j = 0; j < PER; ++j) most = fmaxf(most, fabsf(v[j]));
    }
    const bool some = CAP && __any(most > A.cap.half_cap);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (!__any(v[j] >= c.least)) continue;
        const float xs = seen(clean(v[j]), R);
        bool real = xs > -INFINITY;
        if (some) {
            const bool f = is_far(xs, A.cap);
            far |= __any(f && v[j] >= c.least) ? 1u << j : 0u;
            real = real && !f;
        }
        take(j, near_distance<CAP>(xs, R, A), real);
    }
    if (CAP)
        for (; far; far &= far - 1) {
            const int j = __ffs(far) - 1, i = base + unit_place(j, lane, A.vec);
            const float xs = i < A.vocab ? x[i] : -INFINITY;
            take(j, distance<CAP>(xs, R, A), is_far(xs, A.cap));
        }
    if (many) {
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&A.listed[(int64_t)row * kLineWords], (uint32_t)many);
        at = __shfl(at, 0);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool mine = in >> j & 1;
            const u64 who = __ballot(mine);
            const uint32_t place = at + __popcll(who & ((1ull << lane) - 1));
            if (mine && place < (uint32_t)kList)
                A.list[(int64_t)row * kList + place] = order_key(seen(v[j], R), base + unit_place(j, lane, A.vec));
            at += __popcll(who);
        }
    }
    return wave_sum(sure);
}

// Grid (spans, rows): a block finds its row's cuts itself, its logits on their way. One row 5.2 us, 32 rows of 262144 11.6.
template <bool CAP, int WAVES, int SHARE>
__global__ __launch_bounds__(64 * WAVES) void sample_cut_kernel(SampleArgs A) {
    __shared__ Cuts shared_cuts;
    __shared__ u64 ss[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.y;
    const int place = blockIdx.x * WAVES + wave, unit = place / SHARE, base = place * (kSampleUnit / SHARE);
    const float *x = row_of(A, row);
    const float top = unit < A.units ? A.unit_max[(int64_t)row * A.units + unit] : -INFINITY;
    float v[kSamplePer / SHARE];
    load_unit(x + base, x ? A.vocab - base : 0, lane, A.vec, v);
    LaneBins B;
    if (wave == 0) B.load(A, row);
    const Row R = uniform_at(A.row + row);
    if (!R.filtered) return;  // (a row without a logit, too)
    if (wave == 0) {
        const Cuts C = find_cuts(A, R, B);
        if (lane == 0) {
            shared_cuts = C;
            if (blockIdx.x == 0) A.cut[row] = C;
        }
    }
    __syncthreads();
    const Cuts c = uniform(shared_cuts);
    if (SHARE == 1 && unit >= A.units) return;
    const u64 sure = unit < A.units && top >= c.least ? cut_unit<CAP>(A, R, c, row, x, base, v) : 0;
    if (SHARE == 1) {
        if (lane == 0) A.unit_sums[(int64_t)row * A.units + unit] = sure;
        return;
    }
    if (lane == 0) ss[wave] = sure;
    __syncthreads();
    put_unit_sums<WAVES, SHARE>(A, row, ss);
}

// Grid (units by 4, rows), behind sample_find_kernel: units that do not reach up to the cuts are not read. 256 rows of
// mixed filters, a third of whose units do: 40 us, by the operations of those (40 a logit) and the waves that come and go.
template <bool CAP>
__global__ __launch_bounds__(kSampleThreads, 8) void sample_cut_found_kernel(SampleArgs A) {
    const int lane = threadIdx.x & 63, row = blockIdx.y;
    const int unit = blockIdx.x * kSampleWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), base = unit * kSampleUnit;
    const Row R = uniform_at(A.row + row);
    const Cuts c = uniform_at(A.cut + row);
    if (!R.filtered || unit >= A.units) return;
    const float *x = row_of(A, row);
    u64 sure = 0;
    if (uniform_at(A.unit_max + (int64_t)row * A.units + unit) >= c.least) {
        float v[kSamplePer];
        load_unit(x + base, A.vocab - base, lane, A.vec, v);
        sure = cut_unit<CAP>(A, R, c, row, x, base, v);
    }
    if (lane == 0) A.unit_sums[(int64_t)row * A.units + unit] = sure;
}

__device__ __forceinline__ float logit_of(u64 key) {
    const uint32_t up = (uint32_t)(key >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

// A token that a cut is looked for among: in top-k's bin, in top-p's bins, or in neither (then it is none).
struct Near {
    u64 key, w;
    bool k, p, kept;  // kept: by min-p
};
template <bool CAP>
__device__ __forceinline__ Near near_of(const SampleArgs &A, const Row &R, const Cuts &C, u64 key) {
    Near e{key, 0, false, false, false};
    if (!key) return e;
    const double d = distance<CAP>(logit_of(key), R, A);
    e.w = steps(d, R, A);
    const int b = bin_of(d, R);
    e.k = e.w && b == C.k_bin;
    e.p = e.w && b >= C.p_low && b <= C.p_high;
    e.kept = d >= R.d_min;
    return e;
}

__device__ __forceinline__ u64 lane64(u64 v, int lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// Among a wave's tokens, one a lane where `is`, in falling order of their keys: the one where the running weight
// (by_p) or count first reaches `target`. Returns its key, and in *mass the weight up to it; the same in every lane.
__device__ __forceinline__ u64 wave_cut(u64 key, u64 w, bool is, bool by_p, u64 target, u64 *mass) {
    u64 m = 0, n = 0;
    for (u64 left = __ballot(is); left; left &= left - 1) {
        const int j = __ffsll((long long)left) - 1;
        const u64 k = lane64(key, j), o = lane64(w, j);
        m += k > key ? o : 0;
        n += k > key ? 1 : 0;
    }
    const u64 run = by_p ? m : n, one = by_p ? w : 1;
    const u64 at = __ballot(is && run < target && target <= run + one);
    if (!at) return 0;  // nothing reaches it: all are kept
    const int j = __ffsll((long long)at) - 1;
    *mass = lane64(m + w, j);
    return lane64(key, j);
}

constexpr int kCache = 2048;  // entries that the last kernel's block holds in LDS
constexpr u64 kNearK = 1ull << 63, kNearP = 1ull << 62, kNearKept = 1ull << 61, kNearW = (1ull << 53) - 1;

struct PickShared {
    u64 key[kCache], w[kCache];  // the list; w: and the kNear bits
    u64 mass[kSub];
    uint32_t count[kSub];
    u64 sums[2][kSampleWaves];
    u64 few_key[kFew], few_w[kFew];
    u64 high[2], low[2];  // keys among top-k's tokens and top-p's
    u64 before, mass_before;
    uint32_t at, count_at, few;
};

// What a block looks its row's cuts up in where a wave cannot: the list in LDS, the list, or, where that overflowed, the
// row. That is one block's reading of the whole row several times over: a row of 262144 logits on a grid of 0.25, more than
// 4096 of them in top-p's bins, takes 1.8 ms where other such rows take 36 us, 256 of them 2.7 ms and 0.32.
template <bool CAP>
struct Search {
    const SampleArgs &A;
    const Row &R;
    const Cuts &C;
    const float *x;
    PickShared &S;
    const u64 *list;
    int n;

    // Every token of the cuts' bins with f(key, w and bits), from where it lies.
    template <class F>
    __device__ __forceinline__ void each_given(F f) {
        const bool whole = n > kList;
        const int end = whole ? A.vocab : n;
        for (int i = threadIdx.x; i < end; i += kSampleThreads) {
            u64 key;
            if (whole) {
                const float v = seen(clean(x[i]), R);
                key = v > -INFINITY && v >= C.least ? order_key(v, i) : 0;
            } else {
                key = list[i];
            }
            const Near e = near_of<CAP>(A, R, C, key);
            f(i, key, e.w | (e.k ? kNearK : 0) | (e.p ? kNearP : 0) | (e.kept ? kNearKept : 0));
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) {
        if (n <= kCache) {
            for (int i = threadIdx.x; i < n; i += kSampleThreads) f(S.key[i], S.w[i]);
        } else {
            each_given([&](int, u64 key, u64 w) { f(key, w); });
        }
    }
    // First of all: the list to LDS, and the ranges of keys.
    __device__ __forceinline__ void begin() {
        const int t = threadIdx.x;
        if (t < 2) {
            S.high[t] = 0;
            S.low[t] = ~0ull;
        }
        __syncthreads();
        u64 high[2] = {0, 0}, low[2] = {~0ull, ~0ull};
        each_given([&](int i, u64 key, u64 w) {
            if (n <= kCache) {
                S.key[i] = key;
                S.w[i] = w;
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const bool is = w & (p ? kNearP : kNearK);
                high[p] = is && key > high[p] ? key : high[p];
                low[p] = is && key < low[p] ? key : low[p];
            }
        });
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int s = 32; s; s >>= 1) {
                const u64 h = __shfl_xor(high[p], s), l = __shfl_xor(low[p], s);
                high[p] = h > high[p] ? h : high[p];
                low[p] = l < low[p] ? l : low[p];
            }
            if ((t & 63) == 0) {
                atomicMax(&S.high[p], high[p]);
                atomicMin(&S.low[p], low[p]);
            }
        }
        __syncthreads();
    }

    // As wave_cut, among top-p's (by_p) or top-k's tokens with a key of at least `least`. Each step splits the range of
    // keys in 1024, until a wave can order what is left.
    __device__ u64 refine(bool by_p, u64 least, u64 target, u64 *mass) {
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
        const u64 bit = by_p ? kNearP : kNearK;
        u64 hi = S.high[by_p], lo = S.low[by_p], mass_sum = 0;
        lo = lo < least ? least : lo;
        while (true) {
            const int bits = 64 - __clzll((long long)((hi - lo) | 1)), sh = bits > 10 ? bits - 10 : 0;
#pragma unroll
            for (int i = 0; i < kSubPer; ++i) S.mass[t * kSubPer + i] = S.count[t * kSubPer + i] = 0;
            if (t == 0) {
                S.at = kSub;
                S.few = 0;
            }
            __syncthreads();
            each([&](u64 key, u64 w) {
                if (!(w & bit) || key < lo || key > hi) return;
                atomicAdd(&S.mass[(hi - key) >> sh], w & kNearW);
                atomicAdd(&S.count[(hi - key) >> sh], 1u);
            });
            __syncthreads();
            u64 m[kSubPer], c[kSubPer], m_run = 0, c_run = 0;
#pragma unroll
            for (int i = 0; i < kSubPer; ++i) {
                m[i] = S.mass[t * kSubPer + i];
                c[i] = S.count[t * kSubPer + i];
                m_run += m[i];
                c_run += c[i];
            }
            const u64 m_mine = m_run, c_mine = c_run;
            m_run = wave_run(m_run);
            c_run = wave_run(c_run);
            if (lane == 63) {
                S.sums[0][wave] = m_run;
                S.sums[1][wave] = c_run;
            }
            __syncthreads();
            m_run -= m_mine;
            c_run -= c_mine;
            u64 m_all = 0;
#pragma unroll
            for (int o = 0; o < kSampleWaves; ++o) {
                m_all += S.sums[0][o];
                if (o < wave) {
                    m_run += S.sums[0][o];
                    c_run += S.sums[1][o];
                }
            }
#pragma unroll
            for (int i = 0; i < kSubPer; ++i) {
                const u64 run = by_p ? m_run : c_run, one = by_p ? m[i] : c[i];
                if (run < target && target <= run + one) {  // one thread, or none where nothing reaches it
                    S.at = t * kSubPer + i;
                    S.before = run;
                    S.mass_before = m_run;
                    S.count_at = (uint32_t)c[i];
                }
                m_run += m[i];
                c_run += c[i];
            }
            __syncthreads();
            const uint32_t at = S.at, left = S.count_at;
            if (at == kSub) {
                *mass = mass_sum + m_all;
                __syncthreads();
                return lo;
            }
            target -= S.before;
            mass_sum += S.mass_before;
            hi -= (u64)at << sh;
            const u64 width = (1ull << sh) - 1;
            lo = hi - lo > width ? hi - width : lo;
            if (left > kFew) {  // (a range of one key holds one token)
                __syncthreads();
                continue;
            }
            each([&](u64 key, u64 w) {
                if (!(w & bit) || key < lo || key > hi) return;
                const uint32_t place = atomicAdd(&S.few, 1u);
                S.few_key[place] = key;
                S.few_w[place] = w & kNearW;
            });
            __syncthreads();
            const bool is = lane < (int)left;
            u64 rest = 0;
            const u64 cut = wave_cut(is ? S.few_key[lane] : 0, is ? S.few_w[lane] : 0, is, by_p, target, &rest);
            *mass = mass_sum + rest;
            __syncthreads();
            return cut;
        }
    }
};

// One block per row. Dynamic LDS: a sum a unit, of the list's weights where that has more than kFew. Bound by its chain: the
// list and the units' sums, the cuts, the unit, its logits, the token. 5.9 us for a row, 17.6 for 256 of mixed filters.
template <bool CAP>
__global__ __launch_bounds__(kSampleThreads) void sample_pick_kernel(SampleArgs A) {
    extern __shared__ u64 extra[];
    __shared__ PickShared S;
    const int t = threadIdx.x, lane = t & 63, row = blockIdx.x;
    const float *x = row_of(A, row);
    // all that may be asked for, at once; of a row without cuts the last three are not used
    const float u = A.u[row];
    const u64 *list = A.list + (int64_t)row * kList;
    const uint32_t n = A.listed[(int64_t)row * kLineWords];
    const u64 first_key = list[lane];
    const Cuts C = uniform_at(A.cut + row);
    u64 all = 0;
    for (int c = lane; c < A.spans; c += 64) all += A.span_sums[(int64_t)row * A.spans + c];
    const u64 *units = A.unit_sums + (int64_t)row * A.units;
    const int per = (A.units + kSampleThreads - 1) / kSampleThreads, u0 = min(t * per, A.units), u1 = min(u0 + per, A.units);
    u64 mine = 0;
    for (int i = u0; i < u1; ++i) mine += units[i];
    const Row R = uniform_at(A.row + row);
    if (R.index < 0) {
        if (t == 0) {
            A.tokens[row] = -1;
            if (A.logprobs) A.logprobs[row] = 0.0f;
        }
        return;
    }
    all = wave_sum(all);  // every wave by itself
    if (R.greedy) {
        if (t == 0) {
            A.tokens[row] = R.index;
            if (A.logprobs) A.logprobs[row] = (float)(A.shift * 0.69314718055994530942 - log((double)all));
        }
        return;
    }
    u64 cut = 0;  // the last kept key
    bool spread = false;  // the list's weights are in `extra`
    Near e{0, 0, false, false, false};
    u64 few = 0;  // lanes with an element that is kept
    if (R.filtered && C.p_low < kBins) {
        u64 mass = all;
        if (n <= kFew) {
            e = near_of<CAP>(A, R, C, lane < (int)n ? first_key : 0);
            if (C.k_bin < kBins) {
                cut = wave_cut(e.key, e.w, e.k, false, C.k_rest, &mass);
                mass += C.k_before;
            }
            if (R.p < 1.0)
                cut = wave_cut(e.key, e.w, e.p && e.key >= cut, true, mass_target(R.p, mass) - C.p_before, &mass);
            few = __ballot((e.k || e.p) && e.key >= cut && e.kept);
            for (u64 left = few; left; left &= left - 1) {
                const int j = __ffsll((long long)left) - 1;
                const int unit = (int)(~(uint32_t)__builtin_amdgcn_readlane((int)e.key, j) / kSampleUnit);
                const u64 w = lane64(e.w, j);
                mine += unit >= u0 && unit < u1 ? w : 0;
            }
        } else {
            Search<CAP> L{A, R, C, x, S, list, (int)min(n, (uint32_t)kList + 1)};
            for (int i = t; i < A.units; i += kSampleThreads) extra[i] = 0;
            L.begin();
            if (C.k_bin < kBins) {
                cut = L.refine(false, 0, C.k_rest, &mass);
                mass += C.k_before;
            }
            if (R.p < 1.0) cut = L.refine(true, cut, mass_target(R.p, mass) - C.p_before, &mass);
            L.each([&](u64 key, u64 w) {
                if (key >= cut && (w & (kNearK | kNearP)) && (w & kNearKept))
                    atomicAdd(&extra[~(uint32_t)key / kSampleUnit], w & kNearW);
            });
            __syncthreads();
            spread = true;
            for (int i = u0; i < u1; ++i) mine += extra[i];
        }
    }
    // the unit, then the token, where the running sum passes u of the total
    u64 total;
    if (t == 0) {
        S.at = 0;
        S.before = 0;
    }
    u64 run = block_run(mine, S.sums[0], &total) - mine;
    const float uf = fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f);  // NaN: 0
    u64 target = (u64)((double)uf * (double)total);
    const bool here = run <= target && target < run + mine;  // one thread
    if (__any(here)) {
        for (int i = u0; i < u1; ++i) {
            u64 w = units[i] + (spread ? extra[i] : 0);
            for (u64 left = few; left; left &= left - 1) {
                const int j = __ffsll((long long)left) - 1;
                if ((int)(~(uint32_t)__builtin_amdgcn_readlane((int)e.key, j) / kSampleUnit) == i) w += lane64(e.w, j);
            }
            if (here && run <= target && target < run + w) {
                S.at = i;
                S.before = run;
            }
            run += w;
        }
    }
    __syncthreads();
    const int base = (int)S.at * kSampleUnit + t * kUnitPer;
    target -= S.before;
    u64 w[kUnitPer];
    double d[kUnitPer];
    mine = 0;
#pragma unroll
    for (int i = 0; i < kUnitPer; ++i) {
        const int id = base + i;
        const float v = id < A.vocab ? seen(clean(x[id]), R) : -INFINITY;
        d[i] = distance<CAP>(v, R, A);
        w[i] = v > -INFINITY && d[i] >= R.d_min && order_key(v, id) >= cut ? steps(d[i], R, A) : 0;
        mine += w[i];
    }
    run = block_run(mine, S.sums[1], &total) - mine;
    if (run <= target && target < run + mine) {
#pragma unroll
        for (int i = 0; i < kUnitPer; ++i) {
            if (run <= target && target < run + w[i]) {
                A.tokens[row] = base + i;
                if (A.logprobs)  // less the log of the sum of all weights, from steps
                    A.logprobs[row] = (float)(d[i] * R.inv_t + A.shift * 0.69314718055994530942 - log((double)all));
            }
            run += w[i];
        }
    }
}

template <bool CAP>
static int launch_sample(const SampleArgs &A, int rows, hipStream_t s) {
    hipLaunchKernelGGL(sample_max_kernel, dim3(A.parts, rows), dim3(kSampleThreads), 0, s, A);
    G4_LAUNCHED("sample_max_kernel");
    const dim3 grid(A.spans, rows), block(64 * A.wide), by_row((rows + kSampleWaves - 1) / kSampleWaves);
    if (A.many) {
        hipLaunchKernelGGL(sample_row_kernel, by_row, dim3(kSampleThreads), 0, s, A, rows);
        G4_LAUNCHED("sample_row_kernel");
        hipLaunchKernelGGL((sample_weights_kernel<CAP, 8, 1, true>), grid, block, 0, s, A);
    } else if (A.wide == 16) {
        hipLaunchKernelGGL((sample_weights_kernel<CAP, 16, 4, false>), grid, block, 0, s, A);
    } else if (A.share == 4) {
        hipLaunchKernelGGL((sample_weights_kernel<CAP, 8, 4, false>), grid, block, 0, s, A);
    } else {
        hipLaunchKernelGGL((sample_weights_kernel<CAP, 8, 1, false>), grid, block, 0, s, A);
    }
    G4_LAUNCHED("sample_weights_kernel");
    if (A.cuts && A.many) {
        hipLaunchKernelGGL(sample_find_kernel, by_row, dim3(kSampleThreads), 0, s, A, rows);
        G4_LAUNCHED("sample_find_kernel");
        const dim3 by_unit((A.units + kSampleWaves - 1) / kSampleWaves, rows);
        hipLaunchKernelGGL(sample_cut_found_kernel<CAP>, by_unit, dim3(kSampleThreads), 0, s, A);
        G4_LAUNCHED("sample_cut_found_kernel");
    } else if (A.cuts) {
        if (A.wide == 16) hipLaunchKernelGGL((sample_cut_kernel<CAP, 16, 4>), grid, block, 0, s, A);
        else if (A.share == 4) hipLaunchKernelGGL((sample_cut_kernel<CAP, 8, 4>), grid, block, 0, s, A);
        else hipLaunchKernelGGL((sample_cut_kernel<CAP, 8, 1>), grid, block, 0, s, A);
        G4_LAUNCHED("sample_cut_kernel");
    }
    hipLaunchKernelGGL(sample_pick_kernel<CAP>, dim3(rows), dim3(kSampleThreads), A.units * sizeof(u64), s, A);
    G4_LAUNCHED("sample_pick_kernel");
    return G4_OK;
}

static int64_t sample_parts(int64_t vocab) { return (vocab + kSamplePart - 1) / kSamplePart; }
static int64_t sample_units(int64_t vocab) { return (vocab + kSampleUnit - 1) / kSampleUnit; }

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_sample_workspace_bytes(int rows, int64_t vocab) {
    if (rows <= 0 || rows > 65535 || vocab <= 0 || vocab > kMaxVocab) return 0;
    const size_t row = (size_t)sample_parts(vocab) * sizeof(PartMax) +
                       (size_t)sample_units(vocab) * (2 * sizeof(u64) + sizeof(float)) + kBins * (sizeof(u64) + sizeof(uint32_t)) +
                       kList * sizeof(u64) + sizeof(Row) + sizeof(Cuts) + kLineWords * sizeof(uint32_t);
    return rows * row;
}

int g4_sample_tokens(const float *logits, int logit_rows, int64_t logit_stride, const int32_t *row_index, int rows,
                     int64_t vocab, float cap, const float *temperature, const int32_t *top_k, const float *top_p,
                     const float *min_p, const float *u, void *workspace, size_t workspace_bytes, int32_t *tokens,
                     float *logprobs, void *stream) {
    if (rows <= 0 || logit_rows <= 0 || vocab <= 0)
        return set_error(G4_ERR_INVALID, "sample-tokens: %d rows of %d, vocabulary %lld", rows, logit_rows, (long long)vocab);
    if (vocab > kMaxVocab || rows > 65535)
        return set_error(G4_ERR_UNSUPPORTED, "sample-tokens: %d rows, vocabulary %lld (at most 65535 and %d)", rows,
                         (long long)vocab, kMaxVocab);
    if (!row_index && rows > logit_rows)
        return set_error(G4_ERR_INVALID, "sample-tokens: %d rows from %d rows of logits need row_index", rows, logit_rows);
    if (!(cap >= 0.0f) || std::isinf(cap)) return set_error(G4_ERR_INVALID, "sample-tokens: cap must be finite and at least 0");
    if (!logits || !u || !tokens) return set_error(G4_ERR_INVALID, "sample-tokens needs logits, u and tokens");
    if (logit_stride && logit_stride < vocab)
        return set_error(G4_ERR_INVALID, "sample-tokens: logit_stride %lld < vocabulary %lld", (long long)logit_stride,
                         (long long)vocab);
    const size_t need = g4_sample_workspace_bytes(rows, vocab);
    if (!workspace || workspace_bytes < need)
        return set_error(G4_ERR_INVALID, "sample-tokens: workspace %zu B < %zu B", workspace_bytes, need);
    if ((uintptr_t)workspace & 15) return set_error(G4_ERR_INVALID, "sample-tokens: the workspace must be 16-byte aligned");
    SampleArgs A{};
    A.logits = logits;
    A.stride = logit_stride ? logit_stride : vocab;
    A.row_index = row_index;
    A.temperature = temperature;
    A.top_k = top_k;
    A.top_p = top_p;
    A.min_p = min_p;
    A.u = u;
    A.cap = {cap, cap > 0.0f ? 1.0 / cap : 0.0, cap > 0.0f ? 1.0 / ((double)cap * cap) : 0.0, 0.4999999f * cap};
    A.logit_rows = logit_rows;
    A.vocab = (int)vocab;
    A.parts = (int)sample_parts(vocab);
    A.units = (int)sample_units(vocab);
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    A.shift = 62 - bits < 51 ? 62 - bits : 51;
    A.vec = A.stride % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    A.cuts = top_k || top_p;
    // A block's waves have its fixed work together, the row's parameters, its histogram and its cuts. Where a wave a unit would
    // leave SIMDs with few, four share one: 1 row of 262144 21.3 us, a wave a unit 24.1; 32 rows of 32003 30.3 and 36.2;
    // 6 rows of 262144 (1536 units) 32-45 and 34; 2000 rows of 1024 62 and 88. In a wide row by 16 waves a block, since each
    // block adds to the row's histogram: 1 row of 262144 21.3 us, 8 waves 23.1; 32 rows of 32003 30.3 and 31.0.
    A.share = (int64_t)rows * A.units <= 4 * device_cu_count() || A.units <= 2 ? 4 : 1;
    A.wide = A.share == 4 && A.units >= kWideRow ? 16 : 8;
    A.spans = (A.units * A.share + A.wide - 1) / A.wide;  // at most units
    // More blocks than are there at once would each make the row's parameters and cuts: two launches more, 56 rows (1792
    // blocks) 71.3 us and without 75.5, 32 rows (1024) 55.2 and 51.5
    A.many = A.share == 1 && (int64_t)rows * A.spans > 4 * device_cu_count();
    A.stats = static_cast<PartMax *>(workspace);
    A.row = reinterpret_cast<Row *>(A.stats + (int64_t)rows * A.parts);
    A.cut = reinterpret_cast<Cuts *>(A.row + rows);
    A.span_sums = reinterpret_cast<u64 *>(A.cut + rows);
    A.unit_sums = A.span_sums + (int64_t)rows * A.units;
    A.bin_mass = A.unit_sums + (int64_t)rows * A.units;
    A.list = A.bin_mass + (int64_t)rows * kBins;
    A.bin_count = reinterpret_cast<uint32_t *>(A.list + (int64_t)rows * kList);
    A.listed = A.bin_count + (int64_t)rows * kBins;
    A.unit_max = reinterpret_cast<float *>(A.listed + (int64_t)rows * kLineWords);
    A.tokens = tokens;
    A.logprobs = logprobs;
    hipStream_t s = as_stream(stream);
    return cap > 0.0f ? launch_sample<true>(A, rows, s) : launch_sample<false>(A, rows, s);
}

}  // extern "C"
