// Sampling with temperature, top-k, top-p and min-p from given random numbers (include/g4serve.h).
//
// All filters keep a prefix of the row ordered by (logit down, id up), so a row's kept set is one cut in that
// order, and min-p a bound on the logit beside it. The order is never made: (1) every part's maximum and minimum; (2)
// weights, and for a row with top-k or top-p a histogram of them over bins of the capped logit; (3) the bins where the
// cuts lie, from the histogram, the weights of what lies above them by units of 1024 tokens, and a list of what
// lies in them; (4) a block per row refines the cuts within its list, finds the unit and then the token where the
// running sum passes u of the total. A row without top-k and top-p has its units' weights from (2).
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
constexpr int kBins = 1024, kBinsPer = kBins / kSampleThreads;
constexpr int kList = 4096;  // entries; a row with more is read again
constexpr int kPickThreads = 1024, kListPer = kList / kPickThreads;
constexpr int kSub = 1024;  // ranges of one refinement step, one a thread
static_assert(kSub == kPickThreads && kSampleUnit == kPickThreads, "the last kernel has one thread each");
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
    PartMax *stats;              // [rows][parts]
    u64 *part_sums, *unit_sums;  // [rows][parts], [rows][units]
    u64 *bin_mass;               // [rows][kBins]
    u64 *list;                   // [rows][kList]
    Cuts *cut;                   // [rows]
    uint32_t *bin_count;         // [rows][kBins]
    uint32_t *listed;            // [rows]
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

// The lane's values of the wave's unit at x, `n` of which exist.
__device__ __forceinline__ void load_unit(const float *x, int n, int lane, int vec, float (&v)[kSamplePer]) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < kSamplePer; j += 4) {
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
        for (int j = 0; j < kSamplePer; ++j) {
            const int i = unit_place(j, lane, 0);
            v[j] = i < n ? x[i] : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) v[j] = clean(v[j]);
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

// Grid (parts, rows). Also clears the row's histogram and list for the kernels behind.
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
        for (int i = part * kSampleThreads + t; i < kBins; i += A.parts * kSampleThreads) {
            A.bin_mass[(int64_t)row * kBins + i] = 0;
            A.bin_count[(int64_t)row * kBins + i] = 0;
        }
        if (part == 0 && t == 0) A.listed[row] = 0;
    }
    __syncthreads();
    if (t) return;
#pragma unroll
    for (int w = 1; w < kSampleWaves; ++w) join_max(m, ms[w].max, ms[w].min, ms[w].index);
    A.stats[(int64_t)row * A.parts + part] = m;
}

// What a row's weights are made with.
struct Row {
    double top, slope, d_min, bins;  // weight 2^((y - top) slope), kept from d_min on, bin (top - y) bins
    double inv_t, p;
    int index, k;                // the first maximum (-1: no logit)
    bool greedy, filtered, inf;  // inf: the maximum is +infinity, whose like share all weight
};

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
    const double t = R.greedy ? 1.0 : tf;
    R.inv_t = 1.0 / t;
    R.slope = R.inv_t * 1.4426950408889634074;
    R.inf = A.cap.cap == 0.0 && m.max == INFINITY;
    R.top = R.inf || m.index < 0 ? 0.0 : softcap64(m.max, A.cap);
    R.d_min = mf > 0.0f ? (mf >= 1.0f ? 0.0 : log((double)mf) * t) : -INFINITY;
    R.k = k < A.vocab ? k : 0;
    R.p = pf < 1.0f ? (double)pf : 1.0;  // NaN: off
    R.filtered = !R.greedy && m.index >= 0 && (R.k > 0 || R.p < 1.0);
    // the bins reach from the top to the lowest logit, or to where weights round to no step
    double range = R.inf || m.index < 0 ? 0.0 : R.top - softcap64(m.min, A.cap);
    range = fmin(range, (A.shift + 1) / R.slope);
    R.bins = range > 0.0 ? fmin((kBins - 1) / range, 1e300) : 0.0;
    return R;
}

// Under an infinite maximum a logit is as good as it, or nothing.
__device__ __forceinline__ float seen(float x, const Row &R) { return R.inf ? (x == INFINITY ? 0.0f : -INFINITY) : x; }

// y - top; for a -infinity that, or NaN.
template <bool CAP>
__device__ __forceinline__ double distance(float x, const Row &R, const SampleArgs &A) {
    double y = x;
    if (CAP) {
        y = near_cap(y, A.cap);
        if (is_far(x, A.cap)) y = far_cap(x, A.cap.cap);
    }
    return y - R.top;
}
__device__ __forceinline__ u64 steps(double d, const Row &R, const SampleArgs &A) {
    const double w = pow2(__builtin_fma(d, R.slope, (double)A.shift));  // at most 2^51 and a little
    return (u64)__double_as_longlong(w + 0x1p52) & ((1ull << 52) - 1);
}
__device__ __forceinline__ int bin_of(double d, const Row &R) { return min(max((int)(-d * R.bins), 0), kBins - 1); }

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
template <int THREADS>
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
    for (int w = 0; w < THREADS / 64; ++w) {
        const u64 s = lds[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return before + v;
}

// Grid (parts, rows).
template <bool CAP>
__global__ __launch_bounds__(kSampleThreads) void sample_weights_kernel(SampleArgs A) {
    __shared__ u64 mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ u64 ss[kSampleWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, part = blockIdx.x, row = blockIdx.y;
    const float *x = row_of(A, row);
    const int unit = part * kSampleWaves + wave, base = unit * kSampleUnit;
    float v[kSamplePer];
    if (x && base < A.vocab) {
        load_unit(x + base, A.vocab - base, lane, A.vec, v);
    } else {
#pragma unroll
        for (int j = 0; j < kSamplePer; ++j) v[j] = -INFINITY;
    }
    const Row R = row_params(A, row);
    if (R.index < 0) return;
    if (R.filtered) {
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
            mass[i * kSampleThreads + t] = 0;
            count[i * kSampleThreads + t] = 0;
        }
        __syncthreads();
    }
    u64 all = 0, kept = 0;
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
        const double d = distance<CAP>(seen(v[j], R), R, A);
        const u64 w = steps(d, R, A);
        all += w;
        if (!R.filtered) {
            kept += d >= R.d_min ? w : 0;
        } else if (w) {
            const int b = bin_of(d, R);
            atomicAdd(&mass[b], w);
            atomicAdd(&count[b], 1u);
        }
    }
    all = wave_sum(all);
    if (lane == 0) ss[wave] = all;
    if (!R.filtered) {
        kept = wave_sum(kept);
        if (lane == 0 && unit < A.units) A.unit_sums[(int64_t)row * A.units + unit] = kept;
    }
    __syncthreads();
    if (t == 0) A.part_sums[(int64_t)row * A.parts + part] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
    if (!R.filtered) return;
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
        const int b = i * kSampleThreads + t;
        if (!count[b]) continue;
        atomicAdd(&A.bin_mass[(int64_t)row * kBins + b], mass[b]);
        atomicAdd(&A.bin_count[(int64_t)row * kBins + b], count[b]);
    }
}

// A token is kept while the weight before it is under p * total: while it is under this.
__device__ __forceinline__ u64 mass_target(double p, u64 total) {
    const double m = ceil(p * (double)total);
    return m >= 1.0 ? (u64)m : 1;
}

// Grid (parts, rows): every block finds the bins of its row's cuts, then weighs its tokens above them.
template <bool CAP>
__global__ __launch_bounds__(kSampleThreads) void sample_cut_kernel(SampleArgs A) {
    __shared__ u64 sums[kSampleWaves];
    __shared__ Cuts C;
    __shared__ u64 k_after;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, part = blockIdx.x, row = blockIdx.y;
    const float *x = row_of(A, row);
    const int unit = part * kSampleWaves + wave, base = unit * kSampleUnit;
    float v[kSamplePer];
    if (x && base < A.vocab) {
        load_unit(x + base, A.vocab - base, lane, A.vec, v);
    } else {
#pragma unroll
        for (int j = 0; j < kSamplePer; ++j) v[j] = -INFINITY;
    }
    u64 m[kBinsPer], n[kBinsPer], m_sum = 0, n_sum = 0;
#pragma unroll
    for (int i = 0; i < kBinsPer; ++i) {
        m[i] = A.bin_mass[(int64_t)row * kBins + t * kBinsPer + i];
        n[i] = A.bin_count[(int64_t)row * kBins + t * kBinsPer + i];
        m_sum += m[i];
        n_sum += n[i];
    }
    const Row R = row_params(A, row);
    if (!R.filtered) return;
    if (t == 0) {
        C = {kBins, kBins, kBins, 0, 0, 0};
        k_after = 0;
    }
    u64 m_all, n_all;
    const u64 m_first = block_run<kSampleThreads>(m_sum, sums, &m_all) - m_sum;
    const u64 n_first = block_run<kSampleThreads>(n_sum, sums, &n_all) - n_sum;
    const bool by_k = R.k > 0 && (u64)R.k < n_all;
    if (by_k) {
        u64 mb = m_first, nb = n_first;
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
            if (nb < (u64)R.k && (u64)R.k <= nb + n[i]) {
                C.k_bin = t * kBinsPer + i;
                C.k_rest = R.k - (int)nb;
                C.k_before = mb;
                k_after = mb + m[i];
            }
            mb += m[i];
            nb += n[i];
        }
    }
    __syncthreads();
    if (R.p < 1.0) {
        // the weight that top-k leaves lies between that above its bin and that with it
        const u64 low = mass_target(R.p, by_k ? C.k_before : m_all), high = mass_target(R.p, by_k ? k_after : m_all);
        u64 mb = m_first;
#pragma unroll
        for (int i = 0; i < kBinsPer; ++i) {
            if (mb < low && low <= mb + m[i]) {
                C.p_low = t * kBinsPer + i;
                C.p_before = mb;
            }
            if (mb < high && high <= mb + m[i]) C.p_high = t * kBinsPer + i;
            mb += m[i];
        }
    } else if (by_k && t == 0) {
        C.p_low = C.p_high = C.k_bin;
    }
    __syncthreads();
    const Cuts c = C;
    if (part == 0 && t == 0) A.cut[row] = c;
    const int last = max(c.p_high, c.k_bin < kBins ? c.k_bin : 0);
    u64 sure = 0;
#pragma unroll
    for (int j = 0; j < kSamplePer; ++j) {
        const float xs = seen(v[j], R);
        const double d = distance<CAP>(xs, R, A);
        const bool near = d >= -INFINITY && xs > -INFINITY && bin_of(d, R) <= last;
        if (!__any(near)) continue;
        const int b = bin_of(d, R);
        const u64 w = near ? steps(d, R, A) : 0;
        if (w && b < c.p_low && d >= R.d_min) sure += w;
        const bool in = w && ((b >= c.p_low && b <= c.p_high) || b == c.k_bin);
        const u64 who = __ballot(in);
        if (!who) continue;
        uint32_t at = 0;
        if (lane == __ffsll((long long)who) - 1) at = atomicAdd(&A.listed[row], (uint32_t)__popcll(who));
        at = __shfl(at, __ffsll((long long)who) - 1) + __popcll(who & ((1ull << lane) - 1));
        if (in && at < (uint32_t)kList)
            A.list[(int64_t)row * kList + at] = order_key(xs, base + unit_place(j, lane, A.vec));
    }
    sure = wave_sum(sure);
    if (lane == 0 && unit < A.units) A.unit_sums[(int64_t)row * A.units + unit] = sure;
}

__device__ __forceinline__ float logit_of(u64 key) {
    const uint32_t up = (uint32_t)(key >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

// A token that a cut is looked for among: in top-k's bin, in top-p's bins, or in neither (then it is none).
struct Near {
    u64 key, w;
    double d;
    bool k, p;
};
template <bool CAP>
__device__ __forceinline__ Near near_of(const SampleArgs &A, const Row &R, const Cuts &C, u64 key) {
    Near e{key, 0, 0.0, false, false};
    if (!key) return e;
    e.d = distance<CAP>(logit_of(key), R, A);
    e.w = steps(e.d, R, A);
    const int b = bin_of(e.d, R);
    e.k = e.w && b == C.k_bin;
    e.p = e.w && b >= C.p_low && b <= C.p_high;
    return e;
}
// The same of token `id`, from the row: for lists that overflowed.
template <bool CAP>
__device__ __noinline__ Near near_at(const SampleArgs &A, const Row &R, const Cuts &C, const float *x, int id) {
    const float v = seen(clean(x[id]), R);
    return near_of<CAP>(A, R, C, v > -INFINITY ? order_key(v, id) : 0);
}

struct PickShared {
    u64 extra[kMaxVocab / kSampleUnit];  // of the units, from the list
    u64 mass[kSub];
    uint32_t count[kSub];
    u64 sums[kPickThreads / 64];
    u64 high, low, before, mass_before, mass_at, cut;
    uint32_t at, count_at;
};

// What the last kernel's block looks its row's cuts up in: the list, a few elements a thread, or the row again.
template <bool CAP>
struct Search {
    const SampleArgs &A;
    const Row &R;
    const Cuts &C;
    const float *x;
    PickShared &S;
    Near near[kListPer];
    bool whole;

    __device__ __forceinline__ void load(int row) {
        const uint32_t n = A.listed[row];
        whole = n > (uint32_t)kList;
#pragma unroll
        for (int i = 0; i < kListPer; ++i) {
            const uint32_t at = i * kPickThreads + threadIdx.x;
            near[i] = near_of<CAP>(A, R, C, !whole && at < n ? A.list[(int64_t)row * kList + at] : 0);
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) {
        if (!whole) {
#pragma unroll
            for (int i = 0; i < kListPer; ++i)
                if (near[i].k || near[i].p) f(near[i]);
        } else {
            for (int i = threadIdx.x; i < A.vocab; i += kPickThreads) {
                const Near e = near_at<CAP>(A, R, C, x, i);
                if (e.k || e.p) f(e);
            }
        }
    }

    // Among top-p's (by_p) or top-k's tokens with a key of at least `least`, in falling order: the one where the
    // running weight (by_p) or count first reaches `target`. Returns its key, and in *mass the weight up to
    // it. Each step splits the range of keys in 1024.
    __device__ __forceinline__ u64 refine(bool by_p, u64 least, u64 target, u64 *mass) {
        const int t = threadIdx.x;
        __syncthreads();
        if (t == 0) {
            S.high = 0;
            S.low = ~0ull;
        }
        __syncthreads();
        u64 hi = 0, lo = ~0ull;
        each([&](const Near &e) {
            if (!(by_p ? e.p : e.k) || e.key < least) return;
            hi = e.key > hi ? e.key : hi;
            lo = e.key < lo ? e.key : lo;
        });
        if (hi) {
            atomicMax(&S.high, hi);
            atomicMin(&S.low, lo);
        }
        __syncthreads();
        hi = S.high;
        lo = S.low;
        u64 mass_sum = 0;
        while (true) {
            const int bits = 64 - __clzll((long long)((hi - lo) | 1)), sh = bits > 10 ? bits - 10 : 0;
            S.mass[t] = 0;
            S.count[t] = 0;
            if (t == 0) S.at = kSub;
            __syncthreads();
            each([&](const Near &e) {
                if (!(by_p ? e.p : e.k) || e.key < lo || e.key > hi) return;
                atomicAdd(&S.mass[(hi - e.key) >> sh], e.w);
                atomicAdd(&S.count[(hi - e.key) >> sh], 1u);
                S.cut = e.key;  // the key, where it is the only one
            });
            __syncthreads();
            u64 all, m_all;
            const u64 m = S.mass[t], n = S.count[t];
            const u64 n_run = block_run<kPickThreads>(n, S.sums, &all);
            const u64 m_run = block_run<kPickThreads>(m, S.sums, &m_all);
            const u64 run = by_p ? m_run : n_run, one = by_p ? m : n;
            if (run - one < target && target <= run) {  // one thread, or none where nothing reaches it
                S.at = t;
                S.before = run - one;
                S.mass_before = m_run - m;
                S.mass_at = m;
                S.count_at = (uint32_t)n;
            }
            __syncthreads();
            const uint32_t at = S.at;
            if (at == kSub || all == 1) {
                *mass = mass_sum + m_all;
                return all == 1 ? S.cut : lo;
            }
            target -= S.before;
            mass_sum += S.mass_before;
            hi -= (u64)at << sh;
            const u64 width = (1ull << sh) - 1;
            lo = hi - lo > width ? hi - width : lo;
            if (sh == 0) {  // a range is one key
                *mass = mass_sum + S.mass_at;
                return hi;
            }
            __syncthreads();
        }
    }
};

// One block per row.
template <bool CAP>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleArgs A) {
    __shared__ PickShared S;
    const int t = threadIdx.x, row = blockIdx.x;
    const float *x = row_of(A, row);
    const Row R = row_params(A, row);
    if (R.index < 0) {
        if (t == 0) {
            A.tokens[row] = -1;
            if (A.logprobs) A.logprobs[row] = 0.0f;
        }
        return;
    }
    u64 sum = 0, all;
    for (int c = t; c < A.parts; c += kPickThreads) sum += A.part_sums[(int64_t)row * A.parts + c];
    block_run<kPickThreads>(sum, S.sums, &all);
    // log of the sum of all weights: steps back to weights
    const double log_all = log((double)all) - A.shift * 0.69314718055994530942;
    if (R.greedy) {
        if (t == 0) {
            A.tokens[row] = R.index;
            if (A.logprobs) A.logprobs[row] = (float)-log_all;
        }
        return;
    }
    for (int i = t; i < A.units; i += kPickThreads) S.extra[i] = 0;
    if (t == 0) {
        S.at = 0;
        S.before = 0;
    }
    __syncthreads();
    u64 cut = 0;  // the last kept key
    if (R.filtered) {
        const Cuts C = A.cut[row];
        if (C.p_low < kBins) {
            Search<CAP> L{A, R, C, x, S};
            L.load(row);
            u64 mass = all;
            if (C.k_bin < kBins) {
                cut = L.refine(false, 0, C.k_rest, &mass);
                mass += C.k_before;
            }
            if (R.p < 1.0) cut = L.refine(true, cut, mass_target(R.p, mass) - C.p_before, &mass);
            L.each([&](const Near &e) {
                if (e.key >= cut && e.d >= R.d_min) atomicAdd(&S.extra[~(uint32_t)e.key / kSampleUnit], e.w);
            });
            __syncthreads();
        }
    }
    // the unit, then the token, where the running sum passes u of the total
    const u64 *units = A.unit_sums + (int64_t)row * A.units;
    const int per = (A.units + kPickThreads - 1) / kPickThreads, u0 = min(t * per, A.units), u1 = min(u0 + per, A.units);
    u64 mine = 0, total;
    for (int i = u0; i < u1; ++i) mine += units[i] + S.extra[i];
    u64 run = block_run<kPickThreads>(mine, S.sums, &total) - mine;
    const float uf = fminf(fmaxf(A.u[row], 0.0f), 0x1.fffffep-1f);  // NaN: 0
    u64 target = (u64)((double)uf * (double)total);
    if (run <= target && target < run + mine) {
        for (int i = u0; i < u1; ++i) {
            const u64 w = units[i] + S.extra[i];
            if (target < run + w) {
                S.at = i;
                S.before = run;
                break;
            }
            run += w;
        }
    }
    __syncthreads();
    const int id = (int)S.at * kSampleUnit + t;
    target -= S.before;
    u64 w = 0;
    double d = 0.0;
    if (id < A.vocab) {
        const float v = seen(clean(x[id]), R);
        d = distance<CAP>(v, R, A);
        if (v > -INFINITY && d >= R.d_min && order_key(v, id) >= cut) w = steps(d, R, A);
    }
    run = block_run<kPickThreads>(w, S.sums, &total) - w;
    if (run <= target && target < run + w) {
        A.tokens[row] = id;
        if (A.logprobs) A.logprobs[row] = (float)(d * R.inv_t - log_all);
    }
}

template <bool CAP>
static int launch_sample(const SampleArgs &A, int rows, hipStream_t s) {
    const dim3 grid(A.parts, rows);
    hipLaunchKernelGGL(sample_max_kernel, grid, dim3(kSampleThreads), 0, s, A);
    G4_LAUNCHED("sample_max_kernel");
    hipLaunchKernelGGL(sample_weights_kernel<CAP>, grid, dim3(kSampleThreads), 0, s, A);
    G4_LAUNCHED("sample_weights_kernel");
    if (A.cuts) {
        hipLaunchKernelGGL(sample_cut_kernel<CAP>, grid, dim3(kSampleThreads), 0, s, A);
        G4_LAUNCHED("sample_cut_kernel");
    }
    hipLaunchKernelGGL(sample_pick_kernel<CAP>, dim3(rows), dim3(kPickThreads), 0, s, A);
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
    const size_t row = (size_t)sample_parts(vocab) * (sizeof(PartMax) + sizeof(u64)) + (size_t)sample_units(vocab) * sizeof(u64) +
                       kBins * (sizeof(u64) + sizeof(uint32_t)) + kList * sizeof(u64) + sizeof(Cuts) + sizeof(uint32_t);
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
    A.cap = {cap, cap > 0.0f ? 1.0 / ((double)cap * cap) : 0.0, 0.4999999f * cap};
    A.logit_rows = logit_rows;
    A.vocab = (int)vocab;
    A.parts = (int)sample_parts(vocab);
    A.units = (int)sample_units(vocab);
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    A.shift = 62 - bits < 51 ? 62 - bits : 51;
    A.vec = A.stride % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    A.cuts = top_k || top_p;
    A.stats = static_cast<PartMax *>(workspace);
    A.part_sums = reinterpret_cast<u64 *>(A.stats + (int64_t)rows * A.parts);
    A.unit_sums = A.part_sums + (int64_t)rows * A.parts;
    A.bin_mass = A.unit_sums + (int64_t)rows * A.units;
    A.list = A.bin_mass + (int64_t)rows * kBins;
    A.cut = reinterpret_cast<Cuts *>(A.list + (int64_t)rows * kList);
    A.bin_count = reinterpret_cast<uint32_t *>(A.cut + rows);
    A.listed = A.bin_count + (int64_t)rows * kBins;
    A.tokens = tokens;
    A.logprobs = logprobs;
    hipStream_t s = as_stream(stream);
    return cap > 0.0f ? launch_sample<true>(A, rows, s) : launch_sample<false>(A, rows, s);
}

}  // extern "C"
