// Causal attention of a chunk of new tokens over the paged cache (include/g4serve.h).
//
// Query rows are (token, query head of the group) pairs, 32 to a tile, tokens first, so that every head
// on one KV head shares its loads. Both products run on v_mfma_f32_32x32x16_f16 in the transposed order
//   S^T = K Q^T   (A: 32 keys, B: 32 query rows)       O^T += V^T P^T   (A: 32 dims, B: 32 query rows)
// whose result lane holds one query row (lane % 32) and 16 of the keys: a row's softmax is per-lane
// arithmetic and one exchange with lane ^ 32, and the weights are the second product's B operand where
// they stand. The order of the k index of a product is free as long as both operands agree on it; the
// layouts below use that twice:
//  - P: lane half h holds, for k-step t of 16 keys, keys 16 t + 4 h + 0..3 and 16 t + 8 + 4 h + 0..3;
//  - V: a lane loads DPL = D / 32 consecutive dims of each of these eight keys (a whole row per half
//    wave) and byte-permutes them into DPL operands of eight keys each, the row i of operand j being dim
//    DPL i + j. No LDS transposes anything.
// The softmax keeps a running maximum (base 2) and sum in f32; the maximum moves, and the output is
// rescaled, only when a score passes it by more than 2^8, so weights reach 2^8 at most and are rounded to
// f16 (11 bits; the sum adds them unrounded). int8 rows: codes are exact in f16; K's scale multiplies the
// score, V's the weight, taken relative to a power of two above the largest scale that the row has seen,
// which scales the row's output (f16 would not hold scales of every size).
#include "g4_paged.h"
#include <algorithm>
#include <cmath>

namespace g4 {

typedef float f16x __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct AttnArgs {
    const _Float16 *q;
    int64_t q_stride;
    int heads, group;
    float scale2;  // scale * log2(e): scores are kept in base 2
    int window;
    void *out;
    int out_kind;
    float in_scale;
    int splits;
    float *part_o;   // [tile][split][kv_head][32][D]
    float2 *part_ml; // [tile][split][kv_head][32]: maximum, sum
};

constexpr int kRows = 32, kKeys = 32;
constexpr float kLazy = 8.0f;

__device__ __forceinline__ float other_half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The next power of two above a scale (2^120 and more: 2^121).
__device__ __forceinline__ float pow2_above(float v) {
    return __uint_as_float((__float_as_uint(fminf(v, 0x1p120f)) & 0x7f800000u) + 0x00800000u);
}

__device__ __forceinline__ h2 bits_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ __forceinline__ uint32_t h2_bits(h2 x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ h8 words_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u32x4 w = {a, b, c, d};
    return __builtin_bit_cast(h8, w);
}

// Eight int8 codes (two words) as f16: code + 128 in the low bits of 1024.0, less 1152.
__device__ __forceinline__ h8 codes_h8(uint32_t a, uint32_t b) {
    const h2 bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t m = 0x64646464u;
    return words_h8(h2_bits(bits_h2(__builtin_amdgcn_perm(m, a, 0x04010400u)) + bias),
                    h2_bits(bits_h2(__builtin_amdgcn_perm(m, a, 0x04030402u)) + bias),
                    h2_bits(bits_h2(__builtin_amdgcn_perm(m, b, 0x04010400u)) + bias),
                    h2_bits(bits_h2(__builtin_amdgcn_perm(m, b, 0x04030402u)) + bias));
}

// Code j of words a and b as a pair of f16.
template <int J>
__device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t b) {
    const h2 bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t x = __builtin_amdgcn_perm(b, a, 0x0c000c00u | ((4 + J) << 16) | J) ^ 0x64806480u;
    return h2_bits(bits_h2(x) + bias);
}

// ---- which rows and keys ----------------------------------------------------------------------------

struct Tile {
    int seq, rows, first;  // rows: token rows x group of the sequence; first: this tile's first of them
    SeqSpan S;
    int lo, hi;  // keys [lo, hi) that some row of the tile may see; lo a multiple of kKeys
    bool live;
};

__device__ __forceinline__ int wave_scan_sum(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_up(v, s);
        if (lane >= s) v += o;
    }
    return v;
}

// Tile `id` of the batch: sequences in order, ceil(rows * group / per) tiles each.
__device__ __forceinline__ Tile find_tile(const PagedArgs &A, int group, int window, int id, int per) {
    const int lane = threadIdx.x & 63;
    Tile T{};
    for (int base = 0; base < A.seqs; base += 64) {
        int n = 0;
        SeqSpan S{0, 0, 0};
        if (base + lane < A.seqs) {
            S = seq_span(A, base + lane);
            n = (min(S.rows, A.max_q) * group + per - 1) / per;
        }
        const int end = wave_scan_sum(n);
        const unsigned long long past = __ballot(end > id);
        if (past) {
            const int at = __ffsll((long long)past) - 1;
            T.seq = base + at;
            T.S.start = __builtin_amdgcn_readlane(S.start, at);
            T.S.rows = __builtin_amdgcn_readlane(S.rows, at);
            T.S.kv = __builtin_amdgcn_readlane(S.kv, at);
            T.rows = min(T.S.rows, A.max_q) * group;
            T.first = (id - (__builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(n, at))) * per;
            const int p0 = T.S.kv - T.S.rows + T.first / group;
            const int p1 = T.S.kv - T.S.rows + (min(T.first + per, T.rows) - 1) / group;
            T.lo = window ? max(0, p0 - window + 1) & ~(kKeys - 1) : 0;
            T.hi = max(p1 + 1, 0);
            T.live = true;
            return T;
        }
        id -= __builtin_amdgcn_readlane(end, 63);
    }
    return T;
}

// Key tiles of one split: `n` key tiles cut in runs of `per`, a multiple of `unit`.
__device__ __forceinline__ int split_tiles(const Tile &T, int splits, int unit) {
    const int n = (T.hi - T.lo + kKeys - 1) / kKeys;
    return max((n + splits - 1) / splits + unit - 1, unit) / unit * unit;
}

__device__ __forceinline__ void attn_put8(const AttnArgs &R, int64_t at, const float (&y)[8]) {
    if (R.out_kind == G4_KIND_F16) {
        h8 o;
#pragma unroll
        for (int n = 0; n < 8; ++n) o[n] = (_Float16)y[n];
        *reinterpret_cast<h8 *>(static_cast<_Float16 *>(R.out) + at) = o;
    } else if (R.out_kind == G4_KIND_I8) {
        uint2 o{0, 0};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            o.x |= (uint32_t)(srq_code_i(y[n], R.in_scale) & 255) << (8 * n);
            o.y |= (uint32_t)(srq_code_i(y[n + 4], R.in_scale) & 255) << (8 * n);
        }
        *reinterpret_cast<uint2 *>(static_cast<int8_t *>(R.out) + at) = o;
    } else {
        float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(R.out) + at);
        o[0] = make_float4(y[0], y[1], y[2], y[3]);
        o[1] = make_float4(y[4], y[5], y[6], y[7]);
    }
}

// ---- few rows: the waves of a block split the keys -----------------------------------------------------

constexpr int kWaves = 4;

template <int BYTES> struct Words { uint32_t w[BYTES / 4]; };
template <> struct Words<2> { uint32_t w[1]; };

// BYTES bytes from base + off.
template <int BYTES>
__device__ __forceinline__ Words<BYTES> load_words(const char *base, uint32_t off) {
    Words<BYTES> r;
    const char *p = base + off;
    if constexpr (BYTES == 16) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else if constexpr (BYTES == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    } else if constexpr (BYTES == 4) {
        r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
        r.w[0] = *reinterpret_cast<const uint16_t *>(p);
    }
    return r;
}

// The DPL operands (8 keys each, one per consecutive dim) of eight keys' words.
template <int D, int CK, int J, int NB>
__device__ __forceinline__ h8 v_operand(const Words<NB> (&x)[8]) {
    uint32_t o[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        if constexpr (CK == G4_KIND_I8)
            o[p] = code_pair<J % 4>(x[2 * p].w[J / 4], x[2 * p + 1].w[J / 4]);
        else
            o[p] = __builtin_amdgcn_perm(x[2 * p + 1].w[J / 2], x[2 * p].w[J / 2], J % 2 ? 0x07060302u : 0x05040100u);
    }
    return words_h8(o[0], o[1], o[2], o[3]);
}

// The halves of a word that are NaN or infinite as f16, as a mask; and 1 in their place, 0 elsewhere.
__device__ __forceinline__ uint32_t odd_mask(uint32_t x) {
    return ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}
__device__ __forceinline__ h8 odd_ones(h8 x) {
    const u32x4 w = __builtin_bit_cast(u32x4, x);
    return words_h8(odd_mask(w.x) & 0x3c003c00u, odd_mask(w.y) & 0x3c003c00u, odd_mask(w.z) & 0x3c003c00u,
                    odd_mask(w.w) & 0x3c003c00u);
}

template <int J, int N, typename F>
__device__ __forceinline__ void each(F f) {
    if constexpr (J < N) {
        f(std::integral_constant<int, J>{});
        each<J + 1, N>(f);
    }
}

// Grid (tiles, splits, KV heads), 4 waves: wave w takes key tiles w, w + 4, ... of the split's run. K
// arrives as the A operand itself (a lane's own key, 16 bytes at a time), V as described above, both a
// tile ahead of their use as registers allow.
template <int D, int CK>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void attn_rows_kernel(PagedArgs A, AttnArgs R) {
    constexpr int KS = D / 16, DPL = D / 32;
    constexpr int EB = CK == G4_KIND_I8 ? 1 : 2;          // bytes per element
    constexpr int KL = D * EB / 32;                       // 16-byte K loads of a lane
    constexpr int VB = DPL * EB;                          // bytes of a V load
    __shared__ __align__(16) float sc_lds[kWaves][2][kKeys];
    __shared__ float2 ml_lds[kWaves][kRows];
    __shared__ float o_lds[kWaves][DPL * 16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = lane >> 5, c = lane & 31;
    const int kvh = blockIdx.z;
    const Tile T = find_tile(A, R.group, R.window, blockIdx.x, kRows);
    if (!T.live) return;
    const int per = split_tiles(T, R.splits, kWaves);
    const int k0 = T.lo + blockIdx.y * per * kKeys, k1 = min(T.hi, k0 + per * kKeys);
    if (blockIdx.y && k0 >= T.hi) return;

    // this lane's query row
    const int row = T.first + c;
    const bool real = row < T.rows;
    const int token = real ? row / R.group : 0, head = kvh * R.group + (real ? row % R.group : 0);
    const int pos = real ? T.S.kv - T.S.rows + token : -1;
    const int p_first = T.S.kv - T.S.rows + T.first / R.group;  // the tile's first row
    const int p_last = T.hi - 1;
    h8 q[KS];
    {
        const _Float16 *src = R.q + (int64_t)(T.S.start + token) * R.q_stride + (int64_t)head * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            // the k-step's 8 dims of this half, in the order that K's loads give them
            const int at = CK == G4_KIND_I8 ? 32 * (s / 2) + 16 * h + 8 * (s % 2) : 16 * s + 8 * h;
            q[s] = *reinterpret_cast<const h8 *>(src + at);
            if (!real) q[s] = h8{};
        }
    }

    f16x o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = f16x{};
    float m = -INFINITY, l = 0.0f, vref = 0x1p-100f;  // vref: the power of two of the row's V scales

    const int step = kWaves * kKeys;
    int t0 = k0 + wave * kKeys;
    auto key_pos = [&](int t) { return max(min(t + c, T.S.kv - 1), 0); };
    auto raw_page = [&](int t) { return A.table[T.seq * A.table_stride + (key_pos(t) >> A.page_shift)]; };
    u32x4 k[KL];
    float ks = 1.0f, vs = 1.0f;
    int page = 0, next_page = 0;
    const int smask = (1 << A.page_shift) - 1;
    auto load_k = [&](int t, int pg) {  // this lane's key of tile t (any row of the pool where it is absent)
        const int p = key_pos(t);
        const int64_t at = (int64_t)((unsigned)pg < (unsigned)A.num_pages ? pg : 0) * A.page_stride +
                           (int64_t)(p & smask) * A.slot_stride + (int64_t)kvh * A.head_stride;
        const char *src = static_cast<const char *>(A.k) + at * EB + 16 * h;
#pragma unroll
        for (int i = 0; i < KL; ++i) k[i] = *reinterpret_cast<const u32x4 *>(src + 32 * i);
        if (CK == G4_KIND_I8) {
            const int64_t sa = scale_offset(A, (unsigned)pg < (unsigned)A.num_pages ? pg : 0, p, kvh);
            ks = A.ks[sa];
            vs = A.vs[sa];
        }
    };
    if (t0 < k1) {
        page = raw_page(t0);
        load_k(t0, page);
        if (t0 + step < k1) next_page = raw_page(t0 + step);
    }
    for (; t0 < k1; t0 += step) {
        // keys of the tile that exist
        const bool there = t0 + c < T.S.kv && (unsigned)page < (unsigned)A.num_pages;
        const uint32_t keys = (uint32_t)__ballot(there);
        Words<VB> v[2][8];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int pg = __builtin_amdgcn_readlane(page, 8 * g);
            const int p0 = max(min(t0 + 8 * g, T.S.kv - 1), 0) & ~7;
            const int64_t at = (int64_t)((unsigned)pg < (unsigned)A.num_pages ? pg : 0) * A.page_stride +
                               (int64_t)(p0 & smask) * A.slot_stride + (int64_t)kvh * A.head_stride;
            const char *base = static_cast<const char *>(A.v) + at * EB;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[g / 2][(g % 2) * 4 + i] = load_words<VB>(base, (uint32_t)((4 * h + i) * A.slot_stride * EB) + c * VB);
        }
        f4 kss[4], vss[4];
        if (CK == G4_KIND_I8) {
            if (lane < kKeys) {
                sc_lds[wave][0][c] = ks * R.scale2;
                sc_lds[wave][1][c] = vs;
            }
        }
        f16x sacc = {};
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            if constexpr (CK == G4_KIND_I8) {
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_h8(k[i].x, k[i].y), q[2 * i], sacc, 0, 0, 0);
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_h8(k[i].z, k[i].w), q[2 * i + 1], sacc, 0, 0, 0);
            } else {
                sacc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, k[i]), q[i], sacc, 0, 0, 0);
            }
        }
        if (CK == G4_KIND_I8) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                kss[g] = *reinterpret_cast<const f4 *>(&sc_lds[wave][0][8 * g + 4 * h]);
                vss[g] = *reinterpret_cast<const f4 *>(&sc_lds[wave][1][8 * g + 4 * h]);
            }
        }
        if (t0 + step < k1) {
            page = next_page;
            load_k(t0 + step, page);
            if (t0 + 2 * step < k1) next_page = raw_page(t0 + 2 * step);
        }
        float x[16];
        const bool edge = t0 + kKeys - 1 > p_first || (R.window && t0 <= p_last - R.window);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = sacc[r] * (CK == G4_KIND_I8 ? kss[r / 4][r % 4] : R.scale2);
        uint32_t seen = 0xffff;  // bit r: this row sees the key of register r
        if (edge || keys != 0xffffffffu) {
            seen = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int kk = 8 * (r / 4) + 4 * h + r % 4, j = t0 + kk;
                const bool ok = (keys >> kk & 1) && j <= pos && (!R.window || j > pos - R.window);
                seen |= (uint32_t)ok << r;
                x[r] = ok ? x[r] : -INFINITY;
            }
        }
        float top = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
        top = other_half_max(top);
        if (__any(top > m + kLazy || (m == -INFINITY && top > -INFINITY))) {
            const float mn = fmaxf(m, top);
            const float a = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= a;
#pragma unroll
            for (int j = 0; j < DPL; ++j) o[j] *= a;
            m = mn;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        float vinv = 1.0f;
        if (CK == G4_KIND_I8) {
            // the largest finite scale that the row sees
            float vtop = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float a = fabsf(vss[r / 4][r % 4]);
                vtop = fmaxf(vtop, (seen >> r & 1) && a < INFINITY ? a : 0.0f);
            }
            vtop = other_half_max(vtop);
            if (__any(vtop > vref)) {
                const float to = fmaxf(vref, pow2_above(vtop)), f = vref / to;
                vref = to;
#pragma unroll
                for (int j = 0; j < DPL; ++j) o[j] *= f;
            }
            vinv = 1.0f / vref;
        }
        h8 p[2];
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(x[r] - mu);
            sum += e;
            float w = e;
            if (CK == G4_KIND_I8) {
                w = e * (vss[r / 4][r % 4] * vinv);
                if (!(seen >> r & 1)) w = 0.0f;  // a masked scale may be anything
            }
            p[r / 8][r % 8] = (_Float16)w;
        }
        l += sum;
        if (CK == G4_KIND_F16 && (edge || keys != 0xffffffffu)) {
            // absent keys hold anything: their V counts as zero. A NaN or an infinity at a key that some rows
            // see and others do not is kept out of the product and put into the rows that see it.
            uint32_t odd = 0;
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kk = 8 * g + 4 * h + i;
                    const bool ok = keys >> kk & 1;
                    Words<VB> &y = v[g / 2][(g % 2) * 4 + i];
#pragma unroll
                    for (int n = 0; n < (VB + 3) / 4; ++n) {
                        y.w[n] = ok ? y.w[n] : 0u;
                        odd |= odd_mask(y.w[n]);
                    }
                }
            if (__any(odd)) {
                h8 one[2];
#pragma unroll
                for (int r = 0; r < 16; ++r) one[r / 8][r % 8] = (seen >> r & 1) ? (_Float16)1.0f : (_Float16)0.0f;
                each<0, DPL>([&](auto J) {
                    f16x n = {};
                    n = __builtin_amdgcn_mfma_f32_32x32x16_f16(odd_ones(v_operand<D, CK, J.value>(v[0])), one[0], n, 0, 0, 0);
                    n = __builtin_amdgcn_mfma_f32_32x32x16_f16(odd_ones(v_operand<D, CK, J.value>(v[1])), one[1], n, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (n[r] > 0.0f) o[J.value][r] = __builtin_nanf("");
                });
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int n = 0; n < (VB + 3) / 4; ++n) v[s][i].w[n] &= ~odd_mask(v[s][i].w[n]);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
            each<0, DPL>([&](auto J) {
                o[J.value] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_operand<D, CK, J.value>(v[s]), p[s], o[J.value], 0, 0, 0);
            });
    }
    l = other_half_sum(l);

    // the four waves' parts: relative to the block's maximum, then each wave adds a quarter of the dims
    if (h == 0) ml_lds[wave][c] = make_float2(m, l);
    __syncthreads();
    float top = ml_lds[0][c].x;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml_lds[w][c].x);
    const float mu = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += ml_lds[w][c].y * __builtin_amdgcn_exp2f(ml_lds[w][c].x - mu);
    const float f = __builtin_amdgcn_exp2f(m - mu) * (CK == G4_KIND_I8 ? vref : 1.0f);
#pragma unroll
    for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_lds[wave][j * 16 + r][lane] = o[j][r] * f;
    __syncthreads();
    if (!real) return;
    const bool whole = R.splits == 1;
    const float inv = whole ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f;
    const int64_t slot = (((int64_t)blockIdx.x * R.splits + blockIdx.y) * A.kv_heads + kvh) * kRows + c;
    // register r = 4 wave + i of every operand j: dims DPL (8 wave + 4 h + i) + j, consecutive over i and j
    float y[4 * DPL];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < DPL; ++j) {
            float a = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a += o_lds[w][j * 16 + 4 * wave + i][lane];
            y[i * DPL + j] = a * inv;
        }
    const int d0 = DPL * (8 * wave + 4 * h);
#pragma unroll
    for (int b = 0; b < 4 * DPL; b += 8) {
        const float z[8] = {y[b], y[b + 1], y[b + 2], y[b + 3], y[b + 4], y[b + 5], y[b + 6], y[b + 7]};
        if (whole) {
            attn_put8(R, ((int64_t)(T.S.start + token) * R.heads + head) * D + d0 + b, z);
        } else {
            float4 *dst = reinterpret_cast<float4 *>(R.part_o + slot * D + d0 + b);
            dst[0] = make_float4(z[0], z[1], z[2], z[3]);
            dst[1] = make_float4(z[4], z[5], z[6], z[7]);
        }
    }
    if (!whole && wave == 0 && h == 0) R.part_ml[slot] = make_float2(top, total);
}

// ---- the parts of a split row joined -----------------------------------------------------------------

// Grid (tiles, KV heads, 32 / rows of a block): a thread sums 8 dims of one row over the splits, in order.
template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(PagedArgs A, AttnArgs R, int unit) {
    constexpr int TR = D / 8, RB = 256 / TR;  // threads of a row, rows of a block
    const int t = threadIdx.x, c = blockIdx.z * RB + t / TR, d = (t % TR) * 8, kvh = blockIdx.y;
    const Tile T = find_tile(A, R.group, R.window, blockIdx.x, kRows);
    if (!T.live) return;
    const int row = T.first + c;
    if (c >= kRows || row >= T.rows) return;
    const int per = split_tiles(T, R.splits, unit);
    const int n = max(1, ((T.hi - T.lo + kKeys - 1) / kKeys + per - 1) / per);
    const int64_t stride = (int64_t)A.kv_heads * kRows;
    const int64_t slot = ((int64_t)blockIdx.x * R.splits * A.kv_heads + kvh) * kRows + c;
    float top = -INFINITY;
    for (int s = 0; s < n; ++s) top = fmaxf(top, R.part_ml[slot + s * stride].x);
    const float mu = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, y[8] = {};
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const float2 ml = R.part_ml[slot + s * stride];
        const float4 *src = reinterpret_cast<const float4 *>(R.part_o + (slot + s * stride) * D + d);
        const float4 a = src[0], b = src[1];
        const float f = __builtin_amdgcn_exp2f(ml.x - mu);
        total += ml.y * f;
        y[0] += a.x * f; y[1] += a.y * f; y[2] += a.z * f; y[3] += a.w * f;
        y[4] += b.x * f; y[5] += b.y * f; y[6] += b.z * f; y[7] += b.w * f;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= inv;
    const int token = row / R.group, head = kvh * R.group + row % R.group;
    attn_put8(R, ((int64_t)(T.S.start + token) * R.heads + head) * D + d, y);
}

// ---- host ---------------------------------------------------------------------------------------------

struct AttnPlan {
    int64_t tiles;  // upper bound over the batch
    int splits;
    size_t bytes;
};

// Enough splits for two blocks a CU (one block leaves a CU idle while it joins its waves), no split
// under one round of the block's waves.
static AttnPlan attn_plan(const PagedArgs &A, int head_dim, int heads, int window) {
    const int group = heads / A.kv_heads;
    AttnPlan P;
    const int64_t per_seq = ((int64_t)A.max_q * group + kRows - 1) / kRows;
    P.tiles = std::min(per_seq * A.seqs, (int64_t)A.tokens * group / kRows + A.seqs);
    int64_t keys = A.max_kv;
    if (window) keys = std::min<int64_t>(keys, (int64_t)window + kKeys + kRows / group + 1);
    const int64_t rounds = (keys + kWaves * kKeys - 1) / (kWaves * kKeys);
    const int64_t want = 2 * (int64_t)device_cu_count();
    const int64_t blocks = P.tiles * A.kv_heads;
    P.splits = (int)std::max<int64_t>(1, std::min<int64_t>({rounds, (want + blocks - 1) / blocks, 64}));
    const int64_t slots = P.tiles * P.splits * A.kv_heads * kRows;
    P.bytes = P.splits == 1 ? 16 : (size_t)slots * (head_dim * sizeof(float) + sizeof(float2));
    return P;
}

template <int D>
static int launch_attn(const PagedArgs &A, const AttnArgs &R, const AttnPlan &P, int ck, hipStream_t stream) {
    const dim3 grid((unsigned)P.tiles, P.splits, A.kv_heads);
    if (ck == G4_KIND_F16)
        hipLaunchKernelGGL((attn_rows_kernel<D, G4_KIND_F16>), grid, dim3(64 * kWaves), 0, stream, A, R);
    else
        hipLaunchKernelGGL((attn_rows_kernel<D, G4_KIND_I8>), grid, dim3(64 * kWaves), 0, stream, A, R);
    G4_LAUNCHED("attn_rows_kernel");
    if (P.splits > 1) {
        constexpr int rb = 256 / (D / 8);
        hipLaunchKernelGGL(attn_join_kernel<D>, dim3((unsigned)P.tiles, A.kv_heads, (kRows + rb - 1) / rb), dim3(256), 0,
                           stream, A, R, kWaves);
        G4_LAUNCHED("attn_join_kernel");
    }
    return G4_OK;
}

static int attn_check(const g4_kv_pages *pages, const g4_chunk *chunk, int heads, int window, PagedArgs *A) {
    if (int st = paged_args("attention-chunk", pages, chunk, A)) return st;
    if (heads <= 0 || heads % A->kv_heads)
        return set_error(G4_ERR_INVALID, "attention-chunk: %d query heads do not divide over %d KV heads", heads, A->kv_heads);
    if (window < 0) return set_error(G4_ERR_INVALID, "attention-chunk: window %d", window);
    if ((int64_t)A->tokens * heads > ((int64_t)1 << 30) || A->kv_heads > 65535)
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: more than 2^30 query rows, or 65535 KV heads");
    if (A->slot_stride > ((int64_t)1 << 27))
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: slots more than 2^27 elements apart");
    return G4_OK;
}

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_attention_chunk_workspace_bytes(const g4_kv_pages *pages, const g4_chunk *chunk, int heads,
                                          int window) {
    PagedArgs A;
    if (attn_check(pages, chunk, heads, window, &A)) return 0;
    return attn_plan(A, pages->head_dim, heads, window).bytes;
}

int g4_attention_chunk(const g4_kv_pages *pages, const g4_chunk *chunk, const void *q, int64_t q_stride,
                       int heads, float scale, int window, void *workspace, size_t workspace_bytes,
                       void *out, int out_kind, float in_scale, void *stream) {
    PagedArgs A;
    if (int st = attn_check(pages, chunk, heads, window, &A)) return st;
    if (!q || !out || !workspace) return set_error(G4_ERR_INVALID, "attention-chunk needs q, an output and a workspace");
    if (out_kind != G4_KIND_F16 && out_kind != G4_KIND_F32 && out_kind != G4_KIND_I8)
        return set_error(G4_ERR_INVALID, "attention-chunk: outputs are f16, f32 or int8 codes, got kind %d", out_kind);
    if (out_kind == G4_KIND_I8 && in_scale == 0.0f)
        return set_error(G4_ERR_INVALID, "attention-chunk: int8 codes need the consumer's inScale");
    const int64_t qw = (int64_t)heads * pages->head_dim;
    if (q_stride && (q_stride < qw || q_stride % 8))
        return set_error(G4_ERR_INVALID, "attention-chunk: q_stride must hold a row and be a multiple of 8");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return set_error(G4_ERR_INVALID, "attention-chunk: q, the output and the workspace must be 16-byte aligned");
    const AttnPlan P = attn_plan(A, pages->head_dim, heads, window);
    if (workspace_bytes < P.bytes)
        return set_error(G4_ERR_INVALID, "attention-chunk: workspace %zu B < %zu B", workspace_bytes, P.bytes);
    float *part_o = static_cast<float *>(workspace);
    const AttnArgs R{static_cast<const _Float16 *>(q), q_stride ? q_stride : qw, heads, heads / A.kv_heads,
                     scale * 1.44269504088896340736f, window, out, out_kind, in_scale, P.splits, part_o,
                     reinterpret_cast<float2 *>(part_o + P.tiles * P.splits * A.kv_heads * kRows * pages->head_dim)};
    if (pages->head_dim == 64) return launch_attn<64>(A, R, P, pages->kind, as_stream(stream));
    if (pages->head_dim == 128) return launch_attn<128>(A, R, P, pages->kind, as_stream(stream));
    return launch_attn<256>(A, R, P, pages->kind, as_stream(stream));
}

}  // extern "C"
