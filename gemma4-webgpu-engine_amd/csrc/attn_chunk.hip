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
// f16 (11 bits; an f16 cache's sum adds the rounded ones, an int8 cache's the exact ones, whose weights
// are rounded with V's scale in them). int8 rows: codes are exact in f16; K's scale multiplies the
// score, V's the weight, taken relative to a power of two above the largest scale that the row has seen,
// which scales the row's output and sum (f16 would not hold scales of every size) and enters the weights
// by their exponent.
#include "g4_paged.h"
#include <algorithm>
#include <cmath>

namespace g4 {

typedef float f16x __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

// Division of n < 2^31 by a constant of the call, d > 1: (n * mul) >> (31 + log), log = ceil(log2 d) and
// mul = floor(2^(31 + log) / d) + 1, which is under 2^32 and whose excess over 2^(31 + log) / d is at most
// 1 <= 2^log / d, too little to carry n / d over a whole number. By the high word of the product, which the
// scalar unit has too (a 64-bit product would move uniform values to the vector unit).
struct FastDiv {
    uint32_t d, mul;
    int shift;
    static FastDiv of(int d) {
        int log = 0;
        while ((1ll << log) < d) ++log;
        return {(uint32_t)d, (uint32_t)(((uint64_t)1 << (31 + log)) / d + 1), log - 1};
    }
    __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
    __device__ __forceinline__ int mod(int n) const { return n - div(n) * (int)d; }
};

struct AttnArgs {
    const _Float16 *q;
    int64_t q_stride;
    int heads;
    FastDiv group;
    // Scores are kept as the products give them; the base-2 exponent is score * scale2, scale2 > 0. A
    // negative scale turns Q's signs over; lazy is kLazy / scale2.
    float scale2, lazy;
    uint32_t q_sign;  // 0x80008000: Q is turned over
    uint32_t page_bytes, slot_bytes;
    int window;
    void *out;
    int out_kind;
    float in_scale;
    FastDiv splits;
    float *part_o;    // [tile][split][kv_head][row of the tile][D]
    float2 *part_ml;  // [tile][split][kv_head][row of the tile]: maximum, sum
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

// The next power of two above a scale (2^99 and more: 2^100), and a power of two's exponent.
__device__ __forceinline__ float pow2_above(float v) {
    return __uint_as_float((__float_as_uint(fminf(v, 0x1p99f)) & 0x7f800000u) + 0x00800000u);
}
__device__ __forceinline__ float pow2_log(float v) { return (float)((int)(__float_as_uint(v) >> 23) - 127); }

// The maximum over lanes 0..31, with lanes 32..63 holding the same values.
__device__ __forceinline__ float half_max(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));   // lane ^ 1
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));   // ^ 2
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false)));  // 7 -
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false)));  // 15 -
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ h2 bits_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ __forceinline__ uint32_t h2_bits(h2 x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ h8 words_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u32x4 w = {a, b, c, d};
    return __builtin_bit_cast(h8, w);
}

// An int8 code as f16 without arithmetic: the byte code + 128 zero-extended is the subnormal
// (code + 128) 2^-24, exact, and the matrix products keep subnormals. The 128s come off outside: from the
// scores as the accumulator's start, -128 2^-24 sum(q), and from the output by the sum of the rounded
// weights. (Products of at most 2^8 2^8 codes' bits: f32 sums of them lose about what sums of the codes
// alone would, the bias being three times a typical code.)
// Eight codes, two words:
__device__ __forceinline__ h8 codes_h8(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    return words_h8(__builtin_amdgcn_perm(0u, a, 0x0c010c00u), __builtin_amdgcn_perm(0u, a, 0x0c030c02u),
                    __builtin_amdgcn_perm(0u, b, 0x0c010c00u), __builtin_amdgcn_perm(0u, b, 0x0c030c02u));
}
// Element j of words a and b as a pair; the codes' signs are flipped already.
template <int J>
__device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, 0x0c000c00u | ((4 + J) << 16) | J);
}
template <int J, int N>
__device__ __forceinline__ uint32_t half_pair(const uint32_t (&a)[N], const uint32_t (&b)[N]) {
    return __builtin_amdgcn_perm(b[J / 2], a[J / 2], J % 2 ? 0x07060302u : 0x05040100u);
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
__device__ __forceinline__ Tile find_tile(const PagedArgs &A, const FastDiv &group, int window, int id, int per) {
    const int lane = threadIdx.x & 63;
    Tile T{};
    for (int base = 0; base < A.seqs; base += 64) {
        int n = 0;
        SeqSpan S{0, 0, 0};
        if (base + lane < A.seqs) {
            S = seq_span(A, base + lane);
            n = (min(S.rows, A.max_q) * (int)group.d + per - 1) / per;
        }
        const int end = wave_scan_sum(n);
        const unsigned long long past = __ballot(end > id);
        if (past) {
            const int at = __ffsll((long long)past) - 1;
            T.seq = base + at;
            T.S.start = __builtin_amdgcn_readlane(S.start, at);
            T.S.rows = __builtin_amdgcn_readlane(S.rows, at);
            T.S.kv = __builtin_amdgcn_readlane(S.kv, at);
            T.rows = min(T.S.rows, A.max_q) * (int)group.d;
            T.first = (id - (__builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(n, at))) * per;
            const int p0 = T.S.kv - T.S.rows + group.div(T.first);
            const int p1 = T.S.kv - T.S.rows + group.div(min(T.first + per, T.rows) - 1);
            T.lo = window ? max(0, p0 - window + 1) & ~(kKeys - 1) : 0;
            T.hi = max(p1 + 1, 0);
            T.live = true;
            return T;
        }
        id -= __builtin_amdgcn_readlane(end, 63);
    }
    return T;
}

// Key tiles of one split: `n` key tiles cut in runs of `per`, a multiple of `unit` (a power of two).
__device__ __forceinline__ int split_tiles(const Tile &T, const FastDiv &splits, int unit) {
    const int n = (unsigned)(T.hi - T.lo + kKeys - 1) / kKeys;
    return max(splits.div(n + (int)splits.d - 1) + unit - 1, unit) & ~(unit - 1);
}

__device__ __forceinline__ void attn_put4(const AttnArgs &R, int64_t at, float4 y) {
    if (R.out_kind == G4_KIND_F16) {
        const h4 o = {(_Float16)y.x, (_Float16)y.y, (_Float16)y.z, (_Float16)y.w};
        *reinterpret_cast<h4 *>(static_cast<_Float16 *>(R.out) + at) = o;
    } else if (R.out_kind == G4_KIND_I8) {
        const float s = R.in_scale;
        *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(R.out) + at) =
            (srq_code_i(y.x, s) & 255) | (srq_code_i(y.y, s) & 255) << 8 | (srq_code_i(y.z, s) & 255) << 16 |
            (uint32_t)(srq_code_i(y.w, s) & 255) << 24;
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(R.out) + at) = y;
    }
}

// ---- the attention kernel -------------------------------------------------------------------------------

// The block's shape: RT row tiles (32 query rows each) x KG key groups, a wave each. Key group g takes the
// key tiles g, g + KG, ... of the block's run; the waves of a group share its K and V tiles, which come
// straight to LDS as the rows stand in the cache, a ring of NS tiles each.
//  RT 1: a wave waits for its own loads only, and refills the K half of its buffer as soon as the scores
//        are done and the V half after the output (NS 1);
//  RT 2, 4: one block barrier per key tile, NS tiles in flight.
template <int D, int CK, int RT>
struct Shape {
    static constexpr int EB = CK == G4_KIND_I8 ? 1 : 2;  // bytes of an element
    static constexpr int RB = D * EB;                    // of a row
    static constexpr int HALF = kKeys * RB;              // of a tile's K or V
    static constexpr int KG = RT == 1 ? 4 : (RT == 2 && RB < 512 ? 4 : 2);
    static constexpr int NS = RT == 1 ? 1 : 2;
    static constexpr int WAVES = RT * KG;
    static constexpr int RING = KG * NS * 2 * HALF;
    // int8: the scales of a wave's tiles, ks[32] and vs[32] a tile, and one more tile ahead
    static constexpr int SCALES = CK == G4_KIND_I8 ? WAVES * 2 * 256 : 0;
    static constexpr int JOIN = WAVES * (D / 8) * 72 * 4;  // a quarter of every wave's output (see the end)
    // Q's last operands wait in LDS where two waves a SIMD share the registers: output and Q alone take 192 of 256
    static constexpr int QL = D != 256 ? 0 : (WAVES == 8 ? 3 : (RT == 1 && CK == G4_KIND_I8 ? 3 : 0));
    static constexpr bool TIGHT = D == 256 && CK == G4_KIND_F16 && WAVES == 8;  // no registers for V's reads ahead
    static constexpr int LDS = (RING > JOIN ? RING : JOIN) + SCALES + WAVES * (kRows * 8 + QL * 1024);
    static constexpr int MIN_WAVES = WAVES == 4 && LDS > 80 * 1024 ? 1 : 2;  // per SIMD: one block a CU, or two
};

// Byte of chunk x (16 bytes) of K row c of a tile: the chunk index is XORed so that a b128 read of one
// chunk index over 8 consecutive rows hits 8 different bank groups.
template <int RB>
__device__ __forceinline__ int k_swizzle(int c) {
    return RB >= 128 ? c & 7 : (c >> 2) & 1;
}

// 16 (4) bytes per active lane from base + off to LDS at lds + 16 (4) * lane; see the waits in the kernel.
__device__ __forceinline__ void dma16(const char *base, uint32_t off, uint32_t lds) {
    // readfirstlane gives an int: its words are unsigned before they are put together
    const uint32_t b0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base);
    const uint32_t b1 = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)base >> 32));
    const uint64_t b = (uint64_t)b1 << 32 | b0;
    // 5 wait states: a scalar register that the vector unit wrote (readfirstlane), read as a base address
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(b) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// The halves of a word that are NaN or infinite as f16, as a mask.
__device__ __forceinline__ uint32_t odd_mask(uint32_t x) {
    return ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}
template <int J, int N, typename F>
__device__ __forceinline__ void each(F f) {
    if constexpr (J < N) {
        f(std::integral_constant<int, J>{});
        each<J + 1, N>(f);
    }
}

// Dims of a lane's V operands: UD consecutive ones (4; 2 at head_dim 64) in each of D / (32 UD) blocks of
// 32 UD dims, so that a half wave reads 32 UD consecutive elements of a row. Operand j = UD u + w is dims
// 32 UD u + UD i + w over its rows i.
template <int D> struct VDims {
    static constexpr int UD = D == 64 ? 2 : 4, U = D / (32 * UD);
};

// The pages of a key tile's four 8-key groups, below 0 where absent. Named, not an array: an array is
// indexed in memory, which makes its values per-lane ones.
struct Pages {
    int a, b, c, d;
    __device__ __forceinline__ int of(int g) const {
        const int lo = g & 1 ? b : a, hi = g & 1 ? d : c;
        return g & 2 ? hi : lo;
    }
};

typedef const __attribute__((address_space(4))) int32_t *ConstI32;  // uniform reads by the scalar unit

template <int D, int CK, int RT>
__global__ __launch_bounds__((64 * Shape<D, CK, RT>::WAVES), (Shape<D, CK, RT>::MIN_WAVES))
void attn_kernel(PagedArgs A, AttnArgs R) {
    using P = Shape<D, CK, RT>;
    constexpr bool I8 = CK == G4_KIND_I8;
    constexpr int EB = P::EB, RB = P::RB, KG = P::KG, NS = P::NS, KS = D / 16, DPL = D / 32;
    constexpr int UD = VDims<D>::UD, U = VDims<D>::U, VB = UD * EB;   // VB: bytes of a lane's read of a V row
    constexpr int GB = 8 * RB;                                        // bytes of an 8-key group
    constexpr int NI = GB >= 1024 ? GB / 1024 : 1;                    // loads of a group
    constexpr int LPR = RB / 16;                                      // lanes of a row
    constexpr int GW = 4 / RT;                                        // groups that a wave loads
    constexpr int LOADS = GW * NI;                                    // loads of a wave for a tile's K (or V)
    __shared__ __align__(1024) char lds[P::LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rt = wave % RT, kg = wave / RT;
    const int h = lane >> 5, c = lane & 31;
    const int kvh = blockIdx.z;
    const Tile T = find_tile(A, R.group, R.window, blockIdx.x, kRows * RT);
    if (!T.live) return;
    const int per = split_tiles(T, R.splits, KG);
    const int k0 = T.lo + blockIdx.y * per * kKeys, k1 = min(T.hi, k0 + per * kKeys);
    if (blockIdx.y && k0 >= T.hi) return;
    const int rounds = (k1 - k0 + KG * kKeys - 1) / (KG * kKeys);  // 0 where there are no keys

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    constexpr int SC0 = P::RING > P::JOIN ? P::RING : P::JOIN, ML0 = SC0 + P::SCALES, Q0 = ML0 + P::WAVES * kRows * 8;
    char *const scales = lds + SC0 + wave * 512;
    float2 *const ml = reinterpret_cast<float2 *>(lds + ML0);

    // the page of each 8-key group of this key group's tile t (absent: below 0), by the scalar unit
    const ConstI32 table = (ConstI32)(uintptr_t)(A.table + T.seq * A.table_stride);
    const int last = T.S.kv - 1;  // >= 0 where there are rounds
    auto page_at = [&](int p) {
        const int x = table[min(p, max(last, 0)) >> A.page_shift];
        return (unsigned)x < (unsigned)A.num_pages ? x : -1;
    };
    auto pages_of = [&](int t) { return Pages{page_at(t), page_at(t + 8), page_at(t + 16), page_at(t + 24)}; };
    const int smask = (1 << A.page_shift) - 1;
    const char *const k_pool = static_cast<const char *>(A.k) + (int64_t)kvh * A.head_stride * EB;
    const char *const v_pool = static_cast<const char *>(A.v) + (int64_t)kvh * A.head_stride * EB;
    const uint32_t load_rows = 64 / LPR * R.slot_bytes;  // from one load of a group to the next: 64 / LPR rows
    auto group_base = [&](const char *pool, int t, int g, int page) {  // an absent group reads page 0
        const int slot = min(t + 8 * g, max(last, 0)) & smask & ~7;
        return pool + ((uint64_t)(uint32_t)max(page, 0) * R.page_bytes + (uint32_t)slot * R.slot_bytes);
    };
    // the loop recomputes what hangs on the lane alone (see `fresh`), loads' addresses among it
    auto load_half = [&](const char *pool, bool swizzle, int t, const Pages &pg, uint32_t at, int lane) {
        const uint32_t off_row = (uint32_t)(lane / LPR) * R.slot_bytes;
#pragma unroll
        for (int i = 0; i < GW; ++i) {
            const int g = rt * GW + i;
            const int page = pg.of(g);
            const char *base = group_base(pool, t, g, page);
            if (GB >= 1024 || lane < GB / 16)
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const int x = lane % LPR, r = n * (64 / LPR) + lane / LPR;
                    dma16(base + n * load_rows, off_row + (swizzle ? x ^ k_swizzle<RB>(r) : x) * 16, at + g * GB + n * 1024);
                }
        }
    };
    auto load_scales = [&](int t, const Pages &pg, int slot, int lane) {  // lane c: ks (half 0) or vs of key c
        const int c = lane & 31, h = lane >> 5;
        const int p = min(t + c, max(last, 0));
        const int page = pg.of(c >> 3);
        dma4((h ? A.vs : A.ks) + scale_offset(A, max(page, 0), p, kvh), lds0 + SC0 + wave * 512 + slot * 256);
    };
    auto ring = [&](int slot, int half) { return (uint32_t)(((kg * NS + slot) * 2 + half) * P::HALF); };
    auto tile_at = [&](int i) { return k0 + (i * KG + kg) * kKeys; };

    // this lane's query row
    const int first = T.first + rt * kRows;  // of this wave
    const int row = first + c;
    const bool real = row < T.rows, active = first < T.rows;
    const int token = real ? R.group.div(row) : 0, head = kvh * (int)R.group.d + (real ? R.group.mod(row) : 0);
    const int pos = real ? T.S.kv - T.S.rows + token : -1;
    const int p_first = T.S.kv - T.S.rows + R.group.div(first);  // the wave's first row, and its last
    const int p_last = T.S.kv - T.S.rows + R.group.div(max(min(first + kRows, T.rows) - 1, 0));

    Pages pg{-1, -1, -1, -1}, pg_next = pg;
    if (rounds) {
        pg = pages_of(tile_at(0));
        if (I8) load_scales(tile_at(0), pg, 0, lane);
        load_half(k_pool, true, tile_at(0), pg, lds0 + ring(0, 0), lane);
        load_half(v_pool, false, tile_at(0), pg, lds0 + ring(0, 1), lane);
        if (rounds > 1) pg_next = pages_of(tile_at(1));
    }
    constexpr int QL = P::QL;
    h8 q[KS - QL];
    char *const q_lds = lds + Q0 + wave * QL * 1024;
    float q_sum = 0.0f;
    {
        const _Float16 *src = R.q + (int64_t)(T.S.start + token) * R.q_stride + (int64_t)head * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            // the k-step's 8 dims of this half, in the order that K's reads give them
            const int at = I8 ? 32 * (s / 2) + 16 * h + 8 * (s % 2) : 16 * s + 8 * h;
            h8 x = *reinterpret_cast<const h8 *>(src + at);
            const uint32_t sign = R.q_sign;
            u32x4 y = __builtin_bit_cast(u32x4, x);
#pragma unroll
            for (int n = 0; n < 4; ++n) y[n] = real ? y[n] ^ sign : 0u;
            x = __builtin_bit_cast(h8, y);
            if (I8)
#pragma unroll
                for (int n = 0; n < 8; ++n) q_sum += (float)x[n];
            if (s < KS - QL) q[s] = x;
            else *reinterpret_cast<h8 *>(q_lds + (s - (KS - QL)) * 1024 + lane * 16) = x;
        }
        if (I8) q_sum = other_half_sum(q_sum);
    }
    const float s_init = I8 ? -q_sum * 0x1p-17f : 0.0f;  // the codes' bias, see codes_h8

    f16x o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = f16x{};
    // vref: the power of two of the row's V scales; w_sum: the sum of the rounded weights (int8)
    // off: the exponents' offset, -m scale2 - log2(vref); l is in units of vref too
    float m = -INFINITY, l = 0.0f, vref = 0x1p-100f, w_sum = 0.0f, off = I8 ? 100.0f : 0.0f;

    const int lane_ = lane;
    for (int i = 0; i < rounds; ++i) {
        // A fresh copy of the lane index: addresses and masks that hang on it are worked out again each time
        // (a few instructions); kept across the loop they would not fit beside the output and Q.
        int lane = lane_;
        float bias0 = s_init;
        asm volatile("" : "+v"(lane), "+v"(bias0));
        const int h = lane >> 5, c = lane & 31;
        const int t0 = tile_at(i), slot = NS == 1 ? 0 : i % NS;
        // which keys of the tile exist (scalar)
        uint32_t keys = T.S.kv - t0 >= 32 ? 0xffffffffu : (T.S.kv > t0 ? (1u << (T.S.kv - t0)) - 1 : 0u);
        if (t0 >= k1) keys = 0;
        keys &= (pg.a < 0 ? 0u : 0xffu) | (pg.b < 0 ? 0u : 0xff00u) | (pg.c < 0 ? 0u : 0xff0000u) | (pg.d < 0 ? 0u : 0xff000000u);
        const bool more = i + 1 < rounds;
        if (RT == 1) {
            wait_loads<LOADS>();  // K and the scales are here, V may be on its way
        } else {
            wait_loads<0>();
            wait_lds();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (more) {  // the other buffer was last read before the barrier
                if (I8) load_scales(tile_at(i + 1), pg_next, (i + 1) & 1, lane);
                load_half(k_pool, true, tile_at(i + 1), pg_next, lds0 + ring((i + 1) % NS, 0), lane);
                load_half(v_pool, false, tile_at(i + 1), pg_next, lds0 + ring((i + 1) % NS, 1), lane);
            }
        }
        const bool skip = !active || !keys || t0 > p_last || (R.window && t0 + kKeys - 1 <= p_first - R.window);
        f16x x;
        if (!skip) {
            // chunk 2 n + h of the lane's row, swizzled: the chunk's low three bits, so an XOR of the address
            const uint32_t kb = ring(slot, 0) + c * RB + (h ^ k_swizzle<RB>(c)) * 16;
            constexpr int KC = RB / 32 < 4 ? RB / 32 : 4;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = bias0;
            // K's reads run two products ahead (and no further: the scheduling barriers keep the compiler from
            // either gathering them, for which there are no registers, or waiting for each)
            constexpr int NK = RB / 32, AHEAD = 2;
            u32x4 k[NK];
            h8 q_last[QL > 0 ? QL : 1];
            auto read_k = [&](int n) {
                k[n] = *reinterpret_cast<const u32x4 *>(lds + (kb ^ (n % KC * 32)) + n / KC * KC * 32);
            };
#pragma unroll
            for (int n = 0; n < AHEAD && n < NK; ++n) read_k(n);
            f4 ks[4];
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                if (n + AHEAD < NK) read_k(n + AHEAD);
                if (QL && n == (KS - QL) / (I8 ? 2 : 1) - 1)  // a step before the first that needs one
#pragma unroll
                    for (int s = 0; s < QL; ++s) q_last[s] = *reinterpret_cast<const h8 *>(q_lds + s * 1024 + lane * 16);
                if (I8 && n + 1 == NK)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        ks[g] = *reinterpret_cast<const f4 *>(scales + (i & 1) * 256 + (8 * g + 4 * h) * 4);
                __builtin_amdgcn_sched_barrier(0);
                auto q_at = [&](int s) { return s < KS - QL ? q[s < KS - QL ? s : 0] : q_last[s < KS - QL ? 0 : s - (KS - QL)]; };
                if constexpr (I8) {
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_h8(k[n].x, k[n].y), q_at(2 * n), x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_h8(k[n].z, k[n].w), q_at(2 * n + 1), x, 0, 0, 0);
                } else {
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, k[n]), q_at(n), x, 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (I8)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= ks[r / 4][r % 4];
        }
        if (RT == 1 && more) {
            wait_lds();
            if (I8) load_scales(tile_at(i + 1), pg_next, (i + 1) & 1, lane);
            load_half(k_pool, true, tile_at(i + 1), pg_next, lds0 + ring(0, 0), lane);
        }
        h8 p[2];
        uint32_t seen = 0xffffffffu;  // bit 8 g + n: this row sees the key of register 4 g + n
        bool edge = false;
        if (!skip) {
            edge = t0 + kKeys - 1 > p_first || (R.window && t0 <= p_last - R.window) || keys != 0xffffffffu;
            if (edge) {
                const int hi = pos - t0, lo = R.window ? pos - R.window - t0 : -1;  // keys lo + 1 .. hi of the tile
                seen = hi < 0 ? 0u : (hi >= 31 ? keys : keys & ((2u << hi) - 1));
                if (lo >= 0) seen = lo >= 31 ? 0u : seen & ~((2u << lo) - 1);
                seen >>= 4 * h;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool ok = seen >> (8 * (r / 4) + r % 4) & 1;
                    x[r] = ok ? x[r] : -INFINITY;
                }
            }
            float top = x[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
            top = other_half_max(top);
            float vtop = 0.0f;  // the largest V scale that the row sees
            uint32_t v_scales = (i & 1) * 256 + 128 + 16 * h;
            if (I8) {
                if (edge) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f4 y = *reinterpret_cast<const f4 *>(scales + v_scales + 32 * g);
#pragma unroll
                        for (int n = 0; n < 4; ++n) vtop = fmaxf(vtop, seen >> (8 * g + n) & 1 ? fabsf(y[n]) : 0.0f);
                    }
                    vtop = other_half_max(vtop);
                } else {  // every key: a lane each
                    vtop = half_max(fabsf(*reinterpret_cast<const float *>(scales + (i & 1) * 256 + 128 + 4 * c)));
                }
                asm volatile("" : "+v"(v_scales));  // read again below rather than kept
            }
            if (__any(top > m + R.lazy || (m == -INFINITY && top > -INFINITY) || (I8 && vtop > vref))) {
                const float mn = fmaxf(m, top);
                float f = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * R.scale2);
                if (I8) {
                    const float to = fmaxf(vref, pow2_above(vtop));
                    f *= vref / to;
                    w_sum *= f;
                    vref = to;
                }
                l *= f;
#pragma unroll
                for (int j = 0; j < DPL; ++j) o[j] *= f;
                m = mn;
                off = (m == -INFINITY ? 0.0f : -m * R.scale2) - (I8 ? pow2_log(vref) : 0.0f);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f4 y = {};
                if (I8) y = *reinterpret_cast<const f4 *>(scales + v_scales + 32 * g);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int r = 4 * g + n;
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], R.scale2, off));
                    if (I8) l += e;
                    p[r / 8][r % 8] = (_Float16)(I8 ? e * y[n] : e);
                }
            }
            if (I8 && edge) {  // a masked scale may be anything, NaN included
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int b = 8 * (k / 2) + 2 * (k % 2);  // bits of registers 2 k and 2 k + 1
                    u32x4 w = __builtin_bit_cast(u32x4, p[k / 4]);
                    w[k % 4] &= (seen >> b & 1 ? 0xffffu : 0u) | (seen >> b & 2 ? 0xffff0000u : 0u);
                    p[k / 4] = __builtin_bit_cast(h8, w);
                }
            }
            // the sum of the rounded weights: the row's sum (f16), or what takes the codes' bias off (int8)
            const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
            float &sum = I8 ? w_sum : l;
#pragma unroll
            for (int r = 0; r < 8; ++r)
                sum = __builtin_amdgcn_fdot2(h2{p[r / 4][2 * (r % 4)], p[r / 4][2 * (r % 4) + 1]}, one, sum, false);
        }
        if (RT == 1) {  // V is here, the next K and scales may be on their way
            if (more) wait_loads<LOADS + (I8 ? 1 : 0)>();
            else wait_loads<0>();
        }
        if (!skip) {
            char *const tile = lds + ring(slot, 1);
            bool odd = false;
            if (!I8 && edge) {
                // Absent keys hold anything: their rows are cleared (by every wave that shares the tile, with
                // the same zeros). Then whether the tile has a NaN or an infinity: exponent bits all ones.
                for (uint32_t gone = ~keys; gone; gone &= gone - 1)
                    if (lane < LPR) *reinterpret_cast<u32x4 *>(tile + (__ffs(gone) - 1) * RB + lane * 16) = u32x4{};
                uint32_t any = 0;
#pragma unroll 4
                for (int n = 0; n < P::HALF / 1024; ++n) {
                    const u32x4 y = *reinterpret_cast<const u32x4 *>(tile + n * 1024 + lane * 16);
#pragma unroll
                    for (int w = 0; w < 4; ++w) any |= (y[w] & 0x7fff7fffu) + 0x04000400u;
                }
                odd = __any(any & 0x80008000u);
            }
            const char *vb = tile + c * VB + 4 * h * RB;
            // the lane's dims of block u, of the 8 keys of k-step s
            auto v_words = [&](int s, int u, uint32_t (&v)[8][(VB + 3) / 4]) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const char *at = vb + (16 * s + 8 * (n / 4) + n % 4) * RB + u * 32 * VB;
                    if constexpr (VB == 8) {
                        const uint2 y = *reinterpret_cast<const uint2 *>(at);
                        v[n][0] = y.x;
                        v[n][1] = y.y;
                    } else if constexpr (VB == 4) {
                        v[n][0] = *reinterpret_cast<const uint32_t *>(at);
                    } else {
                        v[n][0] = *reinterpret_cast<const uint16_t *>(at);
                    }
                    if (I8) v[n][0] ^= 0x80808080u;
                }
            };
            auto v_operand = [&](auto W, const uint32_t (&v)[8][(VB + 3) / 4]) {
                constexpr int w = decltype(W)::value;
                if constexpr (I8)
                    return words_h8(code_pair<w>(v[0][0], v[1][0]), code_pair<w>(v[2][0], v[3][0]),
                                    code_pair<w>(v[4][0], v[5][0]), code_pair<w>(v[6][0], v[7][0]));
                else
                    return words_h8(half_pair<w>(v[0], v[1]), half_pair<w>(v[2], v[3]), half_pair<w>(v[4], v[5]),
                                    half_pair<w>(v[6], v[7]));
            };
            if (odd) {
                // A NaN or an infinity at a key that some rows see and others do not is kept out of the
                // product (below) and put into the rows that see it, a key at a time.
#pragma unroll 1
                for (int kk = 0; kk < kKeys; ++kk) {
                    const int j = t0 + kk;
                    const bool sees = (keys >> kk & 1) && j <= pos && (!R.window || j > pos - R.window);
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int d = 32 * UD * u + UD * (8 * (r / 4) + 4 * h + r % 4);
#pragma unroll
                            for (int w = 0; w < UD; ++w) {
                                const uint32_t x = *reinterpret_cast<const uint16_t *>(tile + kk * RB + (d + w) * 2);
                                if (sees && (x & 0x7c00u) == 0x7c00u) o[u * UD + w][r] = __builtin_nanf("");
                            }
                            __builtin_amdgcn_sched_barrier(0);  // a few loads at a time: the registers are full
                        }
                }
            }
            uint32_t v[2 * U + 1][8][(VB + 3) / 4];  // V's reads, one step ahead
            if (!P::TIGHT) v_words(0, 0, v[0]);
            each<0, 2 * U>([&](auto Step) {
                constexpr int step = decltype(Step)::value, ss = step / U, u = step % U;
                constexpr int next = P::TIGHT ? step : step + 1;
                if (next < 2 * U) v_words(next / U, next % U, v[next]);
                __builtin_amdgcn_sched_barrier(0);
                if (odd)
#pragma unroll
                    for (int n = 0; n < 8; ++n)
#pragma unroll
                        for (int w = 0; w < (VB + 3) / 4; ++w) v[step][n][w] &= ~odd_mask(v[step][n][w]);
                each<0, UD>([&](auto W) {
                    f16x &acc = o[u * UD + decltype(W)::value];
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_operand(W, v[step]), p[ss], acc, 0, 0, 0);
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        }
        pg = pg_next;
        if (more) {
            if (RT == 1) {
                wait_lds();
                load_half(v_pool, false, tile_at(i + 1), pg, lds0 + ring(0, 1), lane);
            }
            if (i + 2 < rounds) pg_next = pages_of(tile_at(i + 2));
        }
    }
    l = other_half_sum(l);
    if (I8) {
        w_sum = other_half_sum(w_sum);
        l *= vref;
    }
    m *= R.scale2;  // from here on in exponents

    // The key groups' parts of a row, relative to their common maximum, summed in LDS a quarter of the
    // registers at a time: registers 4 ph .. 4 ph + 3 of the operands of block u are dims
    // 32 UD u + UD (8 ph + 4 h + 0..3) + 0..UD-1, 8 UD consecutive ones over both halves.
    if (h == 0) ml[wave * kRows + c] = make_float2(m, l);
    __syncthreads();
    float f;
    {
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < KG; ++g) top = fmaxf(top, ml[(g * RT + rt) * kRows + c].x);
        f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
        if (I8) f *= vref * 0x1p24f;
    }
    const float bias = I8 ? w_sum * 0x1p-17f : 0.0f;
    float *const part = reinterpret_cast<float *>(lds);
    // summing: 2 UD threads a row of 8 UD dims each (4 dims a thread), 64 / (2 UD) rows a wave and round
    constexpr int TPR = 2 * UD, RPW = 64 / TPR;
    const bool whole = R.splits.d == 1;
#pragma unroll
    for (int ph = 0; ph < 4; ++ph) {
        if (ph) __syncthreads();
#pragma unroll
        for (int j = 0; j < DPL; ++j)
#pragma unroll
            for (int n = 0; n < 4; ++n)
                part[(wave * DPL * 4 + j * 4 + n) * 72 + lane] = (o[j][4 * ph + n] - bias) * f;
        __syncthreads();
        // wave kg of row tile rt: rows kg * RPW .. of each KG * RPW
#pragma unroll
        for (int b = 0; b < kRows / (KG * RPW > kRows ? kRows : KG * RPW); ++b) {
            const int rr = (b * KG + kg) * RPW + lane / TPR;
            if (rr >= kRows || first + rr >= T.rows) continue;
            // this thread's 4 dims of a block: element e of its 8 UD is half hh, register nn, operand w
            float y[U][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int el = (lane % TPR) * 4 + e, hh = el / (4 * UD), nn = el / UD % 4, w = el % UD;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float a = 0.0f;
#pragma unroll
                    for (int g = 0; g < KG; ++g)
                        a += part[((g * RT + rt) * DPL * 4 + (u * UD + w) * 4 + nn) * 72 + hh * 32 + rr];
                    y[u][e] = a;
                }
            }
            float top = -INFINITY, total = 0.0f;
#pragma unroll
            for (int g = 0; g < KG; ++g) top = fmaxf(top, ml[(g * RT + rt) * kRows + rr].x);
#pragma unroll
            for (int g = 0; g < KG; ++g) {
                const float2 x = ml[(g * RT + rt) * kRows + rr];
                total += x.y * __builtin_amdgcn_exp2f(x.x - (top == -INFINITY ? 0.0f : top));
            }
            const int64_t slot = (((int64_t)blockIdx.x * R.splits.d + blockIdx.y) * A.kv_heads + kvh) * (kRows * RT) + rt * kRows + rr;
            const int d = 8 * UD * ph + (lane % TPR) * 4, grow = first + rr;
            const int64_t out = ((int64_t)(T.S.start + R.group.div(grow)) * R.heads + kvh * (int)R.group.d + R.group.mod(grow)) * D;
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float4 z = make_float4(y[u][0], y[u][1], y[u][2], y[u][3]);
                if (whole)
                    attn_put4(R, out + 32 * UD * u + d, make_float4(z.x * inv, z.y * inv, z.z * inv, z.w * inv));
                else
                    *reinterpret_cast<float4 *>(R.part_o + slot * D + 32 * UD * u + d) = z;
            }
            if (!whole && ph == 0 && lane % TPR == 0) R.part_ml[slot] = make_float2(top, total);
        }
    }
}

// ---- the parts of a split row joined -----------------------------------------------------------------

// Grid (tiles, row blocks, KV heads): D / 4 threads a row, G groups of them taking the splits in turn.
template <int D, int G>
__global__ __launch_bounds__(256) void attn_join_kernel(PagedArgs A, AttnArgs R, int tile_rows, int unit) {
    constexpr int TR = D / 4, RBK = 256 / (TR * G);
    __shared__ float4 os[G > 1 ? 256 : 1];
    __shared__ float2 mls[G > 1 ? 256 : 1];
    const int t = threadIdx.x, d = (t % TR) * 4, g = t / TR % G, kvh = blockIdx.z;
    const int rr = blockIdx.y * RBK + t / (TR * G);
    const Tile T = find_tile(A, R.group, R.window, blockIdx.x, tile_rows);
    if (!T.live || T.first + (int)blockIdx.y * RBK >= T.rows) return;
    const int row = T.first + rr;
    const bool real = rr < tile_rows && row < T.rows;
    const int per = split_tiles(T, R.splits, unit);
    const int n = real ? max(1, ((T.hi - T.lo + kKeys - 1) / kKeys + per - 1) / per) : 0;
    const int64_t stride = (int64_t)A.kv_heads * tile_rows;
    const int64_t slot = ((int64_t)blockIdx.x * R.splits.d * A.kv_heads + kvh) * tile_rows + rr;
    float m = -INFINITY, l = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float pm, float pl, float4 a) {
        const float mn = fmaxf(m, pm), mu = mn == -INFINITY ? 0.0f : mn;
        const float fo = __builtin_amdgcn_exp2f(m - mu), fn = __builtin_amdgcn_exp2f(pm - mu);
        l = l * fo + pl * fn;
        y.x = y.x * fo + a.x * fn;
        y.y = y.y * fo + a.y * fn;
        y.z = y.z * fo + a.z * fn;
        y.w = y.w * fo + a.w * fn;
        m = mn;
    };
    for (int s = g; s < n; s += 4 * G) {  // four splits' loads at a time
        float2 pm[4];
        float4 a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t at = slot + min(s + i * G, n - 1) * stride;
            pm[i] = R.part_ml[at];
            a[i] = *reinterpret_cast<const float4 *>(R.part_o + at * D + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s + i * G < n) add(pm[i].x, pm[i].y, a[i]);
    }
    if (G > 1) {
        os[t] = y;
        mls[t] = make_float2(m, l);
        __syncthreads();
        if (g) return;
#pragma unroll
        for (int i = 1; i < G; ++i) add(mls[t + i * TR].x, mls[t + i * TR].y, os[t + i * TR]);
    }
    if (!real) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    attn_put4(R, ((int64_t)(T.S.start + R.group.div(row)) * R.heads + kvh * (int)R.group.d + R.group.mod(row)) * D + d,
              make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
}

// ---- host ---------------------------------------------------------------------------------------------

struct AttnPlan {
    int rt;         // row tiles of a block
    int64_t tiles;  // blocks' row ranges, an upper bound over the batch
    int splits, key_groups;
    size_t bytes;
};

static int key_groups(int rt, int row_bytes) { return rt == 1 ? 4 : (rt == 2 && row_bytes < 512 ? 4 : 2); }

static AttnPlan attn_plan(const PagedArgs &A, const g4_kv_pages *pages, int heads, int window) {
    const int group = heads / A.kv_heads, d = pages->head_dim;
    AttnPlan P;
    const int64_t most = (int64_t)A.max_q * group;  // rows of a sequence
    P.rt = most <= kRows ? 1 : (most <= 2 * kRows ? 2 : 4);
    P.key_groups = key_groups(P.rt, pages->kind == G4_KIND_I8 ? d : 2 * d);
    const int rows = kRows * P.rt;
    P.tiles = std::min((most + rows - 1) / rows * A.seqs, (int64_t)A.tokens * group / rows + A.seqs);
    int64_t keys = A.max_kv;
    if (window) keys = std::min<int64_t>(keys, (int64_t)window + kKeys + rows / group + 1);
    const int64_t rounds = (keys + P.key_groups * kKeys - 1) / (P.key_groups * kKeys);
    const int64_t want = (P.rt == 1 ? 2 : 1) * (int64_t)device_cu_count();
    const int64_t blocks = P.tiles * A.kv_heads;
    P.splits = (int)std::max<int64_t>(1, std::min<int64_t>({rounds, (want + blocks - 1) / blocks, 64}));
    const int64_t slots = P.tiles * P.splits * A.kv_heads * rows;
    P.bytes = P.splits == 1 ? 16 : (size_t)slots * (d * sizeof(float) + sizeof(float2));
    return P;
}

template <int D, int CK, int RT>
static void launch_rows(const PagedArgs &A, const AttnArgs &R, const AttnPlan &P, hipStream_t stream) {
    static_assert(Shape<D, CK, RT>::LDS <= 160 * 1024, "LDS of a CU");
    hipLaunchKernelGGL((attn_kernel<D, CK, RT>), dim3((unsigned)P.tiles, P.splits, A.kv_heads),
                       dim3(64 * Shape<D, CK, RT>::WAVES), 0, stream, A, R);
}

template <int D, int CK>
static int launch_attn(const PagedArgs &A, const AttnArgs &R, const AttnPlan &P, hipStream_t stream) {
    if (P.rt == 1) launch_rows<D, CK, 1>(A, R, P, stream);
    else if (P.rt == 2) launch_rows<D, CK, 2>(A, R, P, stream);
    else launch_rows<D, CK, 4>(A, R, P, stream);
    G4_LAUNCHED("attn_kernel");
    if (P.splits > 1) {
        const int rows = kRows * P.rt;
        if (P.splits >= 8) {
            constexpr int rb = 256 / (D / 4 * 4);
            hipLaunchKernelGGL((attn_join_kernel<D, 4>), dim3((unsigned)P.tiles, rows / rb, A.kv_heads), dim3(256), 0,
                               stream, A, R, rows, P.key_groups);
        } else {
            constexpr int rb = 256 / (D / 4);
            hipLaunchKernelGGL((attn_join_kernel<D, 1>), dim3((unsigned)P.tiles, rows / rb, A.kv_heads), dim3(256), 0,
                               stream, A, R, rows, P.key_groups);
        }
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
    if (A->page_stride > INT32_MAX || A->slot_stride * pages->page_size > INT32_MAX)
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: pages, or a page's slots, 2^31 or more elements apart");
    return G4_OK;
}

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_attention_chunk_workspace_bytes(const g4_kv_pages *pages, const g4_chunk *chunk, int heads,
                                          int window) {
    PagedArgs A;
    if (attn_check(pages, chunk, heads, window, &A)) return 0;
    return attn_plan(A, pages, heads, window).bytes;
}

int g4_attention_chunk(const g4_kv_pages *pages, const g4_chunk *chunk, const void *q, int64_t q_stride,
                       int heads, float scale, int window, void *workspace, size_t workspace_bytes,
                       void *out, int out_kind, float in_scale, void *stream) {
    PagedArgs A;
    if (int st = attn_check(pages, chunk, heads, window, &A)) return st;
    if (!q || !out || !workspace) return set_error(G4_ERR_INVALID, "attention-chunk needs q, an output and a workspace");
    if (out_kind != G4_KIND_F16 && out_kind != G4_KIND_F32 && out_kind != G4_KIND_I8)
        return set_error(G4_ERR_INVALID, "attention-chunk: outputs are f16, f32 or int8 codes, got kind %d", out_kind);
    if (!std::isfinite(scale)) return set_error(G4_ERR_INVALID, "attention-chunk: scale must be finite");
    if (out_kind == G4_KIND_I8 && in_scale == 0.0f)
        return set_error(G4_ERR_INVALID, "attention-chunk: int8 codes need the consumer's inScale");
    const int64_t qw = (int64_t)heads * pages->head_dim;
    if (q_stride && (q_stride < qw || q_stride % 8))
        return set_error(G4_ERR_INVALID, "attention-chunk: q_stride must hold a row and be a multiple of 8");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return set_error(G4_ERR_INVALID, "attention-chunk: q, the output and the workspace must be 16-byte aligned");
    const AttnPlan P = attn_plan(A, pages, heads, window);
    if (workspace_bytes < P.bytes)
        return set_error(G4_ERR_INVALID, "attention-chunk: workspace %zu B < %zu B", workspace_bytes, P.bytes);
    float *part_o = static_cast<float *>(workspace);
    const bool i8 = pages->kind == G4_KIND_I8;
    const int eb = i8 ? 1 : 2;
    AttnArgs R{};
    R.q = static_cast<const _Float16 *>(q);
    R.q_stride = q_stride ? q_stride : qw;
    R.heads = heads;
    R.group = FastDiv::of(heads / A.kv_heads);
    // a scale of 0 as one too small to matter, so that a masked score stays minus infinity
    R.scale2 = std::max(std::fabs(scale) * 1.44269504088896340736f, 0x1p-100f) * (i8 ? 0x1p24f : 1.0f);
    R.lazy = kLazy / R.scale2;
    R.q_sign = scale < 0.0f ? 0x80008000u : 0u;
    R.page_bytes = (uint32_t)(A.page_stride * eb);
    R.slot_bytes = (uint32_t)(A.slot_stride * eb);
    R.window = window;
    R.out = out;
    R.out_kind = out_kind;
    R.in_scale = in_scale;
    R.splits = FastDiv::of(P.splits);
    R.part_o = part_o;
    R.part_ml = reinterpret_cast<float2 *>(part_o + P.tiles * P.splits * A.kv_heads * kRows * P.rt * pages->head_dim);
    hipStream_t st = as_stream(stream);
    switch (pages->head_dim) {
        case 64: return i8 ? launch_attn<64, G4_KIND_I8>(A, R, P, st) : launch_attn<64, G4_KIND_F16>(A, R, P, st);
        case 128: return i8 ? launch_attn<128, G4_KIND_I8>(A, R, P, st) : launch_attn<128, G4_KIND_F16>(A, R, P, st);
        default: return i8 ? launch_attn<256, G4_KIND_I8>(A, R, P, st) : launch_attn<256, G4_KIND_F16>(A, R, P, st);
    }
}

}  // extern "C"
