// Causal attention of a chunk of new tokens over the paged cache (include/g4serve.h).
//
// Query rows are (token, query head of the group) pairs, 32 to a tile, tokens first, so that every head
// on one KV head shares its loads. Both products run on the 32x32 matrix instructions in the transposed order
//   S^T = K Q^T   (A: 32 keys, B: 32 query rows)       O^T += V^T P^T   (A: 32 dims, B: 32 query rows)
// whose result lane holds one query row (lane % 32) and 16 of the keys: a row's softmax is per-lane
// arithmetic and one exchange with lane ^ 32, and the weights are the second product's B operand where
// they stand. The order of the k index of a product is free as long as both operands agree on it; the
// layouts below use that twice:
//  - P: lane half h holds, for k-step t of 16 keys, keys 16 t + 4 h + 0..3 and 16 t + 8 + 4 h + 0..3;
//  - V: a lane reads UD consecutive dims of each of these eight keys and permutes (f16) or converts (int8) them
//    into UD operands of eight keys each. No LDS transposes anything.
// The softmax keeps a running maximum (base 2) and sum in f32; the maximum moves, and the output is
// rescaled, only when a score passes it by more than 2^8, so weights reach 2^8 at most and are rounded to
// f16 (11 bits; an f16 cache's sum adds the rounded ones, an int8 cache's the exact ones, whose weights
// are rounded with V's scale in them).
// int8 rows: the scores are integer products of K's codes with Q as 16-bit fixed point of the row's largest
// magnitude, in two 8-bit digits (v_mfma_i32_32x32x32_i8 twice: the matrix time of one f16 product, K read
// once and not converted, which took 96 vector operations a tile). An element of Q is off by 2^-16 of the
// row's largest at most, K's codes not at all. K's scale multiplies the score, V's the weight. f16 would
// not hold scales of every size: weights are taken relative to a power of two at or up to 4 times the row's largest
// weight times scale, which scales the row's output and sum and enters the weights by their exponent. It moves only
// where the maximum does or a scale is 2^6 times as large, so a weight reaches 2^14 at most. (A power above the
// largest scale alone would lose a key of small scale beside one of large scale that weighs nothing.)
//
// What bounds it. Many rows: a key tile is 32 products of 32 cycles a wave and 354 other vector operations of 4, and a
// SIMD has two waves to overlap them. 2048 tokens on 8192 keys, 8 heads of 256, int8: 160 us, 752 TFLOP/s, 0.62 of
// what a large f16 product reaches. Of its 400 thousand cycles a SIMD's matrix unit is busy 116 and its vector
// unit 160; a wave waits 38% of its time, for loads, LDS and barriers. Neither unit is full: two waves do not hide
// all of each other's waits, and a third has no registers (8192 tokens on their own: 397 us; f16: 396-405 us).
// Few rows: reading the cache (32 single tokens on 16384 keys, f16: 89-94 us, 5.7-6.0 TB/s), and below that a block's
// way from its arguments to the first keys and from its last to memory, 4 us each: 4 tokens on 4096 keys take 9.8 us
// and their join 4.2-4.5.
#include "g4_paged.h"
#include "g4_key_span.h"
#include <algorithm>
#include <cmath>

namespace g4 {

typedef float f16x __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i16x __attribute__((ext_vector_type(16)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

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
    FastDiv group, per_seq;
    bool by_xcd;
    // Scores are kept as the products give them; the base-2 exponent is score * scale2, scale2 > 0. A
    // negative scale turns Q's signs over.
    float scale2;
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

// The next power of two above a scale (2^99 and more: 2^100), the same from 2^-100 on, and a power of two's exponent.
__device__ __forceinline__ float pow2_above(float v) {
    return __uint_as_float((__float_as_uint(fminf(v, 0x1p99f)) & 0x7f800000u) + 0x00800000u);
}
__device__ __forceinline__ float v_unit(float v) { return pow2_above(fmaxf(v, 0x1p-101f)); }
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

// Byte J of each of eight words of V codes, as the f16 operand: converted byte by byte, into the low half of a word
// and then into the high one. (A partial write is read a wait state later at the earliest.) Codes + 128 put together by
// byte permutes as f16 subnormals, the 128s taken off the output by the sum of the weights, are 2 operations a pair
// fewer; but beside a weight near 1 the f32 sums of such products lose what small weights add (an output of 3e-5 in a
// row of 2 was 17% off), and long runs of alike weights lost more (6e-4 over 131072 keys). 2048 tokens on 8192
// keys 161 us for 157, 8192 on their own 398 for 379, 32 single tokens as before.
template <int J>
__device__ __forceinline__ h8 code_operand(const uint32_t (&v)[8][1]) {
    u32x4 r;
#define G4_CVT(to, from, half, keep) \
    "v_cvt_f16_i16_sdwa " to ", sext(" from ") dst_sel:WORD_" half " dst_unused:UNUSED_" keep " src0_sel:BYTE_%12\n\t"
    asm(G4_CVT("%0", "%4", "0", "PAD") G4_CVT("%1", "%6", "0", "PAD") G4_CVT("%2", "%8", "0", "PAD") G4_CVT("%3", "%10", "0", "PAD")
        G4_CVT("%0", "%5", "1", "PRESERVE") G4_CVT("%1", "%7", "1", "PRESERVE") G4_CVT("%2", "%9", "1", "PRESERVE")
        G4_CVT("%3", "%11", "1", "PRESERVE") "s_nop 0"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(v[0][0]), "v"(v[1][0]), "v"(v[2][0]), "v"(v[3][0]), "v"(v[4][0]), "v"(v[5][0]), "v"(v[6][0]), "v"(v[7][0]), "n"(J));
#undef G4_CVT
    return __builtin_bit_cast(h8, r);
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

// The tile of block `id`: tile id % per_seq of sequence id / per_seq (by_xcd: of each eight blocks in a row one
// takes the next tile of each of eight sequences, so that a sequence's tiles run on one XCD, whose L2 they share:
// 32 x 8 tokens of 8 heads on up to 16008 keys 53 us for 59, on up to 4096 26.4 for 27.5); or with per_seq 0, where the grid has no
// room for every sequence's most, the id-th of all: sequences in order, ceil(rows * group / per) tiles each,
// looked for 64 sequences at a time.
__device__ __forceinline__ Tile find_tile(const PagedArgs &A, const FastDiv &group, const FastDiv &per_seq, bool by_xcd,
                                          int window, int id, int per) {
    Tile T{};
    int at = 0;
    if (per_seq.d) {
        const int n = by_xcd ? id >> 3 : id;
        T.seq = by_xcd ? per_seq.div(n) * 8 + (id & 7) : per_seq.div(n);
        at = per_seq.mod(n);
        if (T.seq >= A.seqs) return T;
        T.S = seq_span(A, T.seq);
        T.rows = min(T.S.rows, A.max_q) * (int)group.d;
        T.live = at * per < T.rows;
    } else {
        const int lane = threadIdx.x & 63;
        for (int base = 0; base < A.seqs && !T.live; base += 64) {
            int n = 0;
            SeqSpan S{0, 0, 0};
            if (base + lane < A.seqs) {
                S = seq_span(A, base + lane);
                n = (min(S.rows, A.max_q) * (int)group.d + per - 1) / per;
            }
            const int end = wave_scan_sum(n);
            const unsigned long long past = __ballot(end > id);
            if (past) {
                const int l = __ffsll((long long)past) - 1;
                T.seq = base + l;
                T.S.start = __builtin_amdgcn_readlane(S.start, l);
                T.S.rows = __builtin_amdgcn_readlane(S.rows, l);
                T.S.kv = __builtin_amdgcn_readlane(S.kv, l);
                T.rows = min(T.S.rows, A.max_q) * (int)group.d;
                at = id - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(n, l));
                T.live = true;
            }
            id -= __builtin_amdgcn_readlane(end, 63);
        }
    }
    T.first = at * per;
    const int p0 = T.S.kv - T.S.rows + group.div(T.first);
    const int p1 = T.S.kv - T.S.rows + group.div(max(min(T.first + per, T.rows) - 1, 0));
    const KeySpan K = key_span(p0, p1, window, kKeys);
    T.lo = K.lo;
    T.hi = K.hi;
    return T;
}

// Key tiles of one split: `n` key tiles cut in runs of `per`, a multiple of `unit` (a power of two).
__device__ __forceinline__ int split_tiles(const Tile &T, const FastDiv &splits, int unit) {
    const int n = (unsigned)(T.hi - T.lo + kKeys - 1) / kKeys;
    return max(splits.div(n + (int)splits.d - 1) + unit - 1, unit) & ~(unit - 1);
}

// N times 4 values to elements at(n), rounded or quantised as the output's kind says.
template <int N, typename F>
__device__ __forceinline__ void attn_put(void *out, int kind, float in_scale, const float4 (&y)[N], F at) {
    if (kind == G4_KIND_F32) {
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<float4 *>(static_cast<float *>(out) + at(n)) = y[n];
    } else if (kind == G4_KIND_F16) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const h4 o = {(_Float16)y[n].x, (_Float16)y[n].y, (_Float16)y[n].z, (_Float16)y[n].w};
            *reinterpret_cast<h4 *>(static_cast<_Float16 *>(out) + at(n)) = o;
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
            *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(out) + at(n)) =
                (srq_code_i(y[n].x, in_scale) & 255) | (srq_code_i(y[n].y, in_scale) & 255) << 8 |
                (srq_code_i(y[n].z, in_scale) & 255) << 16 | (uint32_t)(srq_code_i(y[n].w, in_scale) & 255) << 24;
    }
}

// ---- the attention kernel -------------------------------------------------------------------------------

// The block's shape: RT row tiles (32 query rows each) x KG key groups, a wave each. Key group g takes the
// key tiles g, g + KG, ... of the block's run; the waves of a group share its K and V tiles, which come
// straight to LDS as the rows stand in the cache, a ring of NS tiles each.
//  RT 1: a wave waits for its own loads only, and refills the K half of its buffer as soon as the scores
//        are done and the V half after the output (NS 1).
//  RT 2, 4: two block barriers a key tile, one before the softmax and one after it, and waves 4..7 one barrier
//        behind waves 0..3: of the two waves that share a SIMD, one has the matrix unit (a tile's output and
//        the next tile's scores) while the other has the vector unit. K comes two tiles ahead and V one. In
//        step, 8192 tokens took 447 us for 381 (int8, RT 2, V's codes by permutes) and 436 for 402 (f16, RT 4),
//        head_dim 128 221 for 181.
template <int D, int CK, int RT>
struct Shape {
    static constexpr int EB = CK == G4_KIND_I8 ? 1 : 2;  // bytes of an element
    static constexpr int RB = D * EB;                    // of a row
    static constexpr int HALF = kKeys * RB;              // of a tile's K or V
    static constexpr int KG = RT == 1 || (RT == 2 && CK == G4_KIND_I8) ? 4 : 2;
    static constexpr int NS = RT == 1 ? 1 : 2;
    static constexpr int WAVES = RT * KG;
    static constexpr int RING = KG * NS * 2 * HALF;
    // int8: the scales of a key group's tiles, for each 8 keys K's and then V's; they come with K
    static constexpr int NSC = NS + 1, SCALES = CK == G4_KIND_I8 ? KG * NSC * 256 : 0;
    // quarters of every wave's output that are joined at a time (see the end): as many as the ring holds
    static constexpr int PH = WAVES * D * 128 <= RING ? 4 : (WAVES * D * 64 <= RING ? 2 : 1);
    static constexpr int JOIN = WAVES * D * 32 * PH;
    // Q's last operands wait in LDS where two waves a SIMD share the registers: output and Q alone take 192 of 256
    static constexpr int QL = D == 256 && (CK == G4_KIND_I8 || RT == 4) ? 3 : 0;
    static constexpr bool TIGHT = D == 256 && CK == G4_KIND_F16 && RT == 4;  // no registers for V's reads ahead
    static constexpr int LDS = (RING > JOIN ? RING : JOIN) + SCALES + WAVES * (kRows * 8 + QL * 1024);
    // per SIMD: one block a CU, or two; int8 of 64 is a register over what four blocks may have
    static constexpr int MIN_WAVES = WAVES == 4 && LDS > 80 * 1024 ? 1 : (D == 64 && CK == G4_KIND_I8 ? 4 : 2);
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
template <int LANES>
__device__ __forceinline__ void dma4(const void *src, uint32_t lds) {
    // the first LANES lanes, by the mask rather than by a branch (the wave is whole here)
    uint64_t all;
    if constexpr (LANES == 64)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                     :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, exec\n\ts_mov_b64 exec, %3\n\ts_nop 0\n\t"
                     "global_load_lds_dword %2, off\n\ts_mov_b64 exec, %0"
                     : "=&s"(all)
                     : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src), "s"((1ull << LANES) - 1) : "memory", "m0");
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

// What a wave needs to load its 8-key groups of a key tile: bytes to the group in the pools, and in the
// scales' (int8); there: which of the tile's four groups have a page, a bit each.
template <int GW>
struct Next {
    uint64_t off[GW], row[GW];
    uint32_t there;
};

template <int D, int CK, int RT>
__global__ __launch_bounds__((64 * Shape<D, CK, RT>::WAVES), (Shape<D, CK, RT>::MIN_WAVES))
void attn_kernel(PagedArgs A, AttnArgs R) {
    using P = Shape<D, CK, RT>;
    constexpr bool I8 = CK == G4_KIND_I8;
    constexpr int EB = P::EB, RB = P::RB, KG = P::KG, NS = P::NS, KS = D / 16, DPL = D / 32;
    constexpr int NK = RB / 32;                                       // K reads of a lane
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
    const Tile T = find_tile(A, R.group, R.per_seq, R.by_xcd, R.window, blockIdx.x, kRows * RT);
    if (!T.live) return;
    const int per = split_tiles(T, R.splits, KG);
    const int k0 = T.lo + blockIdx.y * per * kKeys, k1 = min(T.hi, k0 + per * kKeys);
    if (blockIdx.y && k0 >= T.hi) return;
    const int rounds = (k1 - k0 + KG * kKeys - 1) / (KG * kKeys);  // 0 where there are no keys

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    constexpr int SC0 = P::RING > P::JOIN ? P::RING : P::JOIN, ML0 = SC0 + P::SCALES, Q0 = ML0 + P::WAVES * kRows * 8;
    char *const scales = lds + SC0 + kg * P::NSC * 256;
    float2 *const ml = reinterpret_cast<float2 *>(lds + ML0);

    // Pages: lane l looks up 8-key group l % 4 of the key group's tile 16 w + l / 4, 16 tiles at a time and
    // a tile ahead; a tile's four pages are then register reads (a scalar load per tile would be waited
    // for with the tile's LDS reads: they share a counter).
    const int last = max(T.S.kv - 1, 0);
    const int32_t *const table = A.table + T.seq * A.table_stride;
    auto tile_at = [&](int i) { return k0 + (i * KG + kg) * kKeys; };
    auto look_up = [&](int w) {
        return table[min(tile_at(16 * w + lane / 4) + 8 * (lane % 4), last) >> A.page_shift];
    };
    const int smask = (1 << A.page_shift) - 1;
    const char *const k_pool = static_cast<const char *>(A.k) + (int64_t)kvh * A.head_stride * EB;
    const char *const v_pool = static_cast<const char *>(A.v) + (int64_t)kvh * A.head_stride * EB;
    const uint32_t load_rows = 64 / LPR * R.slot_bytes;  // from one load of a group to the next: 64 / LPR rows
    int page_v = 0;      // the pages of 16 tiles, or once the last of them is read out the next 16, not yet checked
    uint64_t there = 0;  // bit l: lane l's is one
    auto next_tile = [&](int j) {  // for j = 0, 1, ... in turn
        if ((j & 15) == 0) {
            there = __ballot((unsigned)page_v < (unsigned)A.num_pages);
            page_v = (unsigned)page_v < (unsigned)A.num_pages ? page_v : 0;  // an absent group reads page 0
        }
        const int l = (j & 15) * 4;
        Next<GW> N;
        N.there = (uint32_t)(there >> l) & 15;
#pragma unroll
        for (int i = 0; i < GW; ++i) {
            const uint32_t page = __builtin_amdgcn_readlane(page_v, l + rt * GW + i);
            const uint32_t at = min(tile_at(j) + 8 * (rt * GW + i), last) & smask & ~7;
            N.off[i] = (uint64_t)page * R.page_bytes + at * R.slot_bytes;
            N.row[i] = (((uint64_t)page * A.kv_heads + kvh) << A.page_shift) + at;
        }
        if ((j & 15) == 15) page_v = look_up(j / 16 + 1);
        return N;
    };
    // the loop recomputes what hangs on the lane alone (see `fresh`), loads' addresses among it
    auto load_half = [&](const char *pool, bool swizzle, const Next<GW> &N, uint32_t at, uint32_t lane) {
        const uint32_t off_row = lane / LPR * R.slot_bytes, x = lane % LPR;
#pragma unroll
        for (int i = 0; i < GW; ++i) {
            const char *base = pool + N.off[i];
            if (GB >= 1024 || lane < GB / 16)
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const int r = n * (64 / LPR) + lane / LPR;
                    dma16(base + n * load_rows, off_row + (swizzle ? x ^ k_swizzle<RB>(r) : x) * 16,
                          at + (rt * GW + i) * GB + n * 1024);
                }
        }
    };
    // The scales of the wave's groups: lane 16 i + n is key n of group rt GW + i, of K (n < 8) or V.
    auto load_scales = [&](const Next<GW> &N, int slot, uint32_t lane) {
        uint64_t row = N.row[0];
#pragma unroll
        for (int i = 1; i < GW; ++i) {
            uint64_t r = N.row[i];
            asm volatile("" : "+s"(r));  // a value: or the array is kept in memory and indexed by the lane
            row = lane >> 4 == (uint32_t)i ? r : row;
        }
        dma4<16 * GW>((lane & 8 ? A.vs : A.ks) + row + (lane & 7),
                      lds0 + SC0 + (kg * P::NSC + slot) * 256 + rt * GW * 64);
    };
    auto ring = [&](int slot, int half) { return (uint32_t)(((kg * NS + slot) * 2 + half) * P::HALF); };

    // this lane's query row
    const int first = T.first + rt * kRows;  // of this wave
    const int row = first + c;
    const bool real = row < T.rows, active = first < T.rows;
    const int token = real ? R.group.div(row) : 0, head = kvh * (int)R.group.d + (real ? R.group.mod(row) : 0);
    const int pos = real ? T.S.kv - T.S.rows + token : -1;
    const int p_first = T.S.kv - T.S.rows + R.group.div(first);  // the wave's first row, and its last
    const int p_last = T.S.kv - T.S.rows + R.group.div(max(min(first + kRows, T.rows) - 1, 0));
    const int t_inner = R.window ? p_last - R.window + 1 : 0;  // the first key that every row of the wave sees

    // of the tile whose V is loaded next; and the bits `there` of the tiles i and i + 1
    Next<GW> ahead{};
    uint32_t there0 = 0, there1 = 0;
    if (rounds) {
        page_v = look_up(0);
        const Next<GW> N = next_tile(0);
        there0 = N.there;
        if (I8) load_scales(N, 0, lane);
        load_half(k_pool, true, N, lds0 + ring(0, 0), lane);
        if (RT > 1 && rounds > 1) {
            ahead = next_tile(1);
            there1 = ahead.there;
            if (I8) load_scales(ahead, 1, lane);
            load_half(k_pool, true, ahead, lds0 + ring(1, 0), lane);
        }
        if (RT == 1) ahead = N;
        if (RT > 1 || !I8) load_half(v_pool, false, N, lds0 + ring(0, 1), lane);
    }
    auto lds_sync = [&]() {  // LDS writes and reads of the block's waves are done; loads may be on their way
        wait_lds();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr int QL = P::QL;
    u32x4 q[KS - QL];
    char *const q_lds = lds + Q0 + wave * QL * 1024;
    float sc = R.scale2;  // exponents are score * sc
    {
        auto put_q = [&](int s, u32x4 x) {
            if (s < KS - QL) q[s < KS - QL ? s : 0] = x;
            else *reinterpret_cast<u32x4 *>(q_lds + (s - (KS - QL)) * 1024 + lane * 16) = x;
        };
        // a lane without a row takes the sequence's first: nothing of it is kept
        const _Float16 *src = R.q + (int64_t)(T.S.start + token) * R.q_stride + (int64_t)head * D;
        if constexpr (I8) {
            // In steps of 32 dims, shared out among the key groups' waves of a row tile, which exchange them in the V
            // halves of the ring's last slot (RT 1 loads V after this)
            static_assert(RT <= 2, "the V halves of four key groups hold two row tiles' Q");
            constexpr int QN = NK > KG ? NK / KG : 1;
            const int s0 = kg * QN;
            u32x4 x[2 * QN] = {};
            uint32_t top = 0;  // of the row's magnitudes, as f16 bits
            if (s0 < NK) {
#pragma unroll
                for (int s = 0; s < 2 * QN; ++s)  // the dims of this half in the order that K's reads give them
                    x[s] = *reinterpret_cast<const u32x4 *>(src + 32 * (s0 + s / 2) + 16 * h + 8 * (s % 2));
#pragma unroll
                for (int s = 0; s < 2 * QN; ++s)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const u16x2 y = __builtin_bit_cast(u16x2, x[s][n] & 0x7fff7fffu);
                        top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), y));
                    }
            }
            top = max(top & 0xffff, top >> 16);
            const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            top = max(both[0], both[1]);
            if (h == 0) ml[wave * kRows + c].x = __uint_as_float(top);
            lds_sync();
#pragma unroll
            for (int g = 0; g < KG; ++g) top = max(top, __float_as_uint(ml[(g * RT + rt) * kRows + c].x));
            const float amax = (float)bits_h2(top)[0];
            // With a NaN or an infinity in Q the digits are zeros and the scale is infinite: a score of a key that
            // the row sees is NaN, a masked one still minus infinity.
            const bool odd = top >= 0x7c00u;
            const float inv = top && !odd ? (R.q_sign ? -32512.0f : 32512.0f) / amax : 0.0f;
            sc = odd ? INFINITY : fmaxf(R.scale2 * (amax / 32512.0f), 0x1p-126f);
#pragma unroll
            for (int s = 0; s < 2 * QN; ++s)
#pragma unroll
                for (int n = 0; n < 4; ++n) x[s][n] = odd ? 0 : x[s][n];
            auto stage = [&](int at) {  // of the row tile's KS operands
                const int e = rt * KS + at;
                return lds + ring(NS - 1, 1) + (e / (KS / 2) - kg) * (NS * 2 * P::HALF) + e % (KS / 2) * 1024 + lane * 16;
            };
            // n = RNE(32512 q / amax); n + 128 stands in the low 16 bits of 1.5 2^23 + 128 + n: the second byte is
            // the high digit, the low byte less 128 the low one
            if (s0 < NK)
#pragma unroll
                for (int s = 0; s < QN; ++s) {
                    u32x4 hi, lo;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t n[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            n[i] = __float_as_uint(__builtin_fmaf(
                                (float)bits_h2(x[2 * s + w / 2][w % 2 * 2 + i / 2])[i % 2], inv, 0x1.8p23f + 128.0f));
                        const uint32_t a = __builtin_amdgcn_perm(n[1], n[0], 0x05010400u);
                        const uint32_t b = __builtin_amdgcn_perm(n[3], n[2], 0x05010400u);
                        lo[w] = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u;
                        hi[w] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                    }
                    *reinterpret_cast<u32x4 *>(stage(2 * (s0 + s))) = hi;
                    *reinterpret_cast<u32x4 *>(stage(2 * (s0 + s) + 1)) = lo;
                }
            lds_sync();
#pragma unroll
            for (int s = 0; s < KS; ++s) put_q(s, *reinterpret_cast<const u32x4 *>(stage(s)));
            lds_sync();
            if (RT == 1 && rounds) load_half(v_pool, false, ahead, lds0 + ring(0, 1), lane);
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 x = *reinterpret_cast<const u32x4 *>(src + 16 * s + 8 * h);
#pragma unroll
                for (int n = 0; n < 4; ++n) x[n] ^= R.q_sign;
                put_q(s, x);
            }
        }
    }

    f16x o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = f16x{};
    // int8: v_need: the largest weight times V's scale that the row has seen, up to a factor of 2, as of its last
    // rescaling; v_unit(v_need) is what the weights, off (the exponents' offset, -m scale2 - log2 of it) and l are
    // relative to. v_low: V scales up to it need no rescaling.
    float m = -INFINITY, l = 0.0f, off = I8 ? -100.0f : 0.0f;
    float v_low = 0x1p106f;
    if (I8) ml[wave * kRows + c].y = 0x1p99f;  // v_need: rarely used, and the registers are full

    const int lane_ = lane;
    constexpr int KC = NK < 4 ? NK : 4, AHEAD = D == 256 && I8 && RT == 1 ? 1 : 2;
    u32x4 k_first[RT > 1 ? AHEAD : 1];  // the tile's first K reads, made in the tile before (RT > 1)
    int slot = 0, sc_slot = 0;
    auto barrier = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto k_read = [&](int at, int lane, int n) {
        // chunk 2 n + h of the lane's row, swizzled: the chunk's low three bits, so an XOR of the address
        const int c = lane & 31, kb = at + c * RB + ((lane >> 5) ^ k_swizzle<RB>(c)) * 16;
        return *reinterpret_cast<const u32x4 *>(lds + (kb ^ (n % KC * 32)) + n / KC * KC * 32);
    };
    if (RT > 1 && rounds) {
        wait_loads<0>();
        barrier();
        if (P::WAVES > 4 && wave >= 4) barrier();
#pragma unroll
        for (int n = 0; n < AHEAD && n < NK; ++n) k_first[n] = k_read(ring(0, 0), lane, n);
    }
    // Active: a wave with rows. One without only takes its part in the loads. (Two loops, not a branch inside: the
    // output would be merged where the branch ends, and there are no registers for the copies.)
    auto run = [&](auto Active) {
    for (int i = 0; i < rounds; ++i) {
        // A fresh copy of the lane index: addresses and masks that hang on it are worked out again each time
        // (a few instructions); kept across the loop they would not fit beside the output and Q.
        int lane = lane_;
        asm volatile("" : "+v"(lane));
        const int h = lane >> 5, c = lane & 31;
        const int t0 = tile_at(i);
        const int sc_next = sc_slot + 1 == P::NSC ? 0 : sc_slot + 1;
        const int sc_after = sc_next + 1 == P::NSC ? 0 : sc_next + 1;
        const bool more = i + 1 < rounds;
        if (RT == 1) wait_loads<LOADS>();  // K and the scales are here, V may be on its way
        // K's reads run two steps ahead (one where registers are short); the scheduling barriers keep the compiler
        // from gathering them, for which there are no registers, and from waiting for each
        constexpr int KB = AHEAD + 1;
        u32x4 k[KB];
#pragma unroll
        for (int n = 0; n < AHEAD && n < NK; ++n)
            k[n] = RT > 1 ? k_first[n] : k_read(ring(slot, 0), lane, n);
        f16x x;
        uint32_t v[2 * U + 1][8][(VB + 3) / 4];  // V's reads, one step ahead
        char *const tile = lds + ring(slot, 1);
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
            }
        };
        // RT 1, between the products: the K half is free for the next tile; V has landed
        auto refill_k = [&]() {
            if (RT != 1 || !more) return;
            wait_lds();
            ahead = next_tile(i + 1);
            if (I8) load_scales(ahead, sc_next, lane);
            load_half(k_pool, true, ahead, lds0 + ring(0, 0), lane);
        };
        auto wait_v = [&]() {
            if (RT != 1) return;
            if (more) wait_loads<LOADS + (I8 ? 1 : 0)>();  // the next K and scales may be on their way
            else wait_loads<0>();
        };
        // RT > 1, between the scores and the softmax: every wave is done with this tile's K and the last one's V,
        // whose places the next loads take; and after the softmax: the loads made a tile ago have landed
        auto scores_done = [&]() {
            if (RT == 1) return;
            barrier();
            if (more) load_half(v_pool, false, ahead, lds0 + ring(slot ^ 1, 1), lane);
            if (i + 2 < rounds) {
                ahead = next_tile(i + 2);
                if (I8) load_scales(ahead, sc_after, lane);
                load_half(k_pool, true, ahead, lds0 + ring(slot, 0), lane);
            }
        };
        auto softmax_done = [&]() {
            if (RT == 1) return;
            if (i + 2 < rounds) wait_loads<2 * LOADS + (I8 ? 1 : 0)>();
            else if (more) wait_loads<LOADS>();
            else wait_loads<0>();
            barrier();
        };
        if constexpr (decltype(Active)::value) {
            u32x4 q_last[QL > 0 ? QL : 1];
            auto read_q_last = [&]() {
#pragma unroll
                for (int s = 0; s < QL; ++s) q_last[s] = *reinterpret_cast<const u32x4 *>(q_lds + s * 1024 + lane * 16);
            };
            auto q_at = [&](int s) { return s < KS - QL ? q[s < KS - QL ? s : 0] : q_last[s < KS - QL ? 0 : s - (KS - QL)]; };
            f4 ks[4];
            if constexpr (I8) {
                // codes times Q's high digits and low ones, 256 times the first and the second put together
                i16x a = {}, b = {};
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    if (n + AHEAD < NK) k[(n + AHEAD) % KB] = k_read(ring(slot, 0), lane, n + AHEAD);
                    if (QL && n == (KS - QL) / 2 - 1) read_q_last();  // a step before the first that needs one
                    __builtin_amdgcn_sched_barrier(0);
                    const v4i kn = __builtin_bit_cast(v4i, k[n % KB]);
                    a = __builtin_amdgcn_mfma_i32_32x32x32_i8(kn, __builtin_bit_cast(v4i, q_at(2 * n)), a, 0, 0, 0);
                    b = __builtin_amdgcn_mfma_i32_32x32x32_i8(kn, __builtin_bit_cast(v4i, q_at(2 * n + 1)), b, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) a[r] = (int)(((uint32_t)a[r] << 8) + (uint32_t)b[r]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    ks[g] = *reinterpret_cast<const f4 *>(scales + sc_slot * 256 + 64 * g + 16 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = (float)a[r];
            } else {
                x = f16x{};
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    if (n + AHEAD < NK) k[(n + AHEAD) % KB] = k_read(ring(slot, 0), lane, n + AHEAD);
                    if (QL && n == KS - QL - 1) read_q_last();
                    __builtin_amdgcn_sched_barrier(0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, k[n % KB]),
                                                               __builtin_bit_cast(h8, q_at(n)), x, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            scores_done();
            if (I8)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= ks[r / 4][r % 4];
            refill_k();
            h8 p[2];
            uint32_t seen = 0xffffffffu;  // bit 8 g + n: this row sees the key of register 4 g + n
            uint32_t keys = 0xffffffffu;  // that exist (scalar)
            const bool edge = t0 < t_inner || t0 > p_first - (kKeys - 1) || there0 != 15;
            if (edge) {
                keys = T.S.kv - t0 >= 32 ? 0xffffffffu : (T.S.kv > t0 ? (1u << (T.S.kv - t0)) - 1 : 0u);
                if (t0 >= k1) keys = 0;
                keys &= (there0 * 0x00204081u & 0x01010101u) * 0xffu;  // bits to bytes
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
            asm volatile("" : "+v"(seen));  // opaque: or what follows is made twice, with and without a mask
            float top = x[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
            top = other_half_max(top);
            const uint32_t v_scales = sc_slot * 256 + 32 + 16 * h;
            float v_mine = 0.0f;  // of V's scales, lane c key c's
            if (I8) v_mine = fabsf(*reinterpret_cast<const float *>(scales + sc_slot * 256 + (c >> 3) * 64 + 32 + c % 8 * 4));
            if (__any((top - m) * sc > kLazy || (I8 && v_mine > v_low))) {
                const float mn = fmaxf(m, top);
                off = mn == -INFINITY ? 0.0f : -mn * sc;
                float f;
                if (I8) {
                    float need = 0.0f;
                    uint32_t at = v_scales;
                    asm volatile("" : "+v"(at));  // loads of its own: those below would be kept from here on
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f4 y = *reinterpret_cast<const f4 *>(scales + at + 64 * g);
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            // a masked key's exponent is -1000: nothing, whatever its scale is
                            const float e = __builtin_amdgcn_fmed3f(__builtin_fmaf(x[4 * g + n], sc, off), -1000.0f, 0.0f);
                            need = fmaxf(need, __builtin_amdgcn_ldexpf(fminf(fabsf(y[n]), 0x1p100f), (int)e));
                        }
                    }
                    f = m == mn ? 0.0f : (m - mn) * sc;
                    float *const v_need = &ml[wave * kRows + c].y;
                    const float had = *v_need, unit = pow2_log(v_unit(had));
                    need = fmaxf(other_half_max(need), had * __builtin_amdgcn_exp2f(f));
                    *v_need = need;
                    const float vref = v_unit(need), log = pow2_log(vref);
                    f = __builtin_amdgcn_exp2f(f + (unit - log));
                    off -= log;
                    v_low = -half_max(-vref) * 64.0f;
                } else {
                    f = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * sc);
                }
                l *= f;
#pragma unroll
                for (int j = 0; j < DPL; ++j) o[j] *= f;
                m = mn;
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f4 y = {};
                if (I8) y = *reinterpret_cast<const f4 *>(scales + v_scales + 64 * g);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int r = 4 * g + n;
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], sc, off));
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
            if (!I8) {  // the sum of the rounded weights
                const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    l = __builtin_amdgcn_fdot2(h2{p[r / 4][2 * (r % 4)], p[r / 4][2 * (r % 4) + 1]}, one, l, false);
            }
            wait_v();
            softmax_done();
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
            auto v_operand = [&](auto W, const uint32_t (&v)[8][(VB + 3) / 4]) {
                constexpr int w = decltype(W)::value;
                if constexpr (I8)
                    return code_operand<w>(v);
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
        if constexpr (decltype(Active)::value) {
            if (RT > 1)
#pragma unroll
                for (int n = 0; n < AHEAD && n < NK; ++n) k_first[n] = k_read(ring(slot ^ 1, 0), lane, n);
        } else {
            scores_done();
            softmax_done();
        }
        if (RT > 1) slot ^= 1;
        sc_slot = sc_next;
        there0 = RT > 1 ? there1 : ahead.there;
        there1 = ahead.there;
        if (RT == 1 && more) {
            wait_lds();
            load_half(v_pool, false, ahead, lds0 + ring(0, 1), lane);
        }
    }
    };
    if (RT == 1 || active) run(std::integral_constant<bool, true>{});
    else run(std::integral_constant<bool, false>{});
    if (RT > 1 && P::WAVES > 4 && wave < 4 && rounds) barrier();
    l = other_half_sum(l);
    const float vref = I8 ? v_unit(ml[wave * kRows + c].y) : 1.0f;
    if (I8) l *= vref;
    m *= sc;  // from here on in exponents

    // The key groups' parts of a row, relative to their common maximum, summed in LDS PH quarters of the
    // registers at a time: registers 4 ph .. 4 ph + 3 of the operands of block u are dims
    // 32 UD u + UD (8 ph + 4 h + 0..3) + 0..UD-1, UD chunks of 4 in a row on either half.
    if (h == 0) ml[wave * kRows + c] = make_float2(m, l);
    __syncthreads();
    float f;
    {
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < KG; ++g) top = fmaxf(top, ml[(g * RT + rt) * kRows + c].x);
        f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));
        if (I8) f *= vref;
    }
    constexpr int PH = P::PH;
    // chunk e of half h of row c in block u and quarter ph; the XOR spreads a row's chunks over the banks
    auto chunk = [&](int wave, int ph, int u, int e, int h, int c) {
        return lds + ((((wave * PH + ph) * U + u) * UD + e) * 64 + h * 32 + (c ^ (e + UD * h))) * 16;
    };
    // summing: 2 UD threads a row, a chunk each, 64 / (2 UD) rows a wave; the KG waves of a row tile share its rows
    constexpr int TPR = 2 * UD, RPW = 64 / TPR, GROUPS = kRows / RPW, GPW = GROUPS > KG ? GROUPS / KG : 1;
    const int e_sum = lane % UD, h_sum = lane / UD & 1;
    const bool whole = R.splits.d == 1;
    const int kind = whole ? R.out_kind : G4_KIND_F32;
    bool live[GPW];
    float inv[GPW];
    int64_t to[GPW];  // of this thread's first chunk, in elements
#pragma unroll
    for (int i = 0; i < GPW; ++i) {
        const int group = kg * GPW + i, rr = group % GROUPS * RPW + lane / TPR, grow = first + rr;
        live[i] = group < GROUPS && grow < T.rows;
        float top = -INFINITY, total = 0.0f;
        float2 x[KG];
#pragma unroll
        for (int g = 0; g < KG; ++g) {
            x[g] = ml[(g * RT + rt) * kRows + rr];
            top = fmaxf(top, x[g].x);
        }
#pragma unroll
        for (int g = 0; g < KG; ++g) total += x[g].y * __builtin_amdgcn_exp2f(x[g].x - (top == -INFINITY ? 0.0f : top));
        if (whole) {
            inv[i] = total == 0.0f ? 0.0f : 1.0f / total;
            to[i] = ((int64_t)(T.S.start + R.group.div(grow)) * R.heads + kvh * (int)R.group.d + R.group.mod(grow)) * D;
        } else {
            inv[i] = 1.0f;
            to[i] = (((int64_t)blockIdx.x * R.splits.d + blockIdx.y) * A.kv_heads + kvh) * (kRows * RT) + rt * kRows + rr;
            if (live[i] && lane % TPR == 0) R.part_ml[to[i]] = make_float2(top, total);
            to[i] *= D;
        }
        to[i] += lane % TPR * 4;
    }
    void *const dst = whole ? R.out : R.part_o;
#pragma unroll
    for (int ph0 = 0; ph0 < 4; ph0 += PH) {
        if (ph0) __syncthreads();
#pragma unroll
        for (int ph = 0; ph < PH; ++ph)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < UD; ++e) {
                    f4 y;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        y[k] = o[u * UD + (4 * e + k) % UD][4 * (ph0 + ph) + (4 * e + k) / UD] * f;
                    *reinterpret_cast<f4 *>(chunk(wave, ph, u, e, h, c)) = y;
                }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < GPW; ++i) {
            if (!live[i]) continue;
            const int rr = (kg * GPW + i) % GROUPS * RPW + lane / TPR;
            float4 y[PH * U];
#pragma unroll
            for (int n = 0; n < PH * U; ++n) {
                f4 a = {};
#pragma unroll
                for (int g = 0; g < KG; ++g)
                    a += *reinterpret_cast<const f4 *>(chunk(g * RT + rt, n / U, n % U, e_sum, h_sum, rr));
                y[n] = make_float4(a[0] * inv[i], a[1] * inv[i], a[2] * inv[i], a[3] * inv[i]);
            }
            attn_put<PH * U>(dst, kind, R.in_scale, y,
                             [&](int n) { return to[i] + 32 * UD * (n % U) + 8 * UD * (ph0 + n / U); });
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
    const Tile T = find_tile(A, R.group, R.per_seq, R.by_xcd, R.window, blockIdx.x, tile_rows);
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
    const int64_t orow = (int64_t)(T.S.start + R.group.div(row)) * R.heads + kvh * (int)R.group.d + R.group.mod(row);
    const float4 z[1] = {make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv)};
    attn_put<1>(R.out, R.out_kind, R.in_scale, z, [&](int) { return orow * D + d; });
}

// ---- host ---------------------------------------------------------------------------------------------

struct AttnPlan {
    int rt;         // row tiles of a block
    int64_t tiles;  // blocks' row ranges, an upper bound over the batch
    int per_seq;    // tiles is this many for every sequence (0: less)
    bool by_xcd;
    int splits, key_groups;
    size_t bytes;
};

// Row tiles of a block (kRows rows of a sequence or fewer: 1). Blocks of one need no barrier and run two to a
// CU where LDS holds two; blocks of more share each key tile's loads. Measured with 1, 2 and 4 (us; int8 of 256 with
// 1 and 2):
//   int8, head_dim 64 and 128: 1. 2048 tokens, 32 heads on 8, on 4096 keys: 140, 171, 152 and 214, 261, 254.
//   int8, head_dim 256, 8 heads on 1: 2 where a block then has 4096 keys or more of its own, else 1. 8192 tokens on
//     their own 407, 402; 2048 on 8192 keys 173, 163; 16 x 512 on up to 4600 389, 374; 4096 on their own 124, 126;
//     2048 45, 47; 300 on 8300 keys 47, 60; 64 x 64 on up to 2064 62, 80; 32 x 8 on up to 4096 26, 28;
//     1000 tokens, window 512, 30, 37; 100 on 1100 keys 18, 20.
//   f16: 4 where that gives every second CU a block, so that the keys are split in two at most, for the parts'
//     way through memory costs more from there on. head_dim 256, 8 heads on 1: 8192 tokens 555, 580, 402; 2048 on
//     8192 keys 226, 245, 168; head_dim 128, 2048 tokens, 32 heads on 8, 197, 196, 181; head_dim 64 111, 116, 103.
//   f16 otherwise: 2 at head_dim 256, where LDS holds one block a CU anyway (512 tokens, window 512, 27, 20,
//     28; 16 x 64 tokens 40, 29, 40), else 1 (300 tokens, 16 heads on 4, head_dim 128: 20, 26, 22).
static int row_tiles(bool i8, int d, int64_t rows, int64_t keys, int64_t blocks2, int64_t blocks4) {
    const int64_t cus = device_cu_count();
    if (rows <= kRows) return 1;
    if (i8) return d == 256 && keys * std::min(blocks2, cus) >= 4096 * cus ? 2 : 1;
    if (blocks4 * 2 >= cus) return 4;
    return d == 256 ? 2 : 1;
}

static int key_groups(int rt, bool i8) { return rt == 1 || (rt == 2 && i8) ? 4 : 2; }

static AttnPlan attn_plan(const PagedArgs &A, const g4_kv_pages *pages, int heads, int window) {
    const int group = heads / A.kv_heads, d = pages->head_dim;
    AttnPlan P;
    const int64_t most = (int64_t)A.max_q * group;  // rows of a sequence
    const bool i8 = pages->kind == G4_KIND_I8;
    auto tiles = [&](int rows, bool *even) {  // of `rows` rows, at most; even: that is every sequence's most
        const int64_t each = (most + rows - 1) / rows * A.seqs, ragged = (int64_t)A.tokens * group / rows + A.seqs;
        if (even) *even = each <= ragged;
        return std::min(each, ragged);
    };
    auto keys_of = [&](int rows) -> int64_t {
        return window ? std::min<int64_t>(A.max_kv, (int64_t)window + kKeys + rows / group + 1) : A.max_kv;
    };
    P.rt = row_tiles(i8, d, most, keys_of(2 * kRows), tiles(2 * kRows, nullptr) * A.kv_heads,
                     tiles(4 * kRows, nullptr) * A.kv_heads);
    P.key_groups = key_groups(P.rt, i8);
    const int rows = kRows * P.rt;
    bool even;
    P.tiles = tiles(rows, &even);
    P.per_seq = even ? (int)((most + rows - 1) / rows) : 0;
    P.by_xcd = P.per_seq > 1 && A.seqs >= 8;
    if (P.by_xcd) P.tiles = P.per_seq * (((int64_t)A.seqs + 7) & ~7);
    const int64_t keys = keys_of(rows);
    const int64_t rounds = (keys + P.key_groups * kKeys - 1) / (P.key_groups * kKeys);
    // the keys are split until every CU has the blocks that it runs at once (32 x 8 tokens on up to 4096 keys and 512
    // tokens, window 512: 29 and 20 us; with half the splits 34 and 21, with twice as many 39 and 29)
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
    if constexpr (CK == G4_KIND_F16) {
        if (P.rt == 4) launch_rows<D, CK, 4>(A, R, P, stream);
    }
    if constexpr (D == 256) {
        if (P.rt == 2) launch_rows<D, CK, 2>(A, R, P, stream);
    }
    if (P.rt == 1) launch_rows<D, CK, 1>(A, R, P, stream);
    G4_LAUNCHED("attn_kernel");
    if (P.splits > 1) {
        const int rows = kRows * P.rt;
        // four thread groups a row from 8 splits on: a call with 32 splits 13.7 us (one group 19.2), with 8 26.6 and 98.3
        // (26.2 and 99.1), with 4 23.0 (20.1)
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

constexpr int kMaxTiles = 1 << 22;  // times 512 threads, which a grid's x axis holds

// `window` on return: 0 where it hides nothing.
static int attn_check(const g4_kv_pages *pages, const g4_chunk *chunk, int heads, int &window, PagedArgs *A) {
    if (int st = paged_args("attention-chunk", pages, chunk, A)) return st;
    if (heads <= 0 || heads % A->kv_heads)
        return set_error(G4_ERR_INVALID, "attention-chunk: %d query heads do not divide over %d KV heads", heads, A->kv_heads);
    if (window < 0) return set_error(G4_ERR_INVALID, "attention-chunk: window %d", window);
    if ((int64_t)A->tokens * heads > ((int64_t)1 << 30) || A->kv_heads > 65535)
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: more than 2^30 query rows, or 65535 KV heads");
    if (A->max_kv > 1 << 30)
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: max_kv %d is over 2^30 positions", A->max_kv);
    if (A->page_stride > INT32_MAX || A->slot_stride * pages->page_size > INT32_MAX)
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: pages, or a page's slots, 2^31 or more elements apart");
    window = effective_window(window, A->max_kv);
    return G4_OK;
}

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_attention_chunk_workspace_bytes(const g4_kv_pages *pages, const g4_chunk *chunk, int heads,
                                          int window) {
    PagedArgs A;
    if (attn_check(pages, chunk, heads, window, &A)) return 0;
    const AttnPlan P = attn_plan(A, pages, heads, window);
    return P.tiles > kMaxTiles ? 0 : P.bytes;
}

int g4_attention_chunk(const g4_kv_pages *pages, const g4_chunk *chunk, const void *q, int64_t q_stride,
                       int heads, float scale, int window, void *workspace, size_t workspace_bytes,
                       void *out, int out_kind, float in_scale, void *stream) {
    PagedArgs A;
    if (int st = attn_check(pages, chunk, heads, window, &A)) return st;
    if (!q || !out || !workspace) return set_error(G4_ERR_INVALID, "attention-chunk needs q, an output and a workspace");
    if (out_kind != G4_KIND_F16 && out_kind != G4_KIND_F32 && out_kind != G4_KIND_I8)
        return set_error(G4_ERR_INVALID, "attention-chunk: outputs are f16, f32 or int8 codes, got kind %d", out_kind);
    if (!std::isfinite(scale * 2.0f))
        return set_error(G4_ERR_INVALID, "attention-chunk: the scale must be finite and below 2^127");
    if (out_kind == G4_KIND_I8 && in_scale == 0.0f)
        return set_error(G4_ERR_INVALID, "attention-chunk: int8 codes need the consumer's inScale");
    const int64_t qw = (int64_t)heads * pages->head_dim;
    if (q_stride && (q_stride < qw || q_stride % 8))
        return set_error(G4_ERR_INVALID, "attention-chunk: q_stride must hold a row and be a multiple of 8");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return set_error(G4_ERR_INVALID, "attention-chunk: q, the output and the workspace must be 16-byte aligned");
    const AttnPlan P = attn_plan(A, pages, heads, window);
    if (P.tiles > kMaxTiles)
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: more than %d blocks of query rows", kMaxTiles);
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
    if (P.per_seq) R.per_seq = FastDiv::of(P.per_seq);
    R.by_xcd = P.by_xcd;
    // a scale of 0 as one too small to matter, so that a masked score stays minus infinity
    R.scale2 = std::max(std::fabs(scale) * 1.44269504088896340736f, 0x1p-126f);
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
