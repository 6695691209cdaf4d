// Low-rank adapters of a batch's requests beside a shared linear (include/g4serve.h):
//   out[t] = base[t] + scale_a (x[t] A_a^T) B_a^T.
//
// The rows are grouped by adapter once a step (adapter_groups_kernel): a tile is up to 16 rows of one adapter, so that
// a matrix instruction's other operand is that adapter's. Both products are transposed, the adapter's rows by the
// batch's: what a lane holds of H = x A^T, four ranks of one row, is its operand of the second product, and there it has
// runs of consecutive outputs of one row.
//
// Few rows: one launch, every block computes its tile's H for itself. Many: H in f32 by tile pair and range of K, then
// a block per tile and range of outputs, which adds up H's parts.
//
// A, x and B come to LDS in whole lines. A matrix instruction's operands straight from memory are 16 rows' 64 bytes a
// load, which a CU's first-level cache gives at 16 bytes a cycle; whole lines at 58 (2048 rows, K 6144, N 1536, rank 64: 27
// us, and 20.4).
//
// Bound, of one launch: a chain of loads (tile, rows, x and A, B beside them), the product, the stores: 6.6 us for a row of
// K 1536, N 2048, rank 16. Of two, at those 2048 rows: the first takes 10.2 us by its waits, 56% of its waves' cycles (the
// matrix units are busy for 4%, LDS for 9%, and a CU's 0.4 MB would come in 3 us): header, tile and rows one after the other,
// then chunks of 48 KB, two on their way at a time; the second reads base and writes, 19 MB in 11 us, most of it the
// chain's.
#include "g4_internal.h"
#include "../../include/g4serve.h"

namespace g4 {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 16;          // rows of a tile
constexpr int kMaxRank = 128, kMaxAdapters = 4096, kMaxK = 1 << 23, kMaxN = 1 << 30;  // rows are counted in 32 bits
constexpr int kMaxTokens = 1 << 19;  // a grid has a row of blocks per tile
constexpr int kGroupThreads = 1024;
// One launch, where every block makes its tile's H again, saves the second launch and H's way through memory, 2 to 3.5 us.
// It pays up to these bounds (in one launch and in two):
//   blocks a CU: f16 x, K 1536, N 6144, rank 32, 256 rows (396 blocks) 8.2 and 11.6 us; 512 rows (588) 15.7 and 13.7
//   row pairs that a wave loads: f16, 1 row, rank 32, K 3584 (42) 9.8 and 10.4 us; K 6144 (72) 12.7 and 9.3
//   cycles of a SIMD's matrix unit, where f32 x takes 16 times f16's: 64 rows, K 1536, rank 32 (6144) 12.1 and 12.5 us;
//   K 2048, rank 24 (8192) 13.3 and 11.5
constexpr int kFusedBlocks = 2, kFusedLoads = 48, kFusedCycles = 6500;
// Two launches: the ranges of K whose parts of H the second one adds up. 1 row, K 6144, rank 64, f16: 4 ranges 14.4 us, 8 12.3,
// 16 12.7. f32's products take longer: 64 rows, 8 ranges 22.6, 16 20.4.
constexpr int kSplits = 8, kSplitsF32 = 16;

// groups: the header, then the tiles.
struct GroupHeader {
    int tiles, tokens, adapters, pad;
};
struct GroupTile {
    int adapter, first, rows, pad;  // adapter -1: none; first: rows in the tiles before it
    int row[kTile];                 // here and not in a list of their own: a load less on every block's way
};

static int64_t max_tiles(int64_t tokens, int64_t adapters) {
    return tokens / kTile + (tokens < adapters + 1 ? tokens : adapters + 1);
}
static_assert(kMaxTokens / kTile + kMaxAdapters + 1 <= 65535, "tiles of a grid");
static size_t groups_bytes_of(int64_t tokens, int64_t adapters) {
    return sizeof(GroupHeader) + max_tiles(tokens, adapters) * sizeof(GroupTile);
}

// One block. Where a row stands in its group changes no result.
__global__ __launch_bounds__(kGroupThreads) void adapter_groups_kernel(const int32_t *row_adapter, int tokens, int adapters,
                                                                       GroupHeader *header, GroupTile *tiles) {
    extern __shared__ int32_t group_lds[];  // group 0: no adapter
    __shared__ int2 sums[kGroupThreads / 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, groups = adapters + 1;
    int32_t *count = group_lds, *first_tile = group_lds + groups;
    for (int i = t; i < groups; i += kGroupThreads) count[i] = 0;
    __syncthreads();
    auto group_of = [&](int row) {
        const int a = row < tokens ? row_adapter[row] : -2;
        return a == -2 ? -1 : (unsigned)a < (unsigned)adapters ? a + 1 : 0;
    };
    // Where many of a wave's rows have the first one's group, as in a prompt, those are counted together: additions to one
    // address wait for each other (2048 rows of 4 groups in runs 5.1 us and each row by itself 7.3; all others so: 4096
    // rows of 64 groups at random 6.4 us, group by group 50).
    auto place = [&](int g) {
        int mine = 0;
        const unsigned long long real = __ballot(g >= 0);
        if (!real) return 0;
        const int leader = __ffsll((long long)real) - 1;
        unsigned long long same = __ballot(g == __builtin_amdgcn_readlane(g, leader));
        if (__popcll(same) < 16) same = 0;
        if (same >> lane & 1) {
            if (lane == leader) mine = atomicAdd(&count[g], (int)__popcll(same));
            mine = __builtin_amdgcn_readlane(mine, leader) + (int)__popcll(same & ((1ull << lane) - 1));
        } else if (g >= 0) {
            mine = atomicAdd(&count[g], 1);
        }
        return mine;
    };
    for (int row = t; row - lane < tokens; row += kGroupThreads) place(group_of(row));
    __syncthreads();
    // every group's first tile and first row; a thread has a run of groups
    const int per = (groups + kGroupThreads - 1) / kGroupThreads, g0 = min(t * per, groups), g1 = min(g0 + per, groups);
    int2 mine = make_int2(0, 0);
    for (int g = g0; g < g1; ++g) {
        mine.x += count[g];
        mine.y += (count[g] + kTile - 1) / kTile;
    }
    int2 run = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int x = __shfl_up(run.x, s), y = __shfl_up(run.y, s);
        if (lane >= s) {
            run.x += x;
            run.y += y;
        }
    }
    if (lane == 63) sums[wave] = run;
    __syncthreads();
    int2 at = make_int2(run.x - mine.x, run.y - mine.y);
    int all = 0;
    for (int w = 0; w < kGroupThreads / 64; ++w) {
        if (w < wave) {
            at.x += sums[w].x;
            at.y += sums[w].y;
        }
        all += sums[w].y;
    }
    for (int g = g0; g < g1; ++g) {
        const int n = count[g];
        count[g] = 0;
        first_tile[g] = at.y;
        for (int i = 0; i < n; i += kTile) {
            GroupTile &T = tiles[at.y++];
            T.adapter = g - 1;
            T.first = at.x + i;
            T.rows = min(n - i, kTile);
        }
        at.x += n;
    }
    if (t == 0) *header = {all, tokens, adapters, 0};
    __syncthreads();
    for (int row = t; row - lane < tokens; row += kGroupThreads) {
        const int g = group_of(row), i = place(g);
        if (g >= 0) tiles[first_tile[g] + i / kTile].row[i % kTile] = row;
    }
}

struct AdapterArgs {
    const _Float16 *a, *b;
    const float *scales;
    const int32_t *ranks;
    int64_t a_stride, b_stride;
    int max_rank, rank16, k, n, tokens, count;  // rank16: max_rank in whole 16s, H's row
    const GroupHeader *header;
    const GroupTile *tiles;
    const void *x, *base;
    void *out;
    int64_t x_stride, base_stride, out_stride;
    float x_scale, base_scale, out_scale;
    int base_kind, out_kind;
    int splits, k_range, vec;  // K in `splits` ranges; vec: eight outputs may be moved at once
    float *h;                           // [splits][tokens][rank16]
};

// How many tiles there are: none in groups of another batch, whose rows are not these.
__device__ __forceinline__ int tiles_of(const AdapterArgs &A) {
    const GroupHeader h = *A.header;
    return h.tokens == A.tokens && h.adapters == A.count ? h.tiles : 0;
}

// What a block needs to know of a tile; there is room for every block's, also where there are fewer tiles.
struct Tile {
    int index, adapter, first, rows;
};
__device__ __forceinline__ Tile tile_of(const AdapterArgs &A, int index) {
    const GroupTile &T = A.tiles[index];
    return {index, T.adapter, T.first, T.rows};
}
__device__ __forceinline__ int64_t row_of(const AdapterArgs &A, const Tile &T, int col) {
    return A.tiles[T.index].row[min(col, T.rows - 1)];
}

__device__ __forceinline__ int rank_of(const AdapterArgs &A, int adapter) {
    return A.ranks ? min(max(A.ranks[adapter], 0), A.max_rank) : A.max_rank;
}

// Eight elements of x as f32 or, where the type is exact in it, f16.
template <int XK>
struct XPart {
    h8 v;
};
template <>
struct XPart<G4_KIND_F32> {
    f4 v[2];
};

template <int XK>
__device__ __forceinline__ f4 product(h8 a, const XPart<XK> &x, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, x.v, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f4 product<G4_KIND_F32>(h8 a, const XPart<G4_KIND_F32> &x, f4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32((float)a[e], x.v[e / 4][e % 4], c, 0, 0, 0);
    return c;
}

// 16 (4) bytes a lane from memory to LDS at lds + 16 (4) * lane. Through asm, with waits of the kernel's own: the compiler
// would wait for every load before the next LDS read. Nothing else here uses M0.
__device__ __forceinline__ void dma16(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "memory", "m0");
}
// At most N of the wave's loads are still on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt holds 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
// Every wave's LDS reads and writes are done, and what each has waited for is there.
__device__ __forceinline__ void block_meet() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}

constexpr int kWaves = 8, kAdThreads = 64 * kWaves;
constexpr int kChunk = 32 * kWaves;  // of K: a step of a matrix instruction for each wave

// The ring through which chunks of A's and x's rows come: row r of A's 16 RT at 512 r, of x's 16 MT at X + r * XROW. A
// row's units of 16 bytes stand at their number XOR (r % 8), for reads of one unit of eight rows at a time.
template <int XK, int RT, int MT, int ROOM>
struct Ring {
    static constexpr int XROW = kChunk * (XK == G4_KIND_F32 ? 4 : XK == G4_KIND_F16 ? 2 : 1);
    static constexpr int X = RT * 16 * kChunk * 2, BYTES = X + MT * 16 * XROW;
    static constexpr int SLOTS = ROOM / BYTES < 8 ? ROOM / BYTES : 8;
    static constexpr int XLOADS = XK == G4_KIND_F16 ? MT : 2 * MT, LOADS = RT + XLOADS;  // of a wave and chunk
    static_assert(SLOTS >= 2 && (SLOTS - 2) * LOADS < 64, "one chunk is read, others are on their way");
};

// acc[i][r] += tile i's rows by A's rows r0 + 16 r .. over [k0, k1), a wave taking 32 of each chunk's 256. row: the rows of
// x of the lane's column. Loads never leave the matrices: places behind their ends read the last unit or row, and
// enter as 0.
template <int XK, int RT, int MT, int ROOM>
__device__ __forceinline__ void shrink(const AdapterArgs &A, const _Float16 *a, int rank, int r0, const int (&row)[MT], int k0,
                                       int k1, char *lds, f4 (&acc)[MT][RT]) {
    typedef Ring<XK, RT, MT, ROOM> G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, group = lane >> 4;
    const uint32_t lds0 = lds_address(lds);
    const int chunks = (k1 - k0 + kChunk - 1) / kChunk;
    if (chunks <= 0) return;
    // A's rows come by pairs; the lane's row and element of a chunk in each of its wave's loads
    const char *from[RT], *xfrom[G::XLOADS];
    int at[RT], xat[G::XLOADS];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = 2 * (wave * RT + i) + lane / 32;
        from[i] = reinterpret_cast<const char *>(a + (int64_t)min(r0 + r, A.max_rank - 1) * A.k);
        at[i] = 8 * (lane % 32 ^ r % 8);
    }
#pragma unroll
    for (int i = 0; i < G::XLOADS; ++i) {
        const int r = XK == G4_KIND_F16 ? 2 * (wave * MT + i) + lane / 32 : wave * 2 * MT + i;
        int token = row[0];
        if (MT == 1) {
            token = __shfl(row[0], r % 16);
        } else {
            const int t0 = __shfl(row[0], r % 16), t1 = __shfl(row[MT - 1], r % 16);
            token = r < 16 ? t0 : t1;
        }
        xfrom[i] = static_cast<const char *>(A.x) + token * A.x_stride * (G::XROW / kChunk);
        xat[i] = XK == G4_KIND_F16 ? 8 * (lane % 32 ^ r % 8) : XK == G4_KIND_F32 ? 4 * (lane ^ r % 8)
                                                                                 : 16 * (lane / 4 ^ r % 8) + 4 * (lane % 4);
    }
    auto issue = [&](int c) {
        const uint32_t slot = lds0 + c % G::SLOTS * G::BYTES;
        const int k = k0 + c * kChunk;
#pragma unroll
        for (int i = 0; i < RT; ++i) dma16(from[i] + 2 * (int64_t)min(k + at[i], A.k - 8), slot + (wave * RT + i) * 1024);
#pragma unroll
        for (int i = 0; i < G::XLOADS; ++i) {
            if (XK == G4_KIND_I8) {
                dma4(xfrom[i] + min(k + xat[i], A.k - 4), slot + G::X + (wave * 2 * MT + i) * 256);
            } else if (XK == G4_KIND_F16) {
                dma16(xfrom[i] + 2 * (int64_t)min(k + xat[i], A.k - 8), slot + G::X + (wave * MT + i) * 1024);
            } else {
                dma16(xfrom[i] + 4 * (int64_t)min(k + xat[i], A.k - 4), slot + G::X + (wave * 2 * MT + i) * 1024);
            }
        }
    };
    auto multiply_chunk = [&](int c) {
        const char *slot = lds + c % G::SLOTS * G::BYTES;
        const bool in = k0 + c * kChunk + 32 * wave + 8 * group < k1;
        XPart<XK> x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const char *p = slot + G::X + (16 * i + col) * G::XROW;
            if constexpr (XK == G4_KIND_F32) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const f4 v = *reinterpret_cast<const f4 *>(p + ((8 * wave + 2 * group + e) ^ col % 8) * 16);
                    x[i].v[e] = in ? v : f4{};
                }
            } else if constexpr (XK == G4_KIND_F16) {
                const h8 v = *reinterpret_cast<const h8 *>(p + ((4 * wave + group) ^ col % 8) * 16);
                x[i].v = in ? v : h8{};
            } else {
                uint2 q = *reinterpret_cast<const uint2 *>(p + ((2 * wave + group / 2) ^ col % 8) * 16 + group % 2 * 8);
                if (!in) q = make_uint2(0, 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i].v[e] = (_Float16)(float)(int8_t)((e < 4 ? q.x : q.y) >> (8 * (e % 4)));
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const h8 v = *reinterpret_cast<const h8 *>(slot + (16 * r + col) * (kChunk * 2) + ((4 * wave + group) ^ col % 8) * 16);
            const h8 w = in && r0 + 16 * r + col < rank ? v : h8{};
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][r] = product<XK>(w, x[i], acc[i][r]);
        }
    };
    if (chunks <= G::SLOTS) {  // all at once, and one wait
        for (int c = 0; c < chunks; ++c) issue(c);
        wait_loads<0>();
        block_meet();
        for (int c = 0; c < chunks; ++c) multiply_chunk(c);
    } else {
        for (int c = 0; c < G::SLOTS - 1; ++c) issue(c);
        for (int c = 0; c < chunks; ++c) {
            if (c + G::SLOTS - 2 < chunks) wait_loads<(G::SLOTS - 2) * G::LOADS>();
            else wait_loads<0>();
            block_meet();  // chunk c is there, and chunk c - 1 has been read
            if (c + G::SLOTS - 1 < chunks) issue(c + G::SLOTS - 1);
            multiply_chunk(c);
        }
    }
    block_meet();  // the ring is free
}

// The block's sum of the waves' acc, each tile's and rank tile's f4 by lane, at `part`.
template <int N>
__device__ __forceinline__ void sum_waves(const f4 (&acc)[N], f4 *part) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) part[(wave * N + i) * 64 + lane] = acc[i];
    __syncthreads();
    for (int i = t; i < N * 64; i += kAdThreads) {
        f4 s = part[i];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += part[w * N * 64 + i];
        part[i] = s;
    }
    __syncthreads();
}

__device__ __forceinline__ f4 multiply(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 multiply(h4 a, h4 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }

// Eight consecutive elements of a row of `kind`, `n` of which exist (one at least), as they come: packed (vec), or each in
// a word of its own. Nothing waits for them here.
struct Raw8 {
    u32x4 a, b;  // whole vectors in every branch: an array that branches fill in part would be kept in memory
    __device__ __forceinline__ void load(const void *p, int kind, int64_t at, int n, bool vec) {
        b = u32x4{};
        if (vec) {
            if (kind == G4_KIND_F32) {
                const u32x4 *q = reinterpret_cast<const u32x4 *>(static_cast<const float *>(p) + at);
                a = q[0];
                b = q[1];
            } else if (kind == G4_KIND_F16) {
                a = *reinterpret_cast<const u32x4 *>(static_cast<const _Float16 *>(p) + at);
            } else {
                const uint2 c = *reinterpret_cast<const uint2 *>(static_cast<const int8_t *>(p) + at);
                a = u32x4{c.x, c.y, 0, 0};
            }
        } else if (kind == G4_KIND_F32) {
            words(static_cast<const uint32_t *>(p) + at, n);
        } else if (kind == G4_KIND_F16) {
            words(static_cast<const uint16_t *>(p) + at, n);
        } else {
            words(static_cast<const uint8_t *>(p) + at, n);
        }
    }
    template <class T>
    __device__ __forceinline__ void words(const T *p, int n) {
        a = u32x4{p[0], p[min(1, n - 1)], p[min(2, n - 1)], p[min(3, n - 1)]};
        b = u32x4{p[min(4, n - 1)], p[min(5, n - 1)], p[min(6, n - 1)], p[min(7, n - 1)]};
    }
    __device__ __forceinline__ void values(int kind, bool vec, float scale, float (&y)[8]) const {
        if (kind == G4_KIND_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(e < 4 ? a[e % 4] : b[e % 4]);
        } else if (kind == G4_KIND_F16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = vec ? a[e / 2] >> (16 * (e % 2)) : e < 4 ? a[e % 4] : b[e % 4];
                y[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)h);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[e] = (float)(int8_t)(vec ? a[e / 4] >> (8 * (e % 4)) : e < 4 ? a[e % 4] : b[e % 4]) * scale;
        }
    }
};

__device__ __forceinline__ void store8(void *p, int kind, int64_t at, int n, bool vec, const float (&v)[8], float snap) {
    if (kind == G4_KIND_I8) {
        int8_t *q = static_cast<int8_t *>(p) + at;
        uint2 c = make_uint2(0, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) (e < 4 ? c.x : c.y) |= (uint32_t)(uint8_t)srq_code_i(v[e], snap) << (8 * (e % 4));
        if (vec) {
            *reinterpret_cast<uint2 *>(q) = c;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) q[e] = (int8_t)((e < 4 ? c.x : c.y) >> (8 * (e % 4)));
        }
        return;
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = snap != 0.0f ? srq_code_f(v[e], snap) * snap : v[e];
    if (kind == G4_KIND_F16) {
        _Float16 *q = static_cast<_Float16 *>(p) + at;
        h8 c;
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = (_Float16)y[e];
        if (vec) {
            *reinterpret_cast<h8 *>(q) = c;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) q[e] = c[e];
        }
    } else {
        float *q = static_cast<float *>(p) + at;
        if (vec) {
            reinterpret_cast<f4 *>(q)[0] = f4{y[0], y[1], y[2], y[3]};
            reinterpret_cast<f4 *>(q)[1] = f4{y[4], y[5], y[6], y[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) q[e] = y[e];
        }
    }
}

constexpr int kWaveN = 64, kBlockN = kWaves * kWaveN;  // outputs of a wave, and of a block

// B's rows n0 .. n0 + 511 at `lds`, max_rank halves each; loads of whole lines (see Ring). A row's units of 16 bytes
// stand at their number XOR unit_xor(row): a product's lanes read one unit of rows 0-3 and 8-11 at a time.
__device__ __forceinline__ int unit_xor(int row, int units) {
    return units == 8 || units == 16 ? (row & 3) | (row >> 1 & 4)
           : units == 4              ? (row >> 1 & 1) | (row >> 2 & 2)
           : units == 2              ? row >> 3 & 1
                                     : 0;
}
__device__ __forceinline__ void load_b(const AdapterArgs &A, const _Float16 *b, int n0, char *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, units = A.max_rank / 8;
    const uint32_t lds0 = lds_address(lds), by_units = 0xffffffffu / units + 1;
    for (int i = 0; i < units; ++i) {
        const int place = (wave * units + i) * 64 + lane, row = units == 1 ? place : (int)__umulhi(place, by_units);
        const int unit = (place - row * units) ^ unit_xor(row, units);
        dma16(b + (int64_t)min(n0 + row, A.n - 1) * A.max_rank + 8 * unit, lds0 + (wave * units + i) * 1024);
    }
}

// A wave's 64 outputs of a tile's rows. Tile j of the product has the outputs n0 + 32 (j / 2) + 8 q + 4 (j % 2) + e,
// q its row's group and e its place there, so that a lane has eight consecutive outputs in each pair of tiles.
template <int RT>
struct Expand {
    // A lane's ranks of a product: eight consecutive ones of 32, or four of 16 where there are no more.
    static constexpr int kRanks = RT == 1 ? 4 : 8, kSteps = RT == 1 ? 1 : RT / 2;
    typedef _Float16 hr __attribute__((ext_vector_type(kRanks)));
    Raw8 raw[2];
    int n0;

    // Loads the wave's part of base.
    __device__ __forceinline__ void load(const AdapterArgs &A, const Tile &T, int64_t row, int n) {
        const int lane = threadIdx.x & 63, col = lane & 15, group = lane >> 4;
        n0 = n;
        if (!A.base || col >= T.rows) return;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int out = n0 + 32 * p + 8 * group, left = A.n - out;
            if (left > 0) raw[p].load(A.base, A.base_kind, row * A.base_stride + out, left, A.vec);
        }
    }

    // h: the tile's H in LDS, as the first product leaves it, [rank tile][lane], a lane's four ranks of its row; b: of
    // load_b. H enters the product as the sum of two f16 values, relative to the row's largest: off by 2^-23 of itself,
    // as by two roundings to f32.
    __device__ __forceinline__ void finish(const AdapterArgs &A, const Tile &T, const f4 *h, const char *b, int rank, float scale,
                                           int64_t row) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, group = lane >> 4;
        f4 acc[4] = {f4{}, f4{}, f4{}, f4{}};
        float back = 1.0f;
        if (rank > 0) {
            float v[kSteps][kRanks];
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int at = kRanks * (4 * s + group);
#pragma unroll
                for (int e = 0; e < kRanks; e += 4) {
                    const f4 o = at + e < rank ? h[(at + e) / 16 * 64 + (at + e) / 4 % 4 * 16 + col] : f4{};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // (an infinite x leaves NaN behind the rank)
                        v[s][e + i] = at + e + i < rank ? o[i] : 0.0f;
                        top = fmaxf(top, fabsf(v[s][e + i]));
                    }
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // the largest to [2^14, 2^15) of f16's 65504
            int up = 141 - (int)(__float_as_uint(top) >> 23);
            up = min(max(up, -120), 120);
            const float to = __uint_as_float((uint32_t)(127 + up) << 23);
            back = __uint_as_float((uint32_t)(127 - up) << 23);
            const int units = A.max_rank / 8;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                if (4 * kRanks * s >= rank) break;
                const int at = kRanks * (4 * s + group);
                hr hi, lo;
#pragma unroll
                for (int e = 0; e < kRanks; ++e) {
                    const float o = v[s][e] * to;
                    hi[e] = (_Float16)o;
                    lo[e] = (_Float16)(o - (float)hi[e]);
                }
                if (__any(top == INFINITY)) lo = top == INFINITY ? hr{} : lo;  // an infinite H stays one
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = wave * kWaveN + 32 * (j / 2) + 8 * (col / 4) + 4 * (j % 2) + col % 4;
                    hr w{};
                    if (at < A.max_rank)
                        w = *reinterpret_cast<const hr *>(b + (r * units + (at / 8 ^ unit_xor(r, units))) * 16 + at % 8 * 2);
#pragma unroll
                    for (int e = 0; e < kRanks; ++e) w[e] = at + e < rank ? w[e] : (_Float16)0.0f;
                    acc[j] = multiply(w, hi, acc[j]);
                    acc[j] = multiply(w, lo, acc[j]);
                }
            }
        }
        if (col >= T.rows) return;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int out = n0 + 32 * p + 8 * group, left = A.n - out;
            if (left <= 0) continue;
            float y[8] = {};
            if (A.base) raw[p].values(A.base_kind, A.vec, A.base_scale, y);
            if (rank > 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] += scale * (acc[2 * p + e / 4][e % 4] * back);  // (scale * back may be out of range)
            }
            store8(A.out, A.out_kind, row * A.out_stride + out, left, A.vec, y, A.out_scale);
        }
    }
};

__device__ __forceinline__ float scale_of(const AdapterArgs &A, int adapter) {
    return adapter < 0 ? 0.0f : (A.scales ? A.scales[adapter] : 1.0f) * A.x_scale;
}

constexpr int kLds = 144 << 10;  // what a block takes of a CU's 160 KB

// Grid (ranges of 512 outputs, tiles): H, then the outputs.
template <int XK, int RT>
__global__ __launch_bounds__(kAdThreads) void adapter_fused_kernel(AdapterArgs A) {
    constexpr int kRoom = kLds - RT * 16 * kBlockN * 2;
    typedef Ring<XK, RT, 1, kRoom> G;
    __shared__ __align__(1024) char lds[G::SLOTS * G::BYTES], b_lds[RT * 16 * kBlockN * 2];
    static_assert(G::SLOTS * G::BYTES >= kWaves * RT * 64 * (int)sizeof(f4), "the waves' sums take the ring's place");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15;
    const Tile T = tile_of(A, blockIdx.y);
    const int tiles = tiles_of(A);
    if ((int)blockIdx.y >= tiles) return;
    const int row[1] = {(int)row_of(A, T, col)};
    const bool some = T.adapter >= 0;
    const _Float16 *b = A.b + max(T.adapter, 0) * A.b_stride;
    const int n = blockIdx.x * kBlockN;
    Expand<RT> E;
    E.load(A, T, row[0], n + wave * kWaveN);
    if (some) load_b(A, b, n, b_lds);
    const int rank = some ? rank_of(A, T.adapter) : 0;
    const float scale = scale_of(A, T.adapter);
    f4 *const h = reinterpret_cast<f4 *>(lds);
    if (some) {
        f4 acc[1][RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[0][r] = f4{};
        shrink<XK, RT, 1, kRoom>(A, A.a + T.adapter * A.a_stride, rank, 0, row, 0, A.k, lds, acc);
        sum_waves<RT>(acc[0], h);
    }
    E.finish(A, T, h, b_lds, rank, scale, row[0]);
}

// Grid (splits, pairs of tiles, ranks by 64): a range of K of the tiles' H. Two tiles of one adapter share its rows of A.
template <int XK, int RT>
__global__ __launch_bounds__(kAdThreads) void adapter_shrink_kernel(AdapterArgs A) {
    typedef Ring<XK, RT, 2, kLds> G;
    typedef Ring<XK, RT, 1, kLds> One;
    constexpr int kRing = G::SLOTS * G::BYTES > One::SLOTS * One::BYTES ? G::SLOTS * G::BYTES : One::SLOTS * One::BYTES;
    constexpr int kSums = kWaves * 2 * RT * 64 * (int)sizeof(f4);
    __shared__ __align__(1024) char lds[kRing > kSums ? kRing : kSums];
    const int t = threadIdx.x, lane = t & 63, col = lane & 15, r0 = 64 * blockIdx.z;
    const int first = 2 * blockIdx.y, tiles = min(tiles_of(A) - first, 2);
    if (tiles <= 0) return;
    const Tile T0 = tile_of(A, first), T1 = tile_of(A, tiles > 1 ? first + 1 : first);
    const int k0 = blockIdx.x * A.k_range, k1 = min(k0 + A.k_range, A.k);
    f4 acc[2][RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[0][r] = acc[1][r] = f4{};
    const int row[2] = {(int)row_of(A, T0, col), (int)row_of(A, T1, col)};
    if (T0.adapter == T1.adapter) {
        if (T0.adapter < 0) return;
        shrink<XK, RT, 2, kLds>(A, A.a + T0.adapter * A.a_stride, rank_of(A, T0.adapter), r0, row, k0, k1, lds, acc);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int adapter = i ? T1.adapter : T0.adapter;
            if (adapter < 0) continue;
            const int alone[1] = {row[i]};
            f4 mine[1][RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) mine[0][r] = f4{};
            shrink<XK, RT, 1, kLds>(A, A.a + adapter * A.a_stride, rank_of(A, adapter), r0, alone, k0, k1, lds, mine);
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[i][r] = mine[0][r];
        }
    }
    f4 both[2 * RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        both[r] = acc[0][r];
        both[RT + r] = acc[1][r];
    }
    f4 *const part = reinterpret_cast<f4 *>(lds);
    sum_waves<2 * RT>(both, part);
    for (int i = t; i < tiles * RT * 64; i += kAdThreads) {
        const bool second = i >= RT * 64;
        const int r = r0 + i / 64 % RT * 16, l = i & 63, place = (second ? T1.first : T0.first) + (l & 15);
        if ((l & 15) < (second ? T1.rows : T0.rows) && r < A.rank16)
            *reinterpret_cast<f4 *>(A.h + ((int64_t)blockIdx.x * A.tokens + place) * A.rank16 + r + 4 * (l >> 4)) = part[i];
    }
}

// Grid (ranges of 512 outputs, tiles).
template <int RT>
__global__ __launch_bounds__(kAdThreads) void adapter_expand_kernel(AdapterArgs A) {
    __shared__ f4 h[RT * 64];
    __shared__ __align__(1024) char b_lds[RT * 16 * kBlockN * 2];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 15, n = blockIdx.x * kBlockN;
    const Tile T = tile_of(A, blockIdx.y);
    const int tiles = tiles_of(A);
    if ((int)blockIdx.y >= tiles) return;
    const int64_t row = row_of(A, T, col);
    const bool some = T.adapter >= 0;
    if (some) load_b(A, A.b + T.adapter * A.b_stride, n, b_lds);
    Expand<RT> E;
    E.load(A, T, row, n + wave * kWaveN);
    const int rank = some ? rank_of(A, T.adapter) : 0;
    const float scale = scale_of(A, T.adapter);
    if (some) {
        for (int i = t; i < RT * 64; i += kAdThreads) {
            const int r = i >> 6, l = i & 63;
            if (16 * r >= A.rank16) break;
            const float *p = A.h + (int64_t)(T.first + min(l & 15, T.rows - 1)) * A.rank16 + 16 * r + 4 * (l >> 4);
            f4 s{};
#pragma unroll 8
            for (int j = 0; j < A.splits; ++j) s += *reinterpret_cast<const f4 *>(p + (int64_t)j * A.tokens * A.rank16);
            h[i] = s;
        }
        wait_loads<0>();
        block_meet();
    }
    E.finish(A, T, h, b_lds, rank, scale, row);
}

// How a call is run: in one launch (splits 0), or with H's parts of `splits` ranges of K. By the most tiles that the rows can
// make of the pool's adapters: how many they make is known on the device only. Rows of few adapters of a large pool pay for
// it: 512 rows of 4, K 6144, N 1536, rank 64 take 15.1 us of a pool of 4, 17.0 of 64, 26.3 of 256 or more (one range of K);
// 2048 rows 24.5, 24.4, 30.8; 64 rows of 16, K 1536, N 6144, rank 32 8.9 us of 16, 11.1 of 64 or more (two launches).
static int adapter_splits(const g4_adapters *D, int tokens, int x_size) {
    const int64_t tiles = max_tiles(tokens, D->count), blocks = tiles * ((D->n + kBlockN - 1) / kBlockN);
    const int64_t ranks = (D->max_rank + 15) / 16, room = ranks > 2 ? 4 : ranks;  // by 16, and what a kernel has of them
    const int64_t chunks = (D->k + kChunk - 1) / kChunk, loads = chunks * (room + (x_size == 2 ? 1 : 2));
    const int64_t cycles = (int64_t)(D->k / 32) * room * (x_size == 4 ? 256 : 16) / 4;
    if (ranks <= (x_size == 4 ? 2 : 4) && blocks <= kFusedBlocks * device_cu_count() && loads <= kFusedLoads &&
        cycles <= kFusedCycles)
        return 0;
    const int64_t pairs = (tiles + 1) / 2;
    const int64_t most = x_size == 4 ? kSplitsF32 : kSplits;
    int64_t want = device_cu_count() / (pairs * ((D->max_rank + 63) / 64));  // a block a CU at once
    want = want < 1 ? 1 : want > most ? most : want;
    const int64_t each = (chunks + want - 1) / want;
    return (int)((chunks + each - 1) / each);
}

template <int XK>
static int launch_fused(const AdapterArgs &A, dim3 grid, hipStream_t s) {
    const dim3 block(kAdThreads);
    if (A.rank16 <= 16) hipLaunchKernelGGL((adapter_fused_kernel<XK, 1>), grid, block, 0, s, A);
    else if (A.rank16 <= 32) hipLaunchKernelGGL((adapter_fused_kernel<XK, 2>), grid, block, 0, s, A);
    else if constexpr (XK != G4_KIND_F32) hipLaunchKernelGGL((adapter_fused_kernel<XK, 4>), grid, block, 0, s, A);
    G4_LAUNCHED("adapter_fused_kernel");
    return G4_OK;
}

template <int XK>
static int launch_shrink(const AdapterArgs &A, dim3 grid, hipStream_t s) {
    const dim3 block(kAdThreads);
    if (A.rank16 <= 16) hipLaunchKernelGGL((adapter_shrink_kernel<XK, 1>), grid, block, 0, s, A);
    else if (A.rank16 <= 32) hipLaunchKernelGGL((adapter_shrink_kernel<XK, 2>), grid, block, 0, s, A);
    else hipLaunchKernelGGL((adapter_shrink_kernel<XK, 4>), grid, block, 0, s, A);
    G4_LAUNCHED("adapter_shrink_kernel");
    return G4_OK;
}

static int launch_expand(const AdapterArgs &A, dim3 grid, hipStream_t s) {
    const dim3 block(kAdThreads);
    if (A.rank16 <= 16) hipLaunchKernelGGL(adapter_expand_kernel<1>, grid, block, 0, s, A);
    else if (A.rank16 <= 32) hipLaunchKernelGGL(adapter_expand_kernel<2>, grid, block, 0, s, A);
    else if (A.rank16 <= 64) hipLaunchKernelGGL(adapter_expand_kernel<4>, grid, block, 0, s, A);
    else hipLaunchKernelGGL(adapter_expand_kernel<8>, grid, block, 0, s, A);
    G4_LAUNCHED("adapter_expand_kernel");
    return G4_OK;
}

static int check_adapters(const char *who, const g4_adapters *D) {
    if (!D || !D->a || !D->b) return set_error(G4_ERR_INVALID, "%s needs the adapters' A and B", who);
    if (D->count <= 0 || D->count > kMaxAdapters)
        return set_error(G4_ERR_INVALID, "%s: %d adapters (1 to %d)", who, D->count, kMaxAdapters);
    if (D->k <= 0 || D->k % 8 || D->k > kMaxK || D->n <= 0 || D->n > kMaxN)
        return set_error(G4_ERR_INVALID, "%s: k %d, n %d (k a multiple of 8 up to %d, n up to %d)", who, D->k, D->n, kMaxK, kMaxN);
    if (D->max_rank <= 0 || D->max_rank % 8 || D->max_rank > kMaxRank)
        return set_error(G4_ERR_INVALID, "%s: max_rank %d is not a multiple of 8 up to %d", who, D->max_rank, kMaxRank);
    if (((uintptr_t)D->a | (uintptr_t)D->b) & 15) return set_error(G4_ERR_INVALID, "%s: A and B must be 16-byte aligned", who);
    const int64_t a = (int64_t)D->max_rank * D->k, b = (int64_t)D->n * D->max_rank;
    if ((D->a_stride && (D->a_stride < a || D->a_stride % 8)) || (D->b_stride && (D->b_stride < b || D->b_stride % 8)))
        return set_error(G4_ERR_INVALID, "%s: adapter strides must hold an adapter and be multiples of 8", who);
    return G4_OK;
}

static int kind_size(int kind) { return kind == G4_KIND_F32 ? 4 : kind == G4_KIND_F16 ? 2 : 1; }
static bool is_kind(int kind) { return kind == G4_KIND_F32 || kind == G4_KIND_F16 || kind == G4_KIND_I8; }

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_adapter_groups_bytes(int tokens, int adapters) {
    if (tokens <= 0 || tokens > kMaxTokens || adapters <= 0 || adapters > kMaxAdapters) return 0;
    return groups_bytes_of(tokens, adapters);
}

int g4_adapter_groups(const int32_t *row_adapter, int tokens, int adapters, void *groups, size_t groups_bytes,
                      void *stream) {
    const size_t need = g4_adapter_groups_bytes(tokens, adapters);
    if (!need)
        return set_error(G4_ERR_INVALID, "adapter-groups: %d tokens, %d adapters (1 to %d, and to %d)", tokens, adapters,
                         kMaxTokens, kMaxAdapters);
    if (!row_adapter) return set_error(G4_ERR_INVALID, "adapter-groups needs row_adapter");
    if (!groups || groups_bytes < need)
        return set_error(G4_ERR_INVALID, "adapter-groups: groups %zu B < %zu B", groups_bytes, need);
    if ((uintptr_t)groups & 15) return set_error(G4_ERR_INVALID, "adapter-groups: groups must be 16-byte aligned");
    GroupHeader *h = static_cast<GroupHeader *>(groups);
    GroupTile *tiles = reinterpret_cast<GroupTile *>(h + 1);
    hipLaunchKernelGGL(adapter_groups_kernel, dim3(1), dim3(kGroupThreads), 2 * (adapters + 1) * sizeof(int32_t),
                       as_stream(stream), row_adapter, tokens, adapters, h, tiles);
    G4_LAUNCHED("adapter_groups_kernel");
    return G4_OK;
}

size_t g4_adapter_workspace_bytes(const g4_adapters *adapters, int tokens) {
    if (check_adapters("adapter-linear", adapters) || tokens <= 0 || tokens > kMaxTokens) return 0;
    // the most that any type of x takes; one launch takes none
    const int splits = adapter_splits(adapters, tokens, 4);
    return splits ? (size_t)splits * tokens * ((adapters->max_rank + 15) / 16 * 16) * sizeof(float) : 16;
}

int g4_adapter_linear(const g4_adapters *adapters, const void *groups, size_t groups_bytes, int tokens, const void *x,
                      int x_kind, int64_t x_stride, float x_scale, const void *base, int base_kind, int64_t base_stride,
                      float base_scale, void *out, int out_kind, int64_t out_stride, float out_scale, void *workspace,
                      size_t workspace_bytes, void *stream) {
    const g4_adapters *D = adapters;
    if (int st = check_adapters("adapter-linear", D)) return st;
    const size_t need_groups = g4_adapter_groups_bytes(tokens, D->count);
    if (!need_groups) return set_error(G4_ERR_INVALID, "adapter-linear: %d tokens (1 to %d)", tokens, kMaxTokens);
    if (!groups || groups_bytes < need_groups)
        return set_error(G4_ERR_INVALID, "adapter-linear: groups %zu B < %zu B", groups_bytes, need_groups);
    if (!x || !out) return set_error(G4_ERR_INVALID, "adapter-linear needs x and out");
    if (!is_kind(x_kind) || !is_kind(out_kind) || (base && !is_kind(base_kind)))
        return set_error(G4_ERR_INVALID, "adapter-linear: x, base and out are f32, f16 or int8 codes");
    if (out_kind == G4_KIND_I8 && out_scale == 0.0f)
        return set_error(G4_ERR_INVALID, "adapter-linear: int8 output codes need a calibrated outScale");
    if ((x_stride && x_stride < D->k) || (base && base_stride && base_stride < D->n) || (out_stride && out_stride < D->n))
        return set_error(G4_ERR_INVALID, "adapter-linear: a row stride is shorter than the row");
    const int64_t xs = x_stride ? x_stride : D->k, os = out_stride ? out_stride : D->n, bs = base_stride ? base_stride : D->n;
    if (((uintptr_t)x & 15) || (tokens > 1 && xs * kind_size(x_kind) % (x_kind == G4_KIND_I8 ? 8 : 16)))
        return set_error(G4_ERR_INVALID, "adapter-linear: x must be 16-byte aligned, its rows too (int8 codes: 8)");
    if (base == out && (base_kind != out_kind || bs != os))
        return set_error(G4_ERR_INVALID, "adapter-linear: out can be base only with its type and stride");
    if (((uintptr_t)groups | (uintptr_t)workspace) & 15)
        return set_error(G4_ERR_INVALID, "adapter-linear: groups and workspace must be 16-byte aligned");
    const size_t need = g4_adapter_workspace_bytes(D, tokens);
    if (!workspace || workspace_bytes < need)
        return set_error(G4_ERR_INVALID, "adapter-linear: workspace %zu B < %zu B", workspace_bytes, need);
    if (out == x) return set_error(G4_ERR_INVALID, "adapter-linear: out cannot be x, which every block of a row reads");
    if ((uintptr_t)groups < (uintptr_t)workspace + need && (uintptr_t)workspace < (uintptr_t)groups + need_groups)
        return set_error(G4_ERR_INVALID, "adapter-linear: groups and workspace overlap");
    const int64_t tiles = max_tiles(tokens, D->count);
    AdapterArgs A{};
    A.a = static_cast<const _Float16 *>(D->a);
    A.b = static_cast<const _Float16 *>(D->b);
    A.scales = D->scales;
    A.ranks = D->ranks;
    A.max_rank = D->max_rank;
    A.rank16 = (D->max_rank + 15) / 16 * 16;
    A.k = D->k;
    A.n = D->n;
    A.tokens = tokens;
    A.count = D->count;
    A.a_stride = D->a_stride ? D->a_stride : (int64_t)D->max_rank * D->k;
    A.b_stride = D->b_stride ? D->b_stride : (int64_t)D->n * D->max_rank;
    A.header = static_cast<const GroupHeader *>(groups);
    A.tiles = reinterpret_cast<const GroupTile *>(A.header + 1);
    A.x = x;
    A.x_stride = xs;
    A.x_scale = x_kind == G4_KIND_I8 ? x_scale : 1.0f;
    A.base = base;
    A.base_kind = base ? base_kind : G4_KIND_F32;
    A.base_stride = bs;
    A.base_scale = base_scale;
    A.out = out;
    A.out_kind = out_kind;
    A.out_stride = os;
    A.out_scale = out_scale;
    A.splits = adapter_splits(D, tokens, kind_size(x_kind));
    A.vec = D->n % 8 == 0 && os % 8 == 0 && (!base || bs % 8 == 0) && ((uintptr_t)out & 15) == 0 && ((uintptr_t)base & 15) == 0;
    A.h = static_cast<float *>(workspace);
    hipStream_t s = as_stream(stream);
    const dim3 out_grid((unsigned)((D->n + kBlockN - 1) / kBlockN), (unsigned)tiles);
    if (A.splits == 0) {
        if (x_kind == G4_KIND_I8) return launch_fused<G4_KIND_I8>(A, out_grid, s);
        if (x_kind == G4_KIND_F16) return launch_fused<G4_KIND_F16>(A, out_grid, s);
        return launch_fused<G4_KIND_F32>(A, out_grid, s);
    }
    A.k_range = ((D->k + kChunk - 1) / kChunk + A.splits - 1) / A.splits * kChunk;
    const dim3 grid(A.splits, (unsigned)((tiles + 1) / 2), (unsigned)((D->max_rank + 63) / 64));
    int st;
    if (x_kind == G4_KIND_I8) st = launch_shrink<G4_KIND_I8>(A, grid, s);
    else if (x_kind == G4_KIND_F16) st = launch_shrink<G4_KIND_F16>(A, grid, s);
    else st = launch_shrink<G4_KIND_F32>(A, grid, s);
    if (st) return st;
    return launch_expand(A, out_grid, s);
}

}  // extern "C"
