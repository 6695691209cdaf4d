// Low-rank adapters of a batch's requests beside a shared linear (include/g4serve.h):
//   out[t] = base[t] + scale_a (x[t] A_a^T) B_a^T.
//
// The rows are grouped by adapter once a step (adapter_groups_kernel): a tile is up to 16 rows of one adapter, so that
// a matrix instruction's other operand is that adapter's. Two launches a linear: (1) H = x A^T, a block per tile and
// range of K, partial sums in f32; (2) out = base + scale H B^T, a block per tile and range of N, which adds up H's
// partial sums. Both products transposed, the adapter's rows by the batch's: a lane then holds four consecutive
// outputs of one row. Operands come straight from global memory, each used by one wave.
#include "g4_internal.h"
#include "../../include/g4serve.h"

namespace g4 {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr int kAdThreads = 256, kAdWaves = 4;
constexpr int kTile = 16;          // rows of a tile
constexpr int kMaxRank = 128, kMaxAdapters = 4096;
constexpr int kMaxTokens = 1 << 19;  // a grid has a row of blocks per tile
constexpr int kGroupThreads = 1024;

// groups: the header, the tiles, then the rows by adapter.
struct GroupHeader {
    int tiles, tokens, adapters, pad;
};
struct GroupTile {
    int adapter, first, rows, pad;  // adapter -1: none; rows order[first ..]
};

static int64_t max_tiles(int64_t tokens, int64_t adapters) {
    return tokens / kTile + (tokens < adapters + 1 ? tokens : adapters + 1);
}
static_assert(kMaxTokens / kTile + kMaxAdapters + 1 <= 65535, "tiles of a grid");
static size_t groups_bytes_of(int64_t tokens, int64_t adapters) {
    return sizeof(GroupHeader) + max_tiles(tokens, adapters) * sizeof(GroupTile) + tokens * sizeof(int32_t);
}

// One block. Where a row stands in its group changes no result.
__global__ __launch_bounds__(kGroupThreads) void adapter_groups_kernel(const int32_t *row_adapter, int tokens, int adapters,
                                                                       GroupHeader *header, GroupTile *tiles,
                                                                       int32_t *order) {
    extern __shared__ int32_t group_lds[];  // [adapters + 1] counts, then places; group 0: no adapter
    __shared__ int2 sums[kGroupThreads / 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, groups = adapters + 1;
    for (int i = t; i < groups; i += kGroupThreads) group_lds[i] = 0;
    __syncthreads();
    auto group_of = [&](int row) {
        const int a = row < tokens ? row_adapter[row] : -2;
        return a == -2 ? -1 : (unsigned)a < (unsigned)adapters ? a + 1 : 0;
    };
    for (int row = t; row < tokens; row += kGroupThreads) {
        const int g = group_of(row);
        if (g >= 0) atomicAdd(&group_lds[g], 1);
    }
    __syncthreads();
    // every group's first row and first tile; a thread has a run of groups
    const int per = (groups + kGroupThreads - 1) / kGroupThreads, g0 = min(t * per, groups), g1 = min(g0 + per, groups);
    int2 mine = make_int2(0, 0);
    for (int g = g0; g < g1; ++g) {
        mine.x += group_lds[g];
        mine.y += (group_lds[g] + kTile - 1) / kTile;
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
        const int n = group_lds[g];
        group_lds[g] = at.x;
        for (int i = 0; i < n; i += kTile) tiles[at.y++] = {g - 1, at.x + i, min(n - i, kTile), 0};
        at.x += n;
    }
    if (t == 0) *header = {all, tokens, adapters, 0};
    __syncthreads();
    for (int row = t; row - lane < tokens; row += kGroupThreads) {
        const int g = group_of(row);
        // a wave's rows of one group stand together
        unsigned long long left = __ballot(g >= 0);
        while (left) {
            const int leader = __ffsll((long long)left) - 1;
            const unsigned long long same = __ballot(g == __shfl(g, leader));
            if (same >> lane & 1) {
                int place = 0;
                if (lane == leader) place = atomicAdd(&group_lds[g], (int)__popcll(same));
                place = __shfl(place, leader);
                order[place + __popcll(same & ((1ull << lane) - 1))] = row;
            }
            left &= ~same;
        }
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
    const int32_t *order;
    const void *x;
    int64_t x_stride;
    const void *base;
    int64_t base_stride;
    float x_scale, base_scale, out_scale;
    void *out;
    int64_t out_stride;
    int splits, range, vec;  // K in `splits` ranges of `range`; vec: four outputs may be moved at once
    float *h;                // [splits][tokens][rank16]
};

// How many tiles there are: none in groups of another batch, whose rows are not these.
__device__ __forceinline__ int tiles_of(const AdapterArgs &A) {
    const GroupHeader h = *A.header;
    return h.tokens == A.tokens && h.adapters == A.count ? h.tiles : 0;
}

__device__ __forceinline__ int rank_of(const AdapterArgs &A, int adapter) {
    return A.ranks ? min(max(A.ranks[adapter], 0), A.max_rank) : A.max_rank;
}

// Eight elements of x from `at` on as f32 or, where the type is exact in it, f16.
template <int XK>
struct XLoad {
    h8 v;
    __device__ __forceinline__ void load(const void *x, int64_t at, bool in) {
        v = h8{};
        if (!in) return;
        if (XK == G4_KIND_F16) {
            v = *reinterpret_cast<const h8 *>(static_cast<const _Float16 *>(x) + at);
        } else {
            const uint2 c = *reinterpret_cast<const uint2 *>(static_cast<const int8_t *>(x) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (_Float16)(float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e % 4)));
        }
    }
};
template <>
struct XLoad<G4_KIND_F32> {
    f4 v[2];
    __device__ __forceinline__ void load(const void *x, int64_t at, bool in) {
        v[0] = v[1] = f4{};
        if (!in) return;
        const f4 *p = reinterpret_cast<const f4 *>(static_cast<const float *>(x) + at);
        v[0] = p[0];
        v[1] = p[1];
    }
};

template <int XK>
__device__ __forceinline__ f4 product(h8 a, const XLoad<XK> &x, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, x.v, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f4 product<G4_KIND_F32>(h8 a, const XLoad<G4_KIND_F32> &x, f4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32((float)a[e], x.v[e / 4][e % 4], c, 0, 0, 0);
    return c;
}

// Grid (splits, tiles): a range of K of a tile's H; the block's waves take steps of 32 in turn and add up in LDS. RT:
// the pool's rank in tiles of 16.
template <int XK, int RT>
__global__ __launch_bounds__(kAdThreads) void adapter_shrink_kernel(AdapterArgs A) {
    __shared__ f4 part[kAdWaves][RT][64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 15, group = lane >> 4;
    if ((int)blockIdx.y >= tiles_of(A)) return;
    const GroupTile T = A.tiles[blockIdx.y];
    if (T.adapter < 0) return;
    const int rank = rank_of(A, T.adapter);
    const int64_t row = A.order[T.first + min(col, T.rows - 1)];
    const _Float16 *a = A.a + T.adapter * A.a_stride;
    f4 acc[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) acc[r] = f4{};
    const int k0 = blockIdx.x * A.range, k1 = min(k0 + A.range, A.k);
    for (int k = k0 + 32 * wave; k < k1; k += 32 * kAdWaves) {
        const int at = k + 8 * group;
        const bool in = at < k1;
        XLoad<XK> x;
        x.load(A.x, row * A.x_stride + at, in);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            h8 w{};
            if (in && 16 * r + col < rank) w = *reinterpret_cast<const h8 *>(a + (int64_t)(16 * r + col) * A.k + at);
            acc[r] = product<XK>(w, x, acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) part[wave][r][lane] = acc[r];
    __syncthreads();
    for (int i = t; i < RT * 64; i += kAdThreads) {
        const int r = i >> 6, l = i & 63;
        f4 s = part[0][r][l];
#pragma unroll
        for (int w = 1; w < kAdWaves; ++w) s += part[w][r][l];
        if ((l & 15) < T.rows)
            *reinterpret_cast<f4 *>(A.h + ((int64_t)blockIdx.x * A.tokens + T.first + (l & 15)) * A.rank16 + 16 * r +
                                    4 * (l >> 4)) = s;
    }
}

template <int KIND>
__device__ __forceinline__ f4 load4(const void *p, int64_t at, int n, bool vec, float scale) {
    f4 y{};
    if (KIND == G4_KIND_I8) {
        const int8_t *q = static_cast<const int8_t *>(p) + at;
        if (vec) {
            const uint32_t c = *reinterpret_cast<const uint32_t *>(q);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (float)(int8_t)(c >> (8 * e)) * scale;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) y[e] = (float)q[e] * scale;
        }
    } else if (KIND == G4_KIND_F16) {
        const _Float16 *q = static_cast<const _Float16 *>(p) + at;
        if (vec) {
            const h4 c = *reinterpret_cast<const h4 *>(q);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (float)c[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) y[e] = (float)q[e];
        }
    } else {
        const float *q = static_cast<const float *>(p) + at;
        if (vec) {
            y = *reinterpret_cast<const f4 *>(q);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) y[e] = q[e];
        }
    }
    return y;
}

template <int KIND>
__device__ __forceinline__ void store4(void *p, int64_t at, int n, bool vec, f4 y, float snap) {
    if (KIND == G4_KIND_I8) {
        int8_t *q = static_cast<int8_t *>(p) + at;
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) c |= (uint32_t)(uint8_t)srq_code_i(y[e], snap) << (8 * e);
        if (vec) {
            *reinterpret_cast<uint32_t *>(q) = c;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) q[e] = (int8_t)(c >> (8 * e));
        }
        return;
    }
    if (snap != 0.0f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = srq_code_f(y[e], snap) * snap;
    }
    if (KIND == G4_KIND_F16) {
        _Float16 *q = static_cast<_Float16 *>(p) + at;
        h4 c;
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = (_Float16)y[e];
        if (vec) {
            *reinterpret_cast<h4 *>(q) = c;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) q[e] = c[e];
        }
    } else {
        float *q = static_cast<float *>(p) + at;
        if (vec) {
            *reinterpret_cast<f4 *>(q) = y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < n) q[e] = y[e];
        }
    }
}

constexpr int kNTiles = 4;                            // tiles of 16 outputs a wave has
constexpr int kNBlock = kAdWaves * kNTiles * kTile;  // outputs a block has

// Grid (ranges of N, tiles).
template <int BK, int OK, int RT>
__global__ __launch_bounds__(kAdThreads) void adapter_expand_kernel(AdapterArgs A) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 15, group = lane >> 4;
    if ((int)blockIdx.y >= tiles_of(A)) return;
    const GroupTile T = A.tiles[blockIdx.y];
    const bool some = col < T.rows;
    const int64_t row = A.order[T.first + min(col, T.rows - 1)];
    const int n0 = blockIdx.x * kNBlock + wave * (kNTiles * kTile);
    f4 acc[kNTiles];
#pragma unroll
    for (int j = 0; j < kNTiles; ++j) acc[j] = f4{};
    float scale = 0.0f;
    if (T.adapter >= 0) {
        const int rank = rank_of(A, T.adapter);
        scale = (A.scales ? A.scales[T.adapter] : 1.0f) * A.x_scale;
        const _Float16 *b = A.b + T.adapter * A.b_stride;
        const float *h = A.h + (int64_t)(T.first + min(col, T.rows - 1)) * A.rank16;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int at = 16 * r + 4 * group;  // the lane's ranks at .. at + 3
            if (16 * r >= rank) break;
            f4 y{};
            for (int s = 0; s < A.splits; ++s)
                y += *reinterpret_cast<const f4 *>(h + (int64_t)s * A.tokens * A.rank16 + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = at + e < rank ? y[e] : 0.0f;  // (an infinite x leaves NaN there)
#pragma unroll
            for (int j = 0; j < kNTiles; ++j) {
                const int n = n0 + 16 * j + col;
                h4 w{};
                if (n < A.n && at < rank) w = *reinterpret_cast<const h4 *>(b + (int64_t)n * A.max_rank + at);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(at + e < rank ? (float)w[e] : 0.0f, y[e], acc[j], 0, 0, 0);
            }
        }
    }
    if (!some) return;
#pragma unroll
    for (int j = 0; j < kNTiles; ++j) {
        const int n = n0 + 16 * j + 4 * group, left = A.n - n;
        if (left <= 0) continue;
        f4 y{};
        if (A.base) y = load4<BK>(A.base, row * A.base_stride + n, left, A.vec, A.base_scale);
        if (T.adapter >= 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += scale * acc[j][e];
        }
        store4<OK>(A.out, row * A.out_stride + n, left, A.vec, y, A.out_scale);
    }
}

// Ranges of K: blocks for every CU a few times, each with some steps of 32 for each of its waves.
static int adapter_splits(int k, int tokens) {
    const int tiles = (tokens + kTile - 1) / kTile, most = (k + 32 * kAdWaves - 1) / (32 * kAdWaves);
    int want = (1024 + tiles - 1) / tiles;
    if (want > 16) want = 16;
    return want < most ? want : most;
}

template <int XK>
static int launch_shrink(const AdapterArgs &A, dim3 grid, hipStream_t s) {
    switch (A.rank16 / 16) {
#define G4_RT(n) case n: hipLaunchKernelGGL((adapter_shrink_kernel<XK, n>), grid, dim3(kAdThreads), 0, s, A); break
        G4_RT(1); G4_RT(2); G4_RT(3); G4_RT(4); G4_RT(5); G4_RT(6); G4_RT(7); G4_RT(8);
#undef G4_RT
    }
    G4_LAUNCHED("adapter_shrink_kernel");
    return G4_OK;
}

template <int BK, int OK>
static int launch_expand(const AdapterArgs &A, dim3 grid, hipStream_t s) {
    if (A.rank16 <= 32)
        hipLaunchKernelGGL((adapter_expand_kernel<BK, OK, 2>), grid, dim3(kAdThreads), 0, s, A);
    else
        hipLaunchKernelGGL((adapter_expand_kernel<BK, OK, kMaxRank / 16>), grid, dim3(kAdThreads), 0, s, A);
    G4_LAUNCHED("adapter_expand_kernel");
    return G4_OK;
}
template <int BK>
static int launch_expand_out(const AdapterArgs &A, int ok, dim3 grid, hipStream_t s) {
    if (ok == G4_KIND_I8) return launch_expand<BK, G4_KIND_I8>(A, grid, s);
    if (ok == G4_KIND_F16) return launch_expand<BK, G4_KIND_F16>(A, grid, s);
    return launch_expand<BK, G4_KIND_F32>(A, grid, s);
}

static int check_adapters(const char *who, const g4_adapters *D) {
    if (!D || !D->a || !D->b) return set_error(G4_ERR_INVALID, "%s needs the adapters' A and B", who);
    if (D->count <= 0 || D->count > kMaxAdapters)
        return set_error(G4_ERR_INVALID, "%s: %d adapters (1 to %d)", who, D->count, kMaxAdapters);
    if (D->k <= 0 || D->k % 8 || D->n <= 0)
        return set_error(G4_ERR_INVALID, "%s: k %d, n %d (k a multiple of 8)", who, D->k, D->n);
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
    hipLaunchKernelGGL(adapter_groups_kernel, dim3(1), dim3(kGroupThreads), (adapters + 1) * sizeof(int32_t),
                       as_stream(stream), row_adapter, tokens, adapters, h, tiles,
                       reinterpret_cast<int32_t *>(tiles + max_tiles(tokens, adapters)));
    G4_LAUNCHED("adapter_groups_kernel");
    return G4_OK;
}

size_t g4_adapter_workspace_bytes(const g4_adapters *adapters, int tokens) {
    if (check_adapters("adapter-linear", adapters) || tokens <= 0 || tokens > kMaxTokens) return 0;
    return (size_t)adapter_splits(adapters->k, tokens) * tokens * ((adapters->max_rank + 15) / 16 * 16) * sizeof(float);
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
    A.order = reinterpret_cast<const int32_t *>(A.tiles + tiles);
    A.x = x;
    A.x_stride = xs;
    A.x_scale = x_kind == G4_KIND_I8 ? x_scale : 1.0f;
    A.base = base;
    A.base_stride = bs;
    A.base_scale = base_scale;
    A.out = out;
    A.out_stride = os;
    A.out_scale = out_scale;
    A.splits = adapter_splits(D->k, tokens);
    A.range = ((D->k + A.splits - 1) / A.splits + 31) / 32 * 32;
    A.vec = D->n % 4 == 0 && os % 4 == 0 && (!base || bs % 4 == 0) &&
            ((uintptr_t)out % (4 * kind_size(out_kind))) == 0 && (!base || (uintptr_t)base % (4 * kind_size(base_kind)) == 0);
    A.h = static_cast<float *>(workspace);
    hipStream_t s = as_stream(stream);
    const dim3 grid(A.splits, (unsigned)tiles);
    int st;
    if (x_kind == G4_KIND_I8) st = launch_shrink<G4_KIND_I8>(A, grid, s);
    else if (x_kind == G4_KIND_F16) st = launch_shrink<G4_KIND_F16>(A, grid, s);
    else st = launch_shrink<G4_KIND_F32>(A, grid, s);
    if (st) return st;
    const dim3 out_grid((unsigned)((D->n + kNBlock - 1) / kNBlock), (unsigned)tiles);
    if (base && base_kind == G4_KIND_I8) return launch_expand_out<G4_KIND_I8>(A, out_kind, out_grid, s);
    if (base && base_kind == G4_KIND_F16) return launch_expand_out<G4_KIND_F16>(A, out_kind, out_grid, s);
    return launch_expand_out<G4_KIND_F32>(A, out_kind, out_grid, s);
}

}  // extern "C"
