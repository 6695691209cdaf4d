// Causal attention of a chunk of new tokens over the paged cache (include/g4serve.h).
#include "g4_paged.h"

namespace g4 {

struct AttnArgs {
    const _Float16 *q;
    int64_t q_stride;
    int heads, group;
    float scale;
    int window;
    void *out;
    int out_kind;
    float in_scale;
};

__device__ __forceinline__ void attn_put(const AttnArgs &R, int64_t at, float y) {
    if (R.out_kind == G4_KIND_F16)
        static_cast<_Float16 *>(R.out)[at] = (_Float16)y;
    else if (R.out_kind == G4_KIND_I8)
        static_cast<int8_t *>(R.out)[at] = (int8_t)srq_code_i(y, R.in_scale);
    else
        static_cast<float *>(R.out)[at] = y;
}

// One wave per (row, head): the running maximum and sum of the softmax over the keys in order, lane l
// holding dims l, l + 64, ...
template <int D, int CK>
__global__ __launch_bounds__(256) void attn_chunk_kernel(PagedArgs A, AttnArgs R) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (int64_t)A.tokens * R.heads) return;
    const int row = (int)(id / R.heads), h = (int)(id % R.heads), kvh = h / R.group;
    const int seq = seq_of_row(A, row);
    if (seq >= A.seqs) return;
    const SeqSpan S = seq_span(A, seq);
    const int i = row - S.start;
    if (i < 0 || i >= min(S.rows, A.max_q)) return;
    const int pos = S.kv - S.rows + i;
    float q[E], o[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = (float)R.q[row * R.q_stride + (int64_t)h * D + lane + 64 * e];
    float m = -INFINITY, l = 0.0f;
    for (int j = R.window ? max(0, pos - R.window + 1) : 0; j <= pos; ++j) {
        const int page = page_of(A, seq, j);
        if (page < 0) continue;
        const int64_t at = row_offset(A, page, j, kvh) + lane;
        float k[E], v[E];
        float ks = 1.0f, vs = 1.0f;
        if (CK == G4_KIND_I8) {
            ks = A.ks[scale_offset(A, page, j, kvh)];
            vs = A.vs[scale_offset(A, page, j, kvh)];
        }
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (CK == G4_KIND_I8) {
                k[e] = static_cast<const int8_t *>(A.k)[at + 64 * e];
                v[e] = static_cast<const int8_t *>(A.v)[at + 64 * e];
            } else {
                k[e] = (float)static_cast<const _Float16 *>(A.k)[at + 64 * e];
                v[e] = (float)static_cast<const _Float16 *>(A.v)[at + 64 * e];
            }
            s += q[e] * k[e];
        }
#pragma unroll
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
        s *= ks * R.scale;
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY) continue;
        const float a = expf(m - mn), p = expf(s - mn);
        l = l * a + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * a + p * vs * v[e];
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        attn_put(R, ((int64_t)row * R.heads + h) * D + lane + 64 * e, l == 0.0f ? 0.0f : o[e] / l);
}

template <int D>
static int launch_attn(const PagedArgs &A, const AttnArgs &R, int ck, hipStream_t stream) {
    const dim3 grid((unsigned)(((int64_t)A.tokens * R.heads + 3) / 4));
    if (ck == G4_KIND_F16)
        hipLaunchKernelGGL((attn_chunk_kernel<D, G4_KIND_F16>), grid, dim3(256), 0, stream, A, R);
    else
        hipLaunchKernelGGL((attn_chunk_kernel<D, G4_KIND_I8>), grid, dim3(256), 0, stream, A, R);
    G4_LAUNCHED("attn_chunk_kernel");
    return G4_OK;
}

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_attention_chunk_workspace_bytes(const g4_kv_pages *pages, const g4_chunk *chunk, int heads,
                                          int window) {
    PagedArgs A;
    if (paged_args("attention-chunk", pages, chunk, &A) || heads <= 0 || heads % A.kv_heads || window < 0) return 0;
    return 16;
}

int g4_attention_chunk(const g4_kv_pages *pages, const g4_chunk *chunk, const void *q, int64_t q_stride,
                       int heads, float scale, int window, void *workspace, size_t workspace_bytes,
                       void *out, int out_kind, float in_scale, void *stream) {
    PagedArgs A;
    if (int st = paged_args("attention-chunk", pages, chunk, &A)) return st;
    if (!q || !out || !workspace) return set_error(G4_ERR_INVALID, "attention-chunk needs q, an output and a workspace");
    if (heads <= 0 || heads % A.kv_heads)
        return set_error(G4_ERR_INVALID, "attention-chunk: %d query heads do not divide over %d KV heads", heads, A.kv_heads);
    if (window < 0) return set_error(G4_ERR_INVALID, "attention-chunk: window %d", window);
    if (out_kind != G4_KIND_F16 && out_kind != G4_KIND_F32 && out_kind != G4_KIND_I8)
        return set_error(G4_ERR_INVALID, "attention-chunk: outputs are f16, f32 or int8 codes, got kind %d", out_kind);
    if (out_kind == G4_KIND_I8 && in_scale == 0.0f)
        return set_error(G4_ERR_INVALID, "attention-chunk: int8 codes need the consumer's inScale");
    const int64_t qw = (int64_t)heads * pages->head_dim;
    if (q_stride && (q_stride < qw || q_stride % 8))
        return set_error(G4_ERR_INVALID, "attention-chunk: q_stride must hold a row and be a multiple of 8");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return set_error(G4_ERR_INVALID, "attention-chunk: q, the output and the workspace must be 16-byte aligned");
    if ((int64_t)A.tokens * heads > ((int64_t)1 << 31))
        return set_error(G4_ERR_UNSUPPORTED, "attention-chunk: more than 2^31 query rows");
    const size_t need = g4_attention_chunk_workspace_bytes(pages, chunk, heads, window);
    if (workspace_bytes < need)
        return set_error(G4_ERR_INVALID, "attention-chunk: workspace %zu B < %zu B", workspace_bytes, need);
    const AttnArgs R{static_cast<const _Float16 *>(q), q_stride ? q_stride : qw, heads, heads / A.kv_heads,
                     scale, window, out, out_kind, in_scale};
    if (pages->head_dim == 64) return launch_attn<64>(A, R, pages->kind, as_stream(stream));
    if (pages->head_dim == 128) return launch_attn<128>(A, R, pages->kind, as_stream(stream));
    return launch_attn<256>(A, R, pages->kind, as_stream(stream));
}

}  // extern "C"
