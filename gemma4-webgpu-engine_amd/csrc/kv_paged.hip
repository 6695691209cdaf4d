// The paged KV cache's store and read-back (include/g4serve.h): a chunk's q / k norm and RoPE with the
// store of K and V as f16 or as int8 codes with a scale per row, and the rows back as f32 or f16.
#include "g4_paged.h"

namespace g4 {

int paged_args(const char *who, const g4_kv_pages *P, const g4_chunk *C, PagedArgs *out) {
    if (!P || !C) return set_error(G4_ERR_INVALID, "%s needs the pages and the chunk", who);
    if (P->kind != G4_KIND_F16 && P->kind != G4_KIND_I8)
        return set_error(G4_ERR_INVALID, "%s: pages are f16 or int8 codes, got kind %d", who, P->kind);
    if (P->head_dim != 64 && P->head_dim != 128 && P->head_dim != 256)
        return set_error(G4_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 and 256 are served)", who, P->head_dim);
    if (P->kv_heads <= 0 || P->num_pages <= 0)
        return set_error(G4_ERR_INVALID, "%s: %d KV heads, %d pages", who, P->kv_heads, P->num_pages);
    if (P->page_size < 8 || P->page_size > 4096 || (P->page_size & (P->page_size - 1)))
        return set_error(G4_ERR_INVALID, "%s: page_size %d is not a power of two from 8 to 4096", who, P->page_size);
    if (!P->k || !P->v) return set_error(G4_ERR_INVALID, "%s needs both page pools", who);
    if (P->kind == G4_KIND_I8 && (!P->k_scales || !P->v_scales))
        return set_error(G4_ERR_INVALID, "%s: int8 pages need their scales", who);
    const int64_t unit = P->kind == G4_KIND_I8 ? 16 : 8;  // elements of 16 bytes
    int64_t ps = P->page_stride, ss = P->slot_stride, hs = P->head_stride;
    if (!ps && !ss && !hs) {
        hs = P->head_dim;
        ss = hs * P->kv_heads;
        ps = ss * P->page_size;
    }
    if (((uintptr_t)P->k | (uintptr_t)P->v) & 15)
        return set_error(G4_ERR_INVALID, "%s: the page pools must be 16-byte aligned", who);
    if (ps < P->head_dim || ss < P->head_dim || hs < P->head_dim || ps % unit || ss % unit || hs % unit)
        return set_error(G4_ERR_INVALID,
                         "%s: page, slot and head strides must hold a row and be multiples of 16 bytes", who);
    if (C->seqs <= 0 || C->tokens <= 0 || C->max_q <= 0 || C->max_kv <= 0)
        return set_error(G4_ERR_INVALID, "%s: the chunk has %d sequences, %d tokens, max_q %d, max_kv %d", who,
                         C->seqs, C->tokens, C->max_q, C->max_kv);
    if (!C->q_start || !C->kv_len || !C->page_table)
        return set_error(G4_ERR_INVALID, "%s: the chunk needs q_start, kv_len and page_table", who);
    if (C->table_pages <= 0 || (int64_t)C->table_pages * P->page_size < C->max_kv)
        return set_error(G4_ERR_INVALID, "%s: %d table pages of %d slots do not hold max_kv %d positions", who,
                         C->table_pages, P->page_size, C->max_kv);
    if (C->table_stride && C->table_stride < C->table_pages)
        return set_error(G4_ERR_INVALID, "%s: table_stride %lld < %d table pages", who,
                         (long long)C->table_stride, C->table_pages);
    out->k = P->k;
    out->v = P->v;
    out->ks = P->k_scales;
    out->vs = P->v_scales;
    out->page_stride = ps;
    out->slot_stride = ss;
    out->head_stride = hs;
    out->table = C->page_table;
    out->table_stride = C->table_stride ? C->table_stride : C->table_pages;
    out->q_start = C->q_start;
    out->kv_len = C->kv_len;
    out->seqs = C->seqs;
    out->tokens = C->tokens;
    out->max_q = C->max_q < C->tokens ? C->max_q : C->tokens;
    out->max_kv = C->max_kv;
    out->kv_heads = P->kv_heads;
    out->page_shift = __builtin_ctz(P->page_size);
    out->num_pages = P->num_pages;
    return G4_OK;
}

// ---- the prologue and the store -----------------------------------------------------------------------

struct PrologueArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    float q_scale, k_scale, v_scale;
    int heads;
    const float *q_gain, *k_gain, *cos_tab, *sin_tab;
    float eps;
    _Float16 *q_out;
};

template <int XK>
__device__ __forceinline__ float load_x(const void *x, int64_t i, float scale) {
    if (XK == G4_KIND_I8) return (float)static_cast<const int8_t *>(x)[i] * scale;
    if (XK == G4_KIND_F16) return (float)static_cast<const _Float16 *>(x)[i];
    return static_cast<const float *>(x)[i];
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
    return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

// RNE(127 y / amax). The f32 quotient is a few parts in 2^24 off, which matters only next to a half:
// there (and where 1 / amax or 127 y leave the f32 range) the division is done in 64 bits, where a
// quotient of two such values that is not a half rounds to none.
__device__ __forceinline__ int quant_code(float y, float amax, float r) {
    const float t = y * r;  // r = 127 / amax
    float n = __builtin_rintf(t);
    if (!(fabsf(fabsf(t - n) - 0.5f) > 0x1p-12f)) n = (float)__builtin_rint(127.0 * (double)y / (double)amax);
    return (int)n;
}

// Bound by each wave's way, q_start -> kv_len and page -> row (2048 tokens, 10 rows of 256 each, codes in: 13.4 us,
// 16 MB; one token 4 us): a wave per row has all of them on their way at once, but looks its sequence and page up by
// itself.
// One wave per head row: lane l holds elements E l .. E l + E - 1 (E = D / 64), so the RoPE pair
// (i, i + D / 2) is lanes l and l + 32 of the same register. Row 0 .. heads - 1 of a token are its
// queries, then kv_heads of K, then of V.
template <int D, int XK, int CK>
__global__ __launch_bounds__(256) void paged_prologue_kernel(PagedArgs A, PrologueArgs R) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int kvh = R.k ? A.kv_heads : 0;
    const int per = R.heads + 2 * kvh;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (int64_t)A.tokens * per) return;
    const int row = (int)(id / per), h = (int)(id % per);
    const bool is_q = h < R.heads, is_v = h >= R.heads + kvh;
    const int head = is_q ? h : (is_v ? h - R.heads - kvh : h - R.heads);
    const int seq = seq_of_row(A, row);
    if (seq >= A.seqs) return;
    const SeqSpan S = seq_span(A, seq);
    const int i = row - S.start;
    if (i < 0 || i >= min(S.rows, A.max_q)) return;
    const int pos = S.kv - S.rows + i;
    const void *src = is_q ? R.q : (is_v ? R.v : R.k);
    const int64_t base = row * (is_q ? R.q_stride : (is_v ? R.v_stride : R.k_stride)) + (int64_t)head * D + lane * E;
    const float sc = is_q ? R.q_scale : (is_v ? R.v_scale : R.k_scale);
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = load_x<XK>(src, base + e, sc);
    const bool norm = is_q ? R.q_gain != nullptr : R.k_gain != nullptr;
    if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += y[e] * y[e];
        ss = wave_sum(ss);
        const float inv = 1.0f / __fsqrt_rn(ss / (float)D + R.eps);
        const float *gain = is_q ? R.q_gain : R.k_gain;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            y[e] *= inv;
            if (!is_v) y[e] *= gain[lane * E + e];
        }
    }
    if (R.cos_tab && !is_v && pos >= 0) {
        const float *c = R.cos_tab + (int64_t)pos * (D / 2) + (lane & 31) * E;
        const float *s = R.sin_tab + (int64_t)pos * (D / 2) + (lane & 31) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float o = __shfl_xor(y[e], 32);
            y[e] = lane < 32 ? y[e] * c[e] - o * s[e] : y[e] * c[e] + o * s[e];
        }
    }
    if (is_q) {
        _Float16 *dst = R.q_out + ((int64_t)row * R.heads + head) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = (_Float16)y[e];
        return;
    }
    if (pos < 0) return;
    const int page = page_of(A, seq, pos);
    if (page < 0) return;
    const int64_t at = row_offset(A, page, pos, head) + lane * E;
    if (CK == G4_KIND_F16) {
        _Float16 *dst = static_cast<_Float16 *>(is_v ? A.v : A.k) + at;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = (_Float16)y[e];
        return;
    }
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        top = fmaxf(top, fabsf(y[e]));
        bad |= !(fabsf(y[e]) <= 3.402823466e38f);
    }
    const float amax = wave_max(top);
    bad = __any(bad);
    const float r = 127.0f / amax;
    int8_t *dst = static_cast<int8_t *>(is_v ? A.v : A.k) + at;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = (bad || amax == 0.0f) ? 0 : (int8_t)quant_code(y[e], amax, r);
    if (lane == 0)
        (is_v ? A.vs : A.ks)[scale_offset(A, page, pos, head)] = bad ? __builtin_nanf("") : amax / 127.0f;
}

// ---- the read-back ------------------------------------------------------------------------------------

// Bound by HBM: 67000 tokens of 4 heads of 128, codes to f16, 209 MB, on other pages in each call 46.5 us (4.5 TB/s);
// 65 with K and V in blocks of their own and a search per row; batches of 2 and 8 47.6 and 45.6, blocks of 8 and 32
// tokens 45.7 and 46.7. On the same pages call after call, of which the 256 MB cache holds part: 32.7; 34.0, 33.3,
// 33.1 and 34.2.
// A block takes kReadTokens rows: a wave looks them up at once (the first one's sequence by ballots over the
// ends, the others' from there on), then threads move units of 8 elements, K's and V's of kReadBatch at a time.
constexpr int kReadTokens = 16, kReadBatch = 4;

template <int CK, int OK>
__global__ __launch_bounds__(256) void kv_read_kernel(PagedArgs A, int d_shift, void *k_out, void *v_out,
                                                      int64_t seq_stride) {
    __shared__ int64_t src_at[kReadTokens], dst_at[kReadTokens], scale_at[kReadTokens];  // src_at < 0: absent
    const int t = threadIdx.x;
    const int row0 = blockIdx.x * kReadTokens;
    const int64_t width = (int64_t)A.kv_heads << d_shift;
    if (t < 64) {
        int seq = seq_of_row(A, row0);
        if (t < kReadTokens) {
            const int row = row0 + t;
            while (seq < A.seqs && A.q_start[seq + 1] <= row) ++seq;
            int64_t dst = -1, src = -1;
            if (seq < A.seqs && row < A.tokens) {
                const SeqSpan S = seq_span(A, seq);
                const int i = row - S.start, pos = S.kv - S.rows + i;
                if (i >= 0 && i < min(S.rows, A.max_q)) {
                    dst = seq_stride ? seq * seq_stride + i * width : (int64_t)row * width;
                    const int page = pos >= 0 ? page_of(A, seq, pos) : -1;
                    if (page >= 0) {
                        src = row_offset(A, page, pos, 0);
                        scale_at[t] = scale_offset(A, page, pos, 0);
                    }
                }
            }
            dst_at[t] = dst;
            src_at[t] = src;
        }
    }
    __syncthreads();
    const int d = 1 << d_shift, per = (int)(width >> 3);  // units of 8 elements, of a token
    const int units = kReadTokens * per;
    constexpr int EB = CK == G4_KIND_F16 ? 2 : 1;
    for (int u0 = t; u0 < units; u0 += 256 * kReadBatch) {
        int64_t to[kReadBatch];
        uint4 x[2][kReadBatch];
        float s[2][kReadBatch];
#pragma unroll
        for (int b = 0; b < kReadBatch; ++b) {
            const int u = min(u0 + 256 * b, units - 1), j = u / per, e = (u - j * per) * 8, head = e >> d_shift;
            to[b] = u0 + 256 * b < units ? dst_at[j] : -1;
            const int64_t src = src_at[j];
            const int64_t at = (src + head * A.head_stride + (e & (d - 1))) * EB;
            const int64_t sat = CK == G4_KIND_I8 && src >= 0 ? scale_at[j] + ((int64_t)head << A.page_shift) : 0;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                x[w][b] = make_uint4(0, 0, 0, 0);
                s[w][b] = 0.0f;
                if (to[b] < 0 || src < 0 || !(w ? v_out : k_out)) continue;
                const char *p = static_cast<const char *>(w ? A.v : A.k) + at;
                if (CK == G4_KIND_F16) {
                    x[w][b] = *reinterpret_cast<const uint4 *>(p);
                } else {
                    const uint2 y = *reinterpret_cast<const uint2 *>(p);
                    x[w][b].x = y.x;
                    x[w][b].y = y.y;
                    s[w][b] = (w ? A.vs : A.ks)[sat];
                }
            }
            if (to[b] >= 0) to[b] += e;
        }
#pragma unroll
        for (int b = 0; b < kReadBatch; ++b)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                void *out = w ? v_out : k_out;
                if (to[b] < 0 || !out) continue;
                float y[8];
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    y[n] = CK == G4_KIND_F16 ? (float)__builtin_bit_cast(h8, x[w][b])[n]
                                             : (float)(int8_t)((n < 4 ? x[w][b].x : x[w][b].y) >> (8 * (n % 4))) * s[w][b];
                if (OK == G4_KIND_F16) {
                    h8 o;
#pragma unroll
                    for (int n = 0; n < 8; ++n) o[n] = (_Float16)y[n];
                    *reinterpret_cast<h8 *>(static_cast<_Float16 *>(out) + to[b]) = o;
                } else {
                    float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(out) + to[b]);
                    o[0] = make_float4(y[0], y[1], y[2], y[3]);
                    o[1] = make_float4(y[4], y[5], y[6], y[7]);
                }
            }
    }
}

constexpr int64_t kMaxBlocks = (1 << 24) - 1;  // of 256 threads: a grid has less than 2^32 threads

template <int D, int XK>
static int launch_prologue(const PagedArgs &A, const PrologueArgs &R, int ck, hipStream_t stream) {
    const int64_t rows = (int64_t)A.tokens * (R.heads + (R.k ? 2 * A.kv_heads : 0));
    const dim3 grid((unsigned)((rows + 3) / 4));
    if (ck == G4_KIND_F16)
        hipLaunchKernelGGL((paged_prologue_kernel<D, XK, G4_KIND_F16>), grid, dim3(256), 0, stream, A, R);
    else
        hipLaunchKernelGGL((paged_prologue_kernel<D, XK, G4_KIND_I8>), grid, dim3(256), 0, stream, A, R);
    G4_LAUNCHED("paged_prologue_kernel");
    return G4_OK;
}

template <int D>
static int launch_prologue_kind(const PagedArgs &A, const PrologueArgs &R, int xk, int ck, hipStream_t stream) {
    if (xk == G4_KIND_I8) return launch_prologue<D, G4_KIND_I8>(A, R, ck, stream);
    if (xk == G4_KIND_F16) return launch_prologue<D, G4_KIND_F16>(A, R, ck, stream);
    return launch_prologue<D, G4_KIND_F32>(A, R, ck, stream);
}

}  // namespace g4

using namespace g4;

extern "C" {

int g4_paged_prologue(const g4_kv_pages *pages, const g4_chunk *chunk, int x_kind, const void *q,
                      int64_t q_stride, float q_scale, const void *k, int64_t k_stride, float k_scale,
                      const void *v, int64_t v_stride, float v_scale, int heads, const float *q_gain,
                      const float *k_gain, const float *cos_tab, const float *sin_tab,
                      int rope_positions, float eps, void *q_out, void *stream) {
    PagedArgs A;
    if (int st = paged_args("paged-prologue", pages, chunk, &A)) return st;
    if (x_kind != G4_KIND_F32 && x_kind != G4_KIND_F16 && x_kind != G4_KIND_I8)
        return set_error(G4_ERR_INVALID, "paged-prologue: rows are f32, f16 or int8 codes, got kind %d", x_kind);
    if (!q && !k) return set_error(G4_ERR_INVALID, "paged-prologue needs q, or k and v");
    if (!k != !v) return set_error(G4_ERR_INVALID, "paged-prologue needs k and v together");
    if (q ? (heads <= 0 || !q_out) : heads != 0)
        return set_error(G4_ERR_INVALID, "paged-prologue: q needs heads and q_out, and none of them stands alone");
    if (!cos_tab != !sin_tab) return set_error(G4_ERR_INVALID, "paged-prologue needs cosTab and sinTab together");
    if (cos_tab && rope_positions < A.max_kv)
        return set_error(G4_ERR_INVALID, "paged-prologue: the tables hold %d positions, max_kv is %d",
                         rope_positions, A.max_kv);
    const int d = pages->head_dim;
    const int64_t qw = (int64_t)heads * d, kw = (int64_t)A.kv_heads * d;
    if ((q && q_stride && q_stride < qw) || (k && k_stride && k_stride < kw) || (v && v_stride && v_stride < kw))
        return set_error(G4_ERR_INVALID, "paged-prologue: a row stride is shorter than the row");
    if ((int64_t)A.tokens * (heads + (k ? 2 * (int64_t)A.kv_heads : 0)) > 4 * kMaxBlocks)
        return set_error(G4_ERR_UNSUPPORTED, "paged-prologue: more than %lld head rows", (long long)(4 * kMaxBlocks));
    PrologueArgs R{q, k, v, q_stride ? q_stride : qw, k_stride ? k_stride : kw, v_stride ? v_stride : kw,
                   q_scale, k_scale, v_scale, heads, q_gain, k_gain, cos_tab, sin_tab, eps,
                   static_cast<_Float16 *>(q_out)};
    if (d == 64) return launch_prologue_kind<64>(A, R, x_kind, pages->kind, as_stream(stream));
    if (d == 128) return launch_prologue_kind<128>(A, R, x_kind, pages->kind, as_stream(stream));
    return launch_prologue_kind<256>(A, R, x_kind, pages->kind, as_stream(stream));
}

int g4_kv_read(const g4_kv_pages *pages, const g4_chunk *chunk, void *k_out, void *v_out, int out_kind,
               int64_t seq_stride, void *stream) {
    PagedArgs A;
    if (int st = paged_args("kv-read", pages, chunk, &A)) return st;
    if (!k_out && !v_out) return set_error(G4_ERR_INVALID, "kv-read: no output");
    if (out_kind != G4_KIND_F32 && out_kind != G4_KIND_F16)
        return set_error(G4_ERR_INVALID, "kv-read: outputs are f32 or f16, got kind %d", out_kind);
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15)
        return set_error(G4_ERR_INVALID, "kv-read: outputs must be 16-byte aligned");
    const int64_t unit = out_kind == G4_KIND_F16 ? 8 : 4;
    if (seq_stride && (seq_stride % unit || seq_stride < (int64_t)A.max_q * A.kv_heads * pages->head_dim))
        return set_error(G4_ERR_INVALID, "kv-read: seq_stride must hold max_q rows and be a multiple of 16 bytes");
    if (A.tokens > kReadTokens * kMaxBlocks)
        return set_error(G4_ERR_UNSUPPORTED, "kv-read: more than %lld rows", (long long)(kReadTokens * kMaxBlocks));
    const dim3 grid((unsigned)(((int64_t)A.tokens + kReadTokens - 1) / kReadTokens));
    const int ds = __builtin_ctz(pages->head_dim);
    hipStream_t s = as_stream(stream);
    const bool f16 = pages->kind == G4_KIND_F16, o16 = out_kind == G4_KIND_F16;
    if (f16 && o16)
        hipLaunchKernelGGL((kv_read_kernel<G4_KIND_F16, G4_KIND_F16>), grid, dim3(256), 0, s, A, ds, k_out, v_out, seq_stride);
    else if (f16)
        hipLaunchKernelGGL((kv_read_kernel<G4_KIND_F16, G4_KIND_F32>), grid, dim3(256), 0, s, A, ds, k_out, v_out, seq_stride);
    else if (o16)
        hipLaunchKernelGGL((kv_read_kernel<G4_KIND_I8, G4_KIND_F16>), grid, dim3(256), 0, s, A, ds, k_out, v_out, seq_stride);
    else
        hipLaunchKernelGGL((kv_read_kernel<G4_KIND_I8, G4_KIND_F32>), grid, dim3(256), 0, s, A, ds, k_out, v_out, seq_stride);
    G4_LAUNCHED("kv_read_kernel");
    return G4_OK;
}

}  // extern "C"
