/*
 * g4serve.h - serving operators on a paged KV cache: the prologue of a chunk of new tokens with its
 * quantising store, the read-back, attention of the chunk over the cache, and the verification of
 * drafted tokens. No counterpart in the reference, whose cache is one contiguous f32 buffer per
 * sequence and whose chunks are two tokens: these run the same layer (linears of g4w8a8.h, norms and
 * head of g4decode.h) for a batch of sequences of different lengths.
 *
 * Conventions as g4w8a8.h: device pointers, G4_OK or a G4_ERR_* status with g4_last_error(),
 * `stream` NULL = the default stream, launches only (no allocation, no host synchronisation), so
 * every call can be graph-captured. The current device is the one the stream and the buffers belong
 * to. A workspace belongs to one call at a time: calls (or replays of captured graphs) that can run
 * at the same time need one each. It needs no initial contents.
 */
#ifndef G4SERVE_H
#define G4SERVE_H

#include "g4w8a8.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * One layer's pages. K and V have `num_pages` pages of `page_size` slots each; a slot holds
 * kv_heads rows of head_dim. Row (page, slot, head) of K starts at element
 * page * page_stride + slot * slot_stride + head * head_stride of k, of V at the same element of v;
 * so [page][slot][head][dim] and [page][head][slot][dim] pools are both served. All three strides 0:
 * [page][slot][head][dim], packed.
 * kind G4_KIND_F16: the rows are f16. kind G4_KIND_I8: int8 codes, and k_scales / v_scales hold one
 * f32 per row, [page][head][slot], packed; the row's values are code * scale.
 * head_dim 64, 128 or 256; page_size a power of two from 8 to 4096; k and v 16-byte aligned and the
 * strides multiples of 16 bytes.
 */
typedef struct g4_kv_pages {
    void *k, *v;
    float *k_scales, *v_scales; /* G4_KIND_I8 only */
    int kind;
    int num_pages;
    int page_size;
    int kv_heads;
    int head_dim;
    int64_t page_stride, slot_stride, head_stride; /* elements */
} g4_kv_pages;

/*
 * A chunk: the new tokens of a batch of sequences. Sequence s has rows q_start[s] .. q_start[s + 1] of
 * the chunk's [tokens] rows, and kv_len[s] positions in the cache once these are in it; row i of the
 * sequence is position kv_len[s] - (its rows) + i. Position p lives in slot p % page_size of page
 * page_table[s * table_stride + p / page_size]. A page outside [0, num_pages) is absent (a page that
 * a window has left behind, for example): nothing is stored there and it holds no keys.
 * q_start, kv_len and page_table are read when the kernels run. max_q and max_kv bound a sequence's
 * rows and its kv_len (they size grids and workspaces): rows from max_q on are left out, and a longer
 * kv_len counts as max_kv.
 * q_start must ascend; rows behind q_start[seqs] belong to no sequence and their outputs are left as
 * they were. A row at a negative position (more rows than positions) is not stored and sees no keys.
 */
typedef struct g4_chunk {
    int seqs;
    int tokens;
    int max_q;
    int max_kv;
    const int32_t *q_start;    /* [seqs + 1] */
    const int32_t *kv_len;     /* [seqs] */
    const int32_t *page_table; /* [seqs][table_stride], table_pages entries of each row in use */
    int table_pages;           /* table_pages * page_size >= max_kv */
    int64_t table_stride;      /* 0: table_pages */
} g4_chunk;

/*
 * g4_attn_prologue for a chunk: q = rope(rms_norm(q, q_gain)), k = rope(rms_norm(k, k_gain)) and the
 * weightless v = rms_norm(v), the rows of a projection in (x_kind G4_KIND_F32, _F16, or _I8 codes times
 * q_scale / k_scale / v_scale), q out as f16 rows [tokens][heads][head_dim], k and v stored at their
 * positions of the cache. Rows of q, k and v start q_stride / k_stride / v_stride elements apart
 * (0: packed), so the three may be parts of one projection's output.
 *  - q NULL (with heads 0): only the store. k and v NULL: only the queries (a layer that reads another
 *    layer's cache).
 *  - q_gain / k_gain NULL: that side is not normalised (v goes with k).
 *  - cos_tab / sin_tab [rope_positions][head_dim / 2] (the split-half form): NULL: no rotation;
 *    else rope_positions >= max_kv.
 * An int8 cache row: scale = f32(amax / 127) with amax the largest magnitude of the f32 row, code =
 * RNE(127 * y / amax), exactly rounded; a zero row has scale 0, a row with an infinity or a NaN has
 * scale NaN and codes 0. An f16 row is rounded to nearest even (past the f16 range: infinity).
 * Two rows of a chunk must not share a position of the cache. At most 2^26 - 4 head rows (tokens times the heads of
 * q, k and v that are given).
 */
int g4_paged_prologue(const g4_kv_pages *pages, const g4_chunk *chunk, int x_kind, const void *q,
                      int64_t q_stride, float q_scale, const void *k, int64_t k_stride, float k_scale,
                      const void *v, int64_t v_stride, float v_scale, int heads, const float *q_gain,
                      const float *k_gain, const float *cos_tab, const float *sin_tab,
                      int rope_positions, float eps, void *q_out, void *stream);

/*
 * The chunk's rows read back from the cache: row i of sequence s to
 * out + (seq_stride ? s * seq_stride + i * kv_heads * head_dim
 *                   : (q_start[s] + i) * kv_heads * head_dim), f32 (code * scale rounded once) or that as f16. With
 * q_start counting every position of a sequence (its rows = kv_len[s]) the whole sequence is read,
 * for example into a contiguous f32 cache (g4_decode_kv). Rows on absent pages are zeros. k_out or
 * v_out may be NULL; both 16-byte aligned, seq_stride a multiple of 16 bytes. At most 2^28 - 16 rows.
 */
int g4_kv_read(const g4_kv_pages *pages, const g4_chunk *chunk, void *k_out, void *v_out, int out_kind,
               int64_t seq_stride, void *stream);

/*
 * Causal attention of the chunk's rows over the cache (which holds the chunk already): row at position
 * p of its sequence sees the positions j <= p, with window > 0 only j > p - window;
 *   out = sum_j softmax_j(scale * q . k_j) v_j.
 * q: f16 rows [tokens][heads][head_dim], q_stride elements apart (0: packed), 16-byte aligned; heads a
 * multiple of kv_heads (query heads h * heads / kv_heads .. share KV head h). out [tokens][heads]
 * [head_dim], packed: G4_KIND_F16, G4_KIND_F32, or G4_KIND_I8: the consumer's input codes on in_scale
 * (quant.ts:309-334 srqCodes). A row that sees no key is zeros.
 * f16 rows: products of f16 values, added up in f32; a weight is rounded to f16 (relative to a maximum
 * within 2^8 of the row's), and the softmax's sum adds the rounded ones. int8 rows: q enters the scores as
 * 16-bit fixed point of the row's largest magnitude (off by 2^-16 of that at most) and the codes exactly;
 * a weight is rounded to f16 with V's scale in it (scales up to 2^99 in magnitude, K's to 2^96), relative to a power of
 * two of at most 4 times the row's largest such product. A masked position's contents, NaN included, change nothing.
 * Of what a row sees: a NaN or an infinity in V, and a score that is NaN or +infinity, make its outputs non-finite; a
 * score of -infinity has no weight. A NaN or an infinity in q makes an int8 row's outputs non-finite where it sees a key.
 * page_stride and page_size * slot_stride below 2^31 elements; |scale| below 2^127.
 * workspace: g4_attention_chunk_workspace_bytes(...) bytes, 16-byte aligned.
 */
int g4_attention_chunk(const g4_kv_pages *pages, const g4_chunk *chunk, const void *q, int64_t q_stride,
                       int heads, float scale, int window, void *workspace, size_t workspace_bytes,
                       void *out, int out_kind, float in_scale, void *stream);
size_t g4_attention_chunk_workspace_bytes(const g4_kv_pages *pages, const g4_chunk *chunk, int heads,
                                          int window);

/*
 * Verification of drafted tokens: sequence s drafted draft_tokens[draft_start[s] .. draft_start[s + 1]],
 * n of them (at most max_drafts <= 63), and the target model ran over its last token and the drafts,
 * which gave the n + 1 rows of logits from row draft_start[s] + s on. With y = tanh(x / cap) * cap (cap 0: y = x) and
 * p = softmax(y / temperature), q likewise of the drafter's logits:
 *   draft i is taken while u[i] * q_i(t_i) < p_i(t_i);
 *   the first draft refused is replaced by a draw from max(p_i - q_i, 0) (from p_i where that is 0
 *   everywhere), and when all are taken one more token is drawn from p_n: the first token whose running
 *   sum of weights, in token order, exceeds u_next[s] * their sum.
 * draft_logits NULL: a drafter without probabilities, q_i = 1 at t_i. temperature 0: greedy, draft i is
 * taken while it is the first maximum of row i (u, u_next and draft_logits are not read). That is the maximum of the
 * logits as given, whose order the cap keeps. g4_softcap_argmax compares capped f32 values: where it finds another
 * token, that one is earlier and its logit so near the maximum, or both so far past the cap, that they are capped alike.
 * A logit that is NaN or -infinity (a token masked out) has no weight, under a cap too (tanh alone would leave a
 * masked token e^(-cap / temperature)); a drafted id outside the vocabulary is refused; a row without any weight
 * gives token -1 and log probability 0.
 * Out: tokens [seqs][max_drafts + 1]: the drafts taken, the drawn token, then -1; accepted [seqs]; logprobs
 * (optional) [seqs][max_drafts + 1]: log p of each token under the target at the temperature (1 when
 * greedy), 0 past the drawn one.
 * drafts: the length of draft_tokens and u (draft_start is clamped to it); logits has drafts + seqs rows
 * of vocab f32, draft_logits drafts rows. u and u_next in [0, 1).
 * workspace: g4_verify_workspace_bytes(...) bytes, 16-byte aligned.
 */
int g4_verify_drafts(const float *logits, const float *draft_logits, const int32_t *draft_tokens,
                     const int32_t *draft_start, int seqs, int drafts, int max_drafts, int64_t vocab,
                     float cap, float temperature, const float *u, const float *u_next,
                     void *workspace, size_t workspace_bytes, int32_t *tokens, int32_t *accepted,
                     float *logprobs, void *stream);
size_t g4_verify_workspace_bytes(int seqs, int drafts, int64_t vocab);

#ifdef __cplusplus
}
#endif

#endif /* G4SERVE_H */
