/*
 * g4serve.h - serving operators on a paged KV cache: the plan of a chunk of new tokens (pages, block
 * tables, slot maps), its prologue with the quantising store, the read-back, attention of the chunk over
 * the cache, per-request low-rank adapters beside the linears, the verification of drafted tokens, and
 * sampling. No counterpart in the reference, whose cache is one contiguous f32 buffer per
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

/*
 * Pages that no sequence holds: the first *count of `pages` (a count outside [0, capacity] is clamped).
 * A step reads the count and writes the new one elsewhere, so that the step after it can be enqueued
 * before this one has run: two count words (and two `held` arrays, below) in turn.
 */
typedef struct g4_free_pages {
    int32_t *pages;       /* [capacity] ids */
    const int32_t *count; /* [1] */
    int capacity;
    int num_pages; /* of the pools */
    int page_size; /* a power of two from 8 to 4096 */
} g4_free_pages;

/*
 * The plan of a chunk from the requests' lengths: the arrays of g4_chunk, the pages of the new positions, and where
 * each row goes. Sequence s has c = cached[s] positions (clamped to [0, max_kv]) and asks for n = rows[s] new ones
 * (clamped to [0, min(max_q, max_kv - c)]). held[s] entries of its row of page_table have been given, from the first on
 * (held NULL: those that c positions need), and it needs max(0, ceil((c + n) / page_size) - held[s]) more where n > 0, which
 * go behind them. Entry p / page_size is position p's whatever went back in the meantime: pages that a window has left
 * behind stay counted in held, and only a request that ended has its held set back.
 * Sequences are served in order, while their rows fit into `tokens` and their pages into the free ones: from the first
 * that does not fit on, all get no rows and no pages in this chunk. served: how many fit.
 * The pages given are the last ones of the free list, in the list's order: by sequence, then by position.
 * Out: q_start [seqs + 1], kv_len [seqs] (c + the rows given), free_left [1] and served [1], the new entries of
 * page_table (no other entry is touched); optional (NULL): held_out [seqs], last_row [seqs] (q_start[s + 1] - 1, -1
 * without rows: the row of g4_sample_tokens), and of each of the `tokens` rows its position row_pos, its cache slot
 * row_slot (page * page_size + position % page_size, -1 on an absent page) and its adapter row_adapter
 * (seq_adapter[s], -1 where that is NULL). Rows behind the last sequence: -1, -1 and -2.
 * No output may be the free list's count, cached, rows, held or seq_adapter: those are read throughout.
 * At most 4096 sequences, and num_pages * page_size below 2^31.
 */
int g4_plan_chunk(const g4_free_pages *list, const int32_t *cached, const int32_t *rows, const int32_t *held,
                  const int32_t *seq_adapter, int seqs, int tokens, int max_q, int max_kv, int32_t *page_table,
                  int table_pages, int64_t table_stride, int32_t *q_start, int32_t *kv_len, int32_t *held_out,
                  int32_t *free_left, int32_t *served, int32_t *row_pos, int32_t *row_slot, int32_t *row_adapter,
                  int32_t *last_row, void *stream);

/*
 * Pages back to the free list: entries first[s] .. last[s] - 1 of every sequence's row of page_table (clamped to
 * [0, table_pages]) are appended to the free pages, by sequence, then by position; count_out is the new count. Absent
 * entries, outside [0, num_pages), are left out, and pages that would pass the list's capacity dropped.
 * page_table and held stay as they are. An entry must not be released twice, nor one that two sequences share, nor one behind
 * held[s], where an earlier request's may still stand. So the user keeps, a request, the entry that the next release begins at:
 * 0 at first; a window that no later row reaches behind position p gives back up to p / page_size, which is the next first;
 * a finished request gives back up to held[s], and both are 0 again.
 * count_out must not be the list's count, which is the one that the plan or release before has left. At most 4096 sequences.
 */
int g4_release_pages(const g4_free_pages *list, const int32_t *page_table, int table_pages, int64_t table_stride,
                     const int32_t *first, const int32_t *last, int seqs, int32_t *count_out, void *stream);

/*
 * Low-rank adapters of one linear, f16: adapter i adds scales[i] * (x A_i^T) B_i^T to its rows.
 * A_i = a + i * a_stride, [max_rank][k]; B_i = b + i * b_stride, [n][max_rank] (strides in elements, 0: packed). ranks
 * (NULL: max_rank for all): adapter i has ranks[i] (clamped to [0, max_rank]) rows of A_i and columns of B_i; what lies
 * behind them is not used, whatever it holds. k and max_rank multiples of 8, k up to 2^23, max_rank to 128 and n to 2^30;
 * at most 4096 adapters; a and b 16-byte aligned, the strides multiples of 8.
 */
typedef struct g4_adapters {
    const void *a, *b;
    const float *scales;  /* [count], NULL: 1 */
    const int32_t *ranks; /* [count] or NULL */
    int count, max_rank, k, n;
    int64_t a_stride, b_stride;
} g4_adapters;

/*
 * The rows of a batch grouped by their adapter, once for every linear of a step: row_adapter [tokens] (of g4_plan_chunk,
 * for example) into `groups`, g4_adapter_groups_bytes(...) bytes, 16-byte aligned. An id in [0, adapters) is that
 * adapter, -2 no row (its outputs are left as they were), any other one no adapter. At most 2^19 tokens.
 */
int g4_adapter_groups(const int32_t *row_adapter, int tokens, int adapters, void *groups, size_t groups_bytes,
                      void *stream);
size_t g4_adapter_groups_bytes(int tokens, int adapters);

/*
 * A linear's output with its rows' adapters added:
 *   out[t] = base[t] + scales[i] * ((x[t] A_i^T) B_i^T), i the row's adapter, and base[t] for a row without one.
 * x [tokens][k] is the linear's input: f32, f16, or int8 codes times x_scale; base [tokens][n] what the shared
 * linear gave: f32, f16, or int8 codes times base_scale, or NULL (zeros). out: f32, f16, or int8 codes on out_scale;
 * out_scale != 0 snaps f32 and f16 outputs to that grid too, as g4_linear does (a f32 output code * out_scale; the
 * quotient's clamp takes a NaN to -128). Rows start x_stride, base_stride and out_stride elements apart (0: packed); x 16-byte
 * aligned, x_stride a multiple of 16 bytes (codes: of 8). out may be base, of the same type and stride, and not x.
 * groups: of g4_adapter_groups, for the same tokens and number of adapters (of others: nothing is written).
 * x A^T is made of exact products, added up in f32, and enters the second product with 23 bits, relative to its row's
 * largest value; that product's sums are f32 too.
 * workspace: g4_adapter_workspace_bytes(...) bytes, 16-byte aligned, apart from groups, which are read throughout.
 */
int g4_adapter_linear(const g4_adapters *adapters, const void *groups, size_t groups_bytes, int tokens, const void *x,
                      int x_kind, int64_t x_stride, float x_scale, const void *base, int base_kind, int64_t base_stride,
                      float base_scale, void *out, int out_kind, int64_t out_stride, float out_scale, void *workspace,
                      size_t workspace_bytes, void *stream);
size_t g4_adapter_workspace_bytes(const g4_adapters *adapters, int tokens);

/*
 * Sampling: one token for each of `rows` requests, from given random numbers. Request i reads row row_index[i] of
 * logits (NULL: row i; several may read one row), logit_rows rows of vocab f32 that start logit_stride elements apart
 * (0: packed). With y = tanh(x / cap) * cap (cap 0: y = x) and w = exp((y - max y) / temperature[i]), the row's tokens are
 * ordered by their logits, the lower id first among equal ones, and each filter keeps a part of what the one before it left:
 *   top_k[i]: the first top_k (0 or less, or vocab or more: all);
 *   top_p[i]: those before which the sum of weights is under top_p * the sum of all that top_k left, and the
 *             first one always (1 or more: all);
 *   min_p[i]: those with w >= min_p (0 or less: all; more than 1 counts as 1).
 * The token drawn is the first, in token order, where the running sum of the kept weights exceeds u[i] * their sum.
 * A temperature that is not above 0 (NaN too) is greedy: the first maximum. A NULL array: temperature 1, the filter off; a NaN
 * in one turns the filter off. A logit that is NaN or -infinity has no weight. A row without any, or a row_index outside
 * [0, logit_rows), gives token -1 and log probability 0. u in [0, 1) (clamped to it, NaN: 0).
 * logprobs (optional): (y - max y) / temperature - log(the sum of all weights), before the filters (greedy: at 1).
 * Weights are counted in whole steps of 2^-min(51, 62 - ceil(log2 vocab)) of the row's largest (2^-44 for
 * 262144 tokens) and added up exactly, so that a result does not depend on the order of the additions; what rounds to
 * no step is not drawn. vocab up to 2^22, at most 65535 rows.
 * workspace: g4_sample_workspace_bytes(...) bytes, 16-byte aligned.
 */
int g4_sample_tokens(const float *logits, int logit_rows, int64_t logit_stride, const int32_t *row_index, int rows,
                     int64_t vocab, float cap, const float *temperature, const int32_t *top_k, const float *top_p,
                     const float *min_p, const float *u, void *workspace, size_t workspace_bytes, int32_t *tokens,
                     float *logprobs, void *stream);
size_t g4_sample_workspace_bytes(int rows, int64_t vocab);

#ifdef __cplusplus
}
#endif

#endif /* G4SERVE_H */
