// The paged cache as the serving kernels see it (include/g4serve.h): the checked arguments, and the
// lookups from a chunk row to its sequence and from a position to its page.
#pragma once

#include "g4_internal.h"
#include "../../include/g4serve.h"

namespace g4 {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

struct PagedArgs {
    void *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;
    int64_t page_stride = 0, slot_stride = 0, head_stride = 0;
    const int32_t *table = nullptr;
    int64_t table_stride = 0;
    const int32_t *q_start = nullptr, *kv_len = nullptr;
    int seqs = 0, tokens = 0, max_q = 0, max_kv = 0;
    int kv_heads = 0, page_shift = 0, num_pages = 0;
};

// Checks the cache and the chunk and lays them out for a kernel (kv_paged.hip).
int paged_args(const char *who, const g4_kv_pages *pages, const g4_chunk *chunk, PagedArgs *out);

// Rows of sequence `seq` (a call leaves out those from max_q on) and its final length, clamped to max_kv.
struct SeqSpan {
    int start, rows, kv;
};

__device__ __forceinline__ SeqSpan seq_span(const PagedArgs &A, int seq) {
    const int a = min(max(A.q_start[seq], 0), A.tokens);
    const int b = min(max(A.q_start[seq + 1], a), A.tokens);
    return {a, b - a, min(max(A.kv_len[seq], 0), A.max_kv)};
}

// The sequence that chunk row `row` (the same in every lane) belongs to: the number of sequences that
// end at or before it, 64 ends per load instead of a search of dependent loads. seqs: none.
__device__ __forceinline__ int seq_of_row(const PagedArgs &A, int row) {
    const int lane = threadIdx.x & 63;
    int seq = 0;
    for (int base = 0; base < A.seqs; base += 64) {
        const int s = base + lane;
        const bool past = s < A.seqs && A.q_start[s + 1] <= row;
        const int n = __popcll(__ballot(past));
        seq += n;
        if (n < 64) break;
    }
    return seq;
}

// The page of position p (0 <= p < max_kv) of sequence seq, or -1 where it is absent.
__device__ __forceinline__ int page_of(const PagedArgs &A, int seq, int p) {
    const int page = A.table[seq * A.table_stride + (p >> A.page_shift)];
    return (unsigned)page < (unsigned)A.num_pages ? page : -1;
}

__device__ __forceinline__ int64_t row_offset(const PagedArgs &A, int page, int p, int head) {
    return (int64_t)page * A.page_stride + (int64_t)(p & ((1 << A.page_shift) - 1)) * A.slot_stride +
           (int64_t)head * A.head_stride;
}

__device__ __forceinline__ int64_t scale_offset(const PagedArgs &A, int page, int p, int head) {
    return (((int64_t)page * A.kv_heads + head) << A.page_shift) + (p & ((1 << A.page_shift) - 1));
}

}  // namespace g4
