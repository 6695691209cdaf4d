// The plan of a chunk and the release of pages (include/g4serve.h): prefix sums over the requests' rows
// and pages, then one item per chunk row and per page.
//
// No block waits for another: each computes the prefix sums of all sequences (at most 4096, a few loads a
// thread) into LDS and finds its items' sequences there by binary search. That is why a call's counts are
// read from other arrays than it writes. Release counts the pages in front of a block's entries in the same way.
#include "g4_internal.h"
#include "../../include/g4serve.h"

namespace g4 {

constexpr int kPlanSeqs = 4096, kPlanThreads = 256;
// Blocks of a kind, two a CU; more items go round, since every block sums all sequences up.
constexpr int kPlanBlocks = 512;
// Release: 512 threads a block start and meet sooner than 1024 (16 requests of up to 256 pages 4.0 and 5.1 us replayed), and read
// nearly as fast (1024 of up to 1024 pages 46.6 and 40.2).
constexpr int kReleaseLog = 9, kReleaseThreads = 1 << kReleaseLog, kReleaseBlocks = 256;

struct PlanArgs {
    int32_t *free_pages;
    const int32_t *count, *cached, *rows, *held, *seq_adapter;
    int32_t *table;
    int64_t table_stride;
    int32_t *q_start, *kv_len, *held_out, *free_left, *served, *row_pos, *row_slot, *row_adapter, *last_row;
    int capacity, num_pages, page_shift, seqs, tokens, max_q, max_kv, table_pages;
};

// What sequence s asks for, before it is known whether it is served.
struct Wish {
    int cached, rows, held, need;
};

__device__ __forceinline__ Wish wish_of(const PlanArgs &A, int s) {
    Wish w;
    w.cached = min(max(A.cached[s], 0), A.max_kv);
    w.rows = min(max(A.rows[s], 0), min(A.max_q, A.max_kv - w.cached));
    const int last = (1 << A.page_shift) - 1;
    // positions are below table_pages pages, which fit in 32 bits with a page to spare
    const int now = (int)(((int64_t)w.cached + last) >> A.page_shift);
    const int then = (int)(((int64_t)w.cached + w.rows + last) >> A.page_shift);
    w.held = A.held ? min(max(A.held[s], 0), A.table_pages) : now;
    w.need = w.rows > 0 ? max(then - w.held, 0) : 0;
    return w;
}

struct Pair {
    int64_t rows, pages;
};

// Exclusive sum over the block's threads of v; *total: of all. Once a kernel.
template <int THREADS>
__device__ __forceinline__ Pair block_before(Pair v, Pair *total) {
    __shared__ Pair sums[THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Pair run = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int64_t r = __shfl_up((long long)run.rows, s), p = __shfl_up((long long)run.pages, s);
        if (lane >= s) {
            run.rows += r;
            run.pages += p;
        }
    }
    if (lane == 63) sums[wave] = run;
    __syncthreads();
    Pair before{run.rows - v.rows, run.pages - v.pages}, all{0, 0};
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        const Pair s = sums[w];
        if (w < wave) {
            before.rows += s.rows;
            before.pages += s.pages;
        }
        all.rows += s.rows;
        all.pages += s.pages;
    }
    *total = all;
    return before;
}

// The last s with start[s] <= i of an ascending start[0 .. n], for i < start[n].
template <class T>
__device__ __forceinline__ int owner(const T *start, int n, T i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (start[mid] <= i ? lo : hi) = mid;
    }
    return lo;
}

// Bound by its chain of dependent steps: count and lengths, a block sum, a search in LDS, a page, the stores (256 requests
// of 1 to 8 rows 6.4 us, 64 prompts of up to 2048 6.2). One item a thread, the rows' blocks first, then the pages', then
// the sequences'.
__global__ __launch_bounds__(kPlanThreads) void plan_chunk_kernel(PlanArgs A, int row_blocks, int page_blocks) {
    extern __shared__ int32_t plan_lds[];
    __shared__ int fit;
    int32_t *start = plan_lds, *pages = start + A.seqs + 1, *cached = pages + A.seqs + 1;
    const int t = threadIdx.x, per = (A.seqs + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(t * per, A.seqs), s1 = min(s0 + per, A.seqs);
    const int count = min(max(*A.count, 0), A.capacity);
    if (t == 0) fit = 0;
    Pair mine{0, 0}, all;
    for (int s = s0; s < s1; ++s) {
        const Wish w = wish_of(A, s);
        mine.rows += w.rows;
        mine.pages += w.need;
        cached[s] = w.cached;
    }
    Pair at = block_before<kPlanThreads>(mine, &all);
    int fits = 0;
    for (int s = s0; s < s1; ++s) {
        const Wish w = wish_of(A, s);
        // of a sequence that is not served nothing is read but whether it is
        start[s] = (int)min(at.rows, (int64_t)A.tokens);
        pages[s] = (int)min(at.pages, (int64_t)count);
        at.rows += w.rows;
        at.pages += w.need;
        if (at.rows <= A.tokens && at.pages <= count) {
            ++fits;
            start[s + 1] = (int)at.rows;  // the next thread writes the same, or is not served
            pages[s + 1] = (int)at.pages;
        }
    }
    if (fits) atomicAdd(&fit, fits);
    __syncthreads();
    const int served = fit;
    const int total_rows = start[served], total_pages = pages[served], left = count - total_pages;
    const int last = (1 << A.page_shift) - 1;
    // where the new pages of served sequence s begin in its row of the table
    auto first_new = [&](int s) {
        const int then = (int)(((int64_t)cached[s] + (start[s + 1] - start[s]) + last) >> A.page_shift);
        return then - (pages[s + 1] - pages[s]);
    };
    int block = blockIdx.x;
    if (block < row_blocks) {
        for (int64_t i = (int64_t)block * kPlanThreads + t; i < A.tokens; i += (int64_t)row_blocks * kPlanThreads) {
            int pos = -1, slot = -1, adapter = -2;
            if (i < total_rows) {
                const int s = owner(start, served, (int32_t)i);
                adapter = A.seq_adapter && A.row_adapter ? A.seq_adapter[s] : -1;
                pos = cached[s] + ((int)i - start[s]);
                if (A.row_slot) {
                    const int p = pos >> A.page_shift, from = first_new(s);
                    // (a sequence's last page is its last new one, if it has any)
                    const bool is_new = p >= from && pages[s + 1] > pages[s];
                    const int page = is_new ? A.free_pages[left + pages[s] + (p - from)] : A.table[s * A.table_stride + p];
                    if ((unsigned)page < (unsigned)A.num_pages) slot = (page << A.page_shift) + (pos & last);
                }
            }
            if (A.row_pos) A.row_pos[i] = pos;
            if (A.row_slot) A.row_slot[i] = slot;
            if (A.row_adapter) A.row_adapter[i] = adapter;
        }
        return;
    }
    block -= row_blocks;
    if (block < page_blocks) {
        for (int64_t i = (int64_t)block * kPlanThreads + t; i < total_pages; i += (int64_t)page_blocks * kPlanThreads) {
            const int s = owner(pages, served, (int32_t)i);
            A.table[s * A.table_stride + first_new(s) + ((int)i - pages[s])] = A.free_pages[left + i];
        }
        return;
    }
    block -= page_blocks;
    for (int s = block * kPlanThreads + t; s < A.seqs; s += kPlanSeqs) {
        const Wish w = wish_of(A, s);
        const bool in = s < served;
        A.q_start[s + 1] = in ? start[s + 1] : total_rows;
        A.kv_len[s] = w.cached + (in ? w.rows : 0);
        if (A.held_out) A.held_out[s] = w.held + (in ? w.need : 0);
        if (A.last_row) A.last_row[s] = in && w.rows ? start[s + 1] - 1 : -1;
    }
    if (block == 0 && t == 0) {
        A.q_start[0] = 0;
        *A.free_left = left;
        *A.served = served;
    }
}

struct ReleaseArgs {
    int32_t *free_pages;
    const int32_t *count, *table, *first, *last;
    int64_t table_stride;
    int32_t *count_out;
    int capacity, num_pages, seqs, table_pages;
};

__device__ __forceinline__ int2 range_of(const ReleaseArgs &A, int s) {
    const int a = min(max(A.first[s], 0), A.table_pages);
    return make_int2(a, max(min(A.last[s], A.table_pages), a));
}

// 2^grid_log blocks have equal runs of the ranges' entries, a tile of an entry a thread at a time. Absent entries are left
// out, so where a block's pages go depends on how many of those stand in front of its own: it reads all that do. Bound by its
// chain, count, ranges, a block sum, a search, an entry, those in front, a block sum, the store: 16 requests of 170 pages
// 4.0 us replayed, 1000 of which most give back one 5.0; past some 50000 pages by the last block's reads (100074 pages
// 10 us, 655842 46; 3.4 and 9.1 if nobody looked for absent ones).
__global__ __launch_bounds__(kReleaseThreads) void release_pages_kernel(ReleaseArgs A, int grid_log) {
    extern __shared__ int64_t release_lds[];
    __shared__ int wave_absent[kReleaseThreads / 64], wave_pages[kReleaseThreads / 64];
    int64_t *start = release_lds;  // of each request's entries among all
    int32_t *from = reinterpret_cast<int32_t *>(start + A.seqs + 1);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, per = (A.seqs + kReleaseThreads - 1) / kReleaseThreads;
    const int s0 = min(t * per, A.seqs), s1 = min(s0 + per, A.seqs);
    const int count = min(max(*A.count, 0), A.capacity);
    Pair n{0, 0}, all;
    for (int s = s0; s < s1; ++s) {
        const int2 r = range_of(A, s);
        from[s] = r.x;
        start[s] = n.pages;
        n.pages += r.y - r.x;
    }
    const int64_t before = block_before<kReleaseThreads>(n, &all).pages, total = all.pages;
    for (int s = s0; s < s1; ++s) start[s] += before;
    if (t == 0) start[A.seqs] = total;
    __syncthreads();
    const int64_t tiles = (total + kReleaseThreads - 1) / kReleaseThreads;
    const int64_t run = ((tiles + (1 << grid_log) - 1) >> grid_log) * kReleaseThreads;
    const int64_t begin = blockIdx.x * run, end = min(begin + run, total);
    if (begin >= total && (blockIdx.x || total)) return;
    auto page_at = [&](int64_t i) {
        if (i >= end) return -1;
        const int s = owner(start, A.seqs, i);
        return A.table[s * A.table_stride + from[s] + (i - start[s])];
    };
    auto is_page = [&](int page) { return (unsigned)page < (unsigned)A.num_pages; };
    int page = page_at(begin + t);
    int absent = 0;  // in front
    if (begin) {
        // a request's entries by 2^group_log threads: what there is for each, or for its average number to be four loads
        int group_log = 0;
        while (group_log < kReleaseLog &&
               ((A.seqs << (group_log + 1)) <= kReleaseThreads || ((int64_t)A.seqs << (group_log + 5)) <= total))
            ++group_log;
        const int rows = owner(start, A.seqs, begin - 1) + 1;
        const uint32_t step = 4 << group_log, mine = 4 * (t & ((1 << group_log) - 1));
        for (int s = t >> group_log; s < rows; s += kReleaseThreads >> group_log) {
            const uint32_t len = (uint32_t)(min(begin, start[s + 1]) - start[s]);
            const int32_t *row = A.table + s * A.table_stride + from[s];
            if (len < 4) {
                for (uint32_t i = mine; i < len; ++i) absent += !is_page(row[i]);
                continue;
            }
            for (uint32_t i = mine; i < len; i += 4 * step) {
                int32_t e[4][4];
                uint32_t most = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u)  // the last four where fewer are left
                    __builtin_memcpy(e[u], row + min(i + u * step, len - 4), sizeof e[u]);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) most = max(most, (uint32_t)e[u][j]);
                if (is_page(most)) continue;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // (what is not this thread's is not counted)
                        absent += min(i + u * step, len - 4) + j >= i + u * step && !is_page(e[u][j]);
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) absent += __shfl_xor(absent, o);
    }
    if (lane == 0) wave_absent[wave] = absent;
    int64_t at = count + begin;
    for (int64_t i = begin; i < end; i += kReleaseThreads) {
        const bool is = is_page(page);
        const unsigned long long who = __ballot(is);
        if (lane == 0) wave_pages[wave] = __popcll(who);
        __syncthreads();
        int waves_before = 0, tile = 0;
#pragma unroll
        for (int w = 0; w < kReleaseThreads / 64; ++w) {
            if (i == begin) at -= wave_absent[w];
            waves_before += w < wave ? wave_pages[w] : 0;
            tile += wave_pages[w];
        }
        const int64_t to = at + waves_before + __popcll(who & ((1ull << lane) - 1));
        if (is && to < A.capacity) A.free_pages[to] = page;
        at += tile;
        if (i + kReleaseThreads < end) {
            page = page_at(i + kReleaseThreads + t);
            __syncthreads();
        }
    }
    if (t == 0 && end == total) *A.count_out = (int)min(at, (int64_t)A.capacity);
}

static int check_list(const char *who, const g4_free_pages *L) {
    if (!L || !L->pages || !L->count) return set_error(G4_ERR_INVALID, "%s needs the free pages and their count", who);
    if (L->capacity <= 0 || L->num_pages <= 0)
        return set_error(G4_ERR_INVALID, "%s: a free list of %d of %d pages", who, L->capacity, L->num_pages);
    if (L->page_size < 8 || L->page_size > 4096 || (L->page_size & (L->page_size - 1)))
        return set_error(G4_ERR_INVALID, "%s: page_size %d is not a power of two from 8 to 4096", who, L->page_size);
    if ((int64_t)L->num_pages * L->page_size > INT32_MAX)
        return set_error(G4_ERR_UNSUPPORTED, "%s: %d pages of %d slots (slots are 32-bit)", who, L->num_pages, L->page_size);
    return G4_OK;
}

static int check_table(const char *who, const void *table, int table_pages, int64_t table_stride, int seqs) {
    if (!table || seqs <= 0 || table_pages <= 0)
        return set_error(G4_ERR_INVALID, "%s: %d sequences, %d table pages", who, seqs, table_pages);
    if (seqs > kPlanSeqs)
        return set_error(G4_ERR_UNSUPPORTED, "%s: %d sequences in one call (at most %d)", who, seqs, kPlanSeqs);
    if (table_stride && table_stride < table_pages)
        return set_error(G4_ERR_INVALID, "%s: table_stride %lld < %d table pages", who, (long long)table_stride, table_pages);
    return G4_OK;
}

static int plan_blocks(int64_t items) {
    const int64_t n = (items + kPlanThreads - 1) / kPlanThreads;
    return (int)(n < 1 ? 1 : n > kPlanBlocks ? kPlanBlocks : n);
}

}  // namespace g4

using namespace g4;

extern "C" {

int g4_plan_chunk(const g4_free_pages *list, const int32_t *cached, const int32_t *rows, const int32_t *held,
                  const int32_t *seq_adapter, int seqs, int tokens, int max_q, int max_kv, int32_t *page_table,
                  int table_pages, int64_t table_stride, int32_t *q_start, int32_t *kv_len, int32_t *held_out,
                  int32_t *free_left, int32_t *served, int32_t *row_pos, int32_t *row_slot, int32_t *row_adapter,
                  int32_t *last_row, void *stream) {
    if (int st = check_list("plan-chunk", list)) return st;
    if (int st = check_table("plan-chunk", page_table, table_pages, table_stride, seqs)) return st;
    if (!cached || !rows || !q_start || !kv_len || !free_left || !served)
        return set_error(G4_ERR_INVALID, "plan-chunk needs cached, rows, q_start, kv_len, free_left and served");
    if (tokens <= 0 || max_q <= 0 || max_kv <= 0)
        return set_error(G4_ERR_INVALID, "plan-chunk: %d tokens, max_q %d, max_kv %d", tokens, max_q, max_kv);
    if ((int64_t)table_pages * list->page_size < max_kv)
        return set_error(G4_ERR_INVALID, "plan-chunk: %d table pages of %d slots do not hold max_kv %d positions", table_pages,
                         list->page_size, max_kv);
    for (const int32_t *in : {list->count, cached, rows, held, seq_adapter})
        for (const int32_t *out : {q_start, kv_len, held_out, free_left, served, row_pos, row_slot, row_adapter, last_row})
            if (in && in == out)
                return set_error(G4_ERR_INVALID, "plan-chunk: outputs cannot be the arrays they are made from");
    PlanArgs A{list->pages, list->count, cached, rows, held, seq_adapter, page_table,
               table_stride ? table_stride : table_pages, q_start, kv_len, held_out, free_left, served, row_pos, row_slot,
               row_adapter, last_row, list->capacity, list->num_pages, __builtin_ctz(list->page_size), seqs, tokens, max_q,
               max_kv, table_pages};
    const size_t lds = (3 * (size_t)seqs + 2) * sizeof(int32_t);
    const bool per_row = row_pos || row_slot || row_adapter;
    // a sequence's rows open a page each page_size of them, and one more; more pages (not held, though cached) go round
    const int row_blocks = per_row ? plan_blocks(tokens) : 0, page_blocks = plan_blocks((int64_t)tokens / list->page_size + seqs);
    hipLaunchKernelGGL(plan_chunk_kernel, dim3(row_blocks + page_blocks + plan_blocks(seqs)), dim3(kPlanThreads), lds,
                       as_stream(stream), A, row_blocks, page_blocks);
    G4_LAUNCHED("plan_chunk_kernel");
    return G4_OK;
}

int g4_release_pages(const g4_free_pages *list, const int32_t *page_table, int table_pages, int64_t table_stride,
                     const int32_t *first, const int32_t *last, int seqs, int32_t *count_out, void *stream) {
    if (int st = check_list("release-pages", list)) return st;
    if (int st = check_table("release-pages", page_table, table_pages, table_stride, seqs)) return st;
    if (!first || !last || !count_out) return set_error(G4_ERR_INVALID, "release-pages needs first, last and count_out");
    if (count_out == list->count)
        return set_error(G4_ERR_INVALID, "release-pages: count_out cannot be the list's count");
    ReleaseArgs A{list->pages, list->count, page_table, first, last, table_stride ? table_stride : table_pages, count_out,
                  list->capacity, list->num_pages, seqs, table_pages};
    const int64_t most = (int64_t)seqs * table_pages;
    int grid_log = 0;
    while ((1 << grid_log) < kReleaseBlocks && ((int64_t)kReleaseThreads << grid_log) < most) ++grid_log;
    const size_t lds = ((size_t)seqs + 1) * sizeof(int64_t) + (size_t)seqs * sizeof(int32_t);
    hipLaunchKernelGGL(release_pages_kernel, dim3(1 << grid_log), dim3(kReleaseThreads), lds, as_stream(stream), A, grid_log);
    G4_LAUNCHED("release_pages_kernel");
    return G4_OK;
}

}  // extern "C"
