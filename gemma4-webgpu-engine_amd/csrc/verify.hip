// Verification of drafted tokens against the target's logits (include/g4serve.h): the speculative
// sampling rule with given random numbers, or the greedy one.
//
// Three launches: (1) every row's maximum and sum of exp by parts of kPart logits; (2) per sequence the
// decisions, and the sums of the weights that the next token is drawn from, by parts; (3) per sequence
// the part and then the logit where the running sum passes u_next of the total. Greedy runs (1) and (3).
// A token is the one of 262144 whose running sum passes a given point, so sums that are 1e-7 off would
// often name its neighbour: weights and sums are held in 64 bits.
#include "g4_internal.h"
#include "../../include/g4serve.h"
#include <cmath>

namespace g4 {

constexpr int kPart = 8192, kVerThreads = 256, kPerThread = kPart / kVerThreads;
constexpr int kMaxDrafts = 63;

struct PartStat {
    double sum;  // of exp((y - y(max)) / T)
    float max;   // of the logits as given
    int index;   // of the first maximum
};

struct VerifyArgs {
    const float *logits, *draft_logits;
    const int32_t *draft_tokens, *draft_start;
    int seqs, drafts, max_drafts, parts;
    int64_t vocab;
    double cap, inv_t;
    int greedy;
    const float *u, *u_next;
    PartStat *stats;   // [drafts + seqs (+ drafts)][parts]
    double *weights;   // [seqs][parts]
    double *norms;     // [seqs][4]: y(max) and sum of the p row, of the q row
    int *chosen;       // [seqs][2]: drafts taken, whether one was refused
    int32_t *tokens, *accepted;
    float *logprobs;
};

__device__ __forceinline__ double softcap64(double x, double cap) {
    if (cap == 0.0) return x;
    const double a = fabs(x) / cap;
    return copysign(cap * (1.0 - 2.0 / (exp(2.0 * a) + 1.0)), x);
}

// exp((y - top) / T), 1 at the maximum itself (both infinite included).
__device__ __forceinline__ double weight(float x, double top, const VerifyArgs &A) {
    const double y = softcap64(x, A.cap);
    return y == top ? 1.0 : exp((y - top) * A.inv_t);
}

__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }

__device__ __forceinline__ double shfl_xor64(double v, int m) { return __shfl_xor(v, m); }

__device__ __forceinline__ void first_max(float &m, int &at, float om, int oat) {
    if (om > m || (om == m && oat < at)) {
        m = om;
        at = oat;
    }
}

// Grid (parts, rows): part blockIdx.x of row blockIdx.y, the target's rows first.
__global__ __launch_bounds__(kVerThreads) void verify_stats_kernel(VerifyArgs A) {
    __shared__ float ms[4];
    __shared__ int is[4];
    __shared__ double ss[4];
    const int t = threadIdx.x, part = blockIdx.x, row = blockIdx.y, targets = A.drafts + A.seqs;
    const float *x = row < targets ? A.logits + row * A.vocab : A.draft_logits + (int64_t)(row - targets) * A.vocab;
    const int64_t base = (int64_t)part * kPart;
    const int n = (int)(A.vocab - base < kPart ? A.vocab - base : kPart);
    x += base;
    float v[kPerThread];
    float m = -INFINITY;
    int at = INT32_MAX;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = j * kVerThreads + t;
        v[j] = i < n ? clean(x[i]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j)
        if (v[j] > m) {
            m = v[j];
            at = j * kVerThreads + t;
        }
#pragma unroll
    for (int s = 32; s; s >>= 1) first_max(m, at, __shfl_xor(m, s), __shfl_xor(at, s));
    if ((t & 63) == 0) {
        ms[t >> 6] = m;
        is[t >> 6] = at;
    }
    __syncthreads();
    m = ms[0];
    at = is[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) first_max(m, at, ms[w], is[w]);
    double sum = 0.0;
    if (m > -INFINITY) {
        const double top = softcap64(m, A.cap);
#pragma unroll
        for (int j = 0; j < kPerThread; ++j)
            if (j * kVerThreads + t < n && v[j] > -INFINITY) sum += weight(v[j], top, A);
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) sum += shfl_xor64(sum, s);
    if ((t & 63) == 0) ss[t >> 6] = sum;
    __syncthreads();
    if (t == 0)
        A.stats[(int64_t)row * A.parts + part] = {(ss[0] + ss[1]) + (ss[2] + ss[3]), m,
                                                  at == INT32_MAX ? -1 : (int)(base + at)};
}

struct RowStat {
    double top, sum;  // y(max), sum of exp((y - top) / T); sum 0: no weight
    int index;
};

// A row's statistics from its parts, by one wave (the same in every lane).
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &A, int row) {
    const PartStat *p = A.stats + (int64_t)row * A.parts;
    float m = -INFINITY;
    int at = INT32_MAX;
    for (int c = threadIdx.x & 63; c < A.parts; c += 64) first_max(m, at, p[c].max, p[c].index < 0 ? INT32_MAX : p[c].index);
#pragma unroll
    for (int s = 32; s; s >>= 1) first_max(m, at, __shfl_xor(m, s), __shfl_xor(at, s));
    if (!(m > -INFINITY)) return {0.0, 0.0, -1};
    const double top = softcap64(m, A.cap);
    double sum = 0.0;
    for (int c = threadIdx.x & 63; c < A.parts; c += 64)
        if (p[c].max > -INFINITY) sum += p[c].sum * weight(p[c].max, top, A);
#pragma unroll
    for (int s = 32; s; s >>= 1) sum += shfl_xor64(sum, s);
    return {top, sum, at};
}

struct Decision {
    int taken, refused, count, start;
};

__device__ __forceinline__ void draft_span(const VerifyArgs &A, int seq, int *start, int *count) {
    const int a = min(max(A.draft_start[seq], 0), A.drafts);
    const int b = min(max(A.draft_start[seq + 1], a), A.drafts);
    *start = a;
    *count = min(b - a, A.max_drafts);
}

// Every draft of the sequence judged, one wave a draft at a time; the block agrees through LDS.
__device__ __forceinline__ Decision decide(const VerifyArgs &A, int seq, unsigned long long *good_lds) {
    int start, count;
    draft_span(A, seq, &start, &count);
    const int wave = threadIdx.x >> 6;
    if (threadIdx.x < 4) good_lds[threadIdx.x] = 0;
    __syncthreads();
    unsigned long long good = 0;
    for (int i = wave; i < count; i += 4) {
        const int tok = A.draft_tokens[start + i], row = start + seq + i;
        const RowStat P = row_stat(A, row);
        bool ok = false;
        if (tok >= 0 && tok < A.vocab && P.sum > 0.0) {
            if (A.greedy) {
                ok = P.index == tok;
            } else {
                const float xp = clean(A.logits[row * A.vocab + tok]);
                const double p = xp > -INFINITY ? weight(xp, P.top, A) / P.sum : 0.0;
                double q = 1.0;
                if (A.draft_logits) {
                    const RowStat Q = row_stat(A, A.drafts + A.seqs + start + i);
                    const float xq = clean(A.draft_logits[(int64_t)(start + i) * A.vocab + tok]);
                    q = Q.sum > 0.0 && xq > -INFINITY ? weight(xq, Q.top, A) / Q.sum : 0.0;
                }
                ok = (double)A.u[start + i] * q < p;
            }
        }
        if (ok) good |= 1ull << i;
    }
    if ((threadIdx.x & 63) == 0) good_lds[wave] = good;
    __syncthreads();
    good = good_lds[0] | good_lds[1] | good_lds[2] | good_lds[3];
    const int taken = min(__ffsll((long long)~good) - 1, count);
    return {taken, taken < count, count, start};
}

// The distribution that the next token comes from: max(p - q, 0), with q a row, one token, or nothing.
struct Source {
    const float *p, *q;
    double p_top, p_inv, q_top, q_inv;
    int64_t point;  // q is 1 here (-1: nowhere)
};

__device__ __forceinline__ double source_weight(const VerifyArgs &A, const Source &S, int64_t i) {
    const float xp = clean(S.p[i]);
    double w = xp > -INFINITY ? weight(xp, S.p_top, A) * S.p_inv : 0.0;
    if (S.q) {
        const float xq = clean(S.q[i]);
        if (xq > -INFINITY) w -= weight(xq, S.q_top, A) * S.q_inv;
    } else if (i == S.point) {
        w -= 1.0;
    }
    return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ Source source_of(const VerifyArgs &A, int seq, int start, int taken, bool refused,
                                            double p_top, double p_sum, double q_top, double q_sum) {
    Source S;
    S.p = A.logits + (int64_t)(start + seq + taken) * A.vocab;
    S.q = refused && A.draft_logits ? A.draft_logits + (int64_t)(start + taken) * A.vocab : nullptr;
    S.p_top = p_top;
    S.p_inv = p_sum > 0.0 ? 1.0 / p_sum : 0.0;
    S.q_top = q_top;
    S.q_inv = q_sum > 0.0 ? 1.0 / q_sum : 0.0;
    S.point = refused && !A.draft_logits ? A.draft_tokens[start + taken] : -1;
    return S;
}

// Grid (parts, seqs): the decisions, and part blockIdx.x's sum of the weights to draw from. Part 0
// writes the outputs of the drafts taken.
__global__ __launch_bounds__(kVerThreads) void verify_weights_kernel(VerifyArgs A) {
    __shared__ unsigned long long good[4];
    __shared__ double ss[4];
    const int t = threadIdx.x, part = blockIdx.x, seq = blockIdx.y;
    const Decision D = decide(A, seq, good);
    const RowStat P = row_stat(A, D.start + seq + D.taken);
    RowStat Q{0.0, 0.0, -1};
    if (D.refused && A.draft_logits) Q = row_stat(A, A.drafts + A.seqs + D.start + D.taken);
    const Source S = source_of(A, seq, D.start, D.taken, D.refused, P.top, P.sum, Q.top, Q.sum);
    const int64_t base = (int64_t)part * kPart;
    double sum = 0.0;
#pragma unroll 4
    for (int j = 0; j < kPerThread; ++j) {
        const int64_t i = base + j * kVerThreads + t;
        if (i < A.vocab) sum += source_weight(A, S, i);
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) sum += shfl_xor64(sum, s);
    if ((t & 63) == 0) ss[t >> 6] = sum;
    __syncthreads();
    if (t == 0) {
        A.weights[(int64_t)seq * A.parts + part] = (ss[0] + ss[1]) + (ss[2] + ss[3]);
        if (part == 0) {
            double *n = A.norms + 4 * seq;
            n[0] = P.top;
            n[1] = P.sum;
            n[2] = Q.top;
            n[3] = Q.sum;
            A.chosen[2 * seq] = D.taken;
            A.chosen[2 * seq + 1] = D.refused;
        }
    }
}

// The tokens and log probabilities of a sequence but the drawn one, one wave a draft at a time.
__device__ __forceinline__ void put_taken(const VerifyArgs &A, int seq, int start, int taken) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    int32_t *out = A.tokens + (int64_t)seq * (A.max_drafts + 1);
    float *lp = A.logprobs ? A.logprobs + (int64_t)seq * (A.max_drafts + 1) : nullptr;
    for (int i = wave; i < taken; i += waves) {
        const int tok = A.draft_tokens[start + i];
        const RowStat P = row_stat(A, start + seq + i);
        if (lane == 0) {
            out[i] = tok;
            if (lp) {
                const double y = softcap64(A.logits[(int64_t)(start + seq + i) * A.vocab + tok], A.cap);
                lp[i] = (float)((y == P.top ? 0.0 : (y - P.top) * A.inv_t) - log(P.sum));
            }
        }
    }
    for (int i = taken + 1 + threadIdx.x; i <= A.max_drafts; i += blockDim.x) {
        out[i] = -1;
        if (lp) lp[i] = 0.0f;
    }
}

__device__ __forceinline__ void put_drawn(const VerifyArgs &A, int seq, int start, int taken, int token, double top,
                                          double sum) {
    A.tokens[(int64_t)seq * (A.max_drafts + 1) + taken] = token;
    A.accepted[seq] = taken;
    if (!A.logprobs) return;
    double lp = 0.0;
    if (token >= 0) {
        const double y = softcap64(A.logits[(int64_t)(start + seq + taken) * A.vocab + token], A.cap);
        lp = (y == top ? 0.0 : (y - top) * A.inv_t) - log(sum);
    }
    A.logprobs[(int64_t)seq * (A.max_drafts + 1) + taken] = (float)lp;
}

__global__ __launch_bounds__(kVerThreads) void verify_greedy_kernel(VerifyArgs A) {
    __shared__ unsigned long long good[4];
    const int seq = blockIdx.x;
    const Decision D = decide(A, seq, good);
    put_taken(A, seq, D.start, D.taken);
    const RowStat P = row_stat(A, D.start + seq + D.taken);
    if (threadIdx.x == 0) put_drawn(A, seq, D.start, D.taken, P.index, P.top, P.sum);
}

// The first of the block's kPart weights from `base` on whose running sum exceeds `target`; the last
// one with any weight where rounding leaves none (-1: no weight at all). Same in every thread.
__device__ __forceinline__ int64_t pick(const VerifyArgs &A, const Source &S, int64_t base, double target, double *ws,
                                        int *first, int *last) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    double w[kPerThread], sum = 0.0;
    const int64_t at = base + (int64_t)t * kPerThread;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        w[j] = at + j < A.vocab ? source_weight(A, S, at + j) : 0.0;
        sum += w[j];
    }
    double run = sum;  // of the threads up to this one
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double o = __shfl_up(run, s);
        if (lane >= s) run += o;
    }
    if (t == 0) {
        *first = INT32_MAX;
        *last = -1;
    }
    if (lane == 63) ws[wave] = run;
    __syncthreads();
    for (int v = 0; v < wave; ++v) run += ws[v];
    double before = run - sum;
    int hit = INT32_MAX, any = -1;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        before += w[j];
        if (w[j] > 0.0) {
            any = t * kPerThread + j;
            if (hit == INT32_MAX && before > target) hit = any;
        }
    }
    if (hit != INT32_MAX) atomicMin(first, hit);
    if (any >= 0) atomicMax(last, any);
    __syncthreads();
    const int f = *first, l = *last;
    __syncthreads();
    return f != INT32_MAX ? base + f : (l >= 0 ? base + l : -1);
}

// One block per sequence: the part where the running sum of the parts passes the target, then the logit.
__global__ __launch_bounds__(kVerThreads) void verify_pick_kernel(VerifyArgs A) {
    __shared__ double ws[4];
    __shared__ int first, last;
    const int seq = blockIdx.x;
    int start, count;
    draft_span(A, seq, &start, &count);
    const int taken = A.chosen[2 * seq];
    bool refused = A.chosen[2 * seq + 1];
    const double *n = A.norms + 4 * seq, *w = A.weights + (int64_t)seq * A.parts;
    put_taken(A, seq, start, taken);
    double total = 0.0;
    for (int c = 0; c < A.parts; ++c) total += w[c];
    int64_t token = -1;
    const double u = A.u_next[seq];
    if (total > 0.0) {
        const Source S = source_of(A, seq, start, taken, refused, n[0], n[1], n[2], n[3]);
        double before = 0.0, target = u * total;
        int part = -1;
        double part_before = 0.0;
        for (int c = 0; c < A.parts; ++c) {
            if (w[c] > 0.0) {
                part = c;
                part_before = before;
                if (before + w[c] > target) break;
            }
            before += w[c];
        }
        token = pick(A, S, (int64_t)part * kPart, target - part_before, ws, &first, &last);
    } else if (refused && n[1] > 0.0) {
        // p and q are the same everywhere: the draw is from p, whose sum of weights is 1
        const Source S = source_of(A, seq, start, taken, false, n[0], n[1], 0.0, 0.0);
        double before = 0.0;
        for (int c = 0; c < A.parts; ++c) {
            const int64_t base = (int64_t)c * kPart;
            double sum = 0.0;
            for (int j = 0; j < kPerThread; ++j) {
                const int64_t i = base + j * kVerThreads + threadIdx.x;
                if (i < A.vocab) sum += source_weight(A, S, i);
            }
#pragma unroll
            for (int s = 32; s; s >>= 1) sum += shfl_xor64(sum, s);
            if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = sum;
            __syncthreads();
            sum = (ws[0] + ws[1]) + (ws[2] + ws[3]);
            __syncthreads();
            if (sum > 0.0) token = pick(A, S, base, u - before, ws, &first, &last);
            if (before + sum > u) break;
            before += sum;
        }
    }
    if (threadIdx.x == 0) put_drawn(A, seq, start, taken, (int)token, n[0], n[1]);
}

static int64_t verify_rows(int seqs, int drafts) { return 2 * (int64_t)drafts + seqs; }

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_verify_workspace_bytes(int seqs, int drafts, int64_t vocab) {
    if (seqs <= 0 || drafts < 0 || vocab <= 0 || vocab > INT32_MAX) return 0;
    const size_t parts = (size_t)((vocab + kPart - 1) / kPart);
    return (size_t)verify_rows(seqs, drafts) * parts * sizeof(PartStat) + (size_t)seqs * parts * sizeof(double) +
           (size_t)seqs * (4 * sizeof(double) + 2 * sizeof(int));
}

int g4_verify_drafts(const float *logits, const float *draft_logits, const int32_t *draft_tokens,
                     const int32_t *draft_start, int seqs, int drafts, int max_drafts, int64_t vocab,
                     float cap, float temperature, const float *u, const float *u_next,
                     void *workspace, size_t workspace_bytes, int32_t *tokens, int32_t *accepted,
                     float *logprobs, void *stream) {
    if (seqs <= 0 || drafts < 0 || vocab <= 0)
        return set_error(G4_ERR_INVALID, "verify-drafts: %d sequences, %d drafts, vocabulary %lld", seqs, drafts,
                         (long long)vocab);
    if (vocab > INT32_MAX) return set_error(G4_ERR_UNSUPPORTED, "verify-drafts: token ids are 32-bit");
    if (max_drafts < 0 || max_drafts > kMaxDrafts)
        return set_error(G4_ERR_INVALID, "verify-drafts: max_drafts %d (0 to %d)", max_drafts, kMaxDrafts);
    if (!(temperature >= 0.0f) || !(cap >= 0.0f) || std::isinf(temperature) || std::isinf(cap))
        return set_error(G4_ERR_INVALID, "verify-drafts: temperature and cap must be finite and at least 0");
    if (!logits || !draft_start || !tokens || !accepted || (drafts && !draft_tokens))
        return set_error(G4_ERR_INVALID, "verify-drafts needs logits, draft_tokens, draft_start, tokens and accepted");
    const bool greedy = temperature == 0.0f;
    if (!greedy && ((drafts && !u) || !u_next))
        return set_error(G4_ERR_INVALID, "verify-drafts: sampling needs the random numbers u and u_next");
    const size_t need = g4_verify_workspace_bytes(seqs, drafts, vocab);
    if (!workspace || workspace_bytes < need)
        return set_error(G4_ERR_INVALID, "verify-drafts: workspace %zu B < %zu B", workspace_bytes, need);
    if ((uintptr_t)workspace & 15) return set_error(G4_ERR_INVALID, "verify-drafts: the workspace must be 16-byte aligned");
    if (greedy) draft_logits = nullptr;
    const int64_t rows = (int64_t)drafts + seqs + (draft_logits ? drafts : 0);
    if (rows > 65535 || seqs > 65535)
        return set_error(G4_ERR_UNSUPPORTED, "verify-drafts: %lld rows in one call (at most 65535)", (long long)rows);
    VerifyArgs A{};
    A.logits = logits;
    A.draft_logits = draft_logits;
    A.draft_tokens = draft_tokens;
    A.draft_start = draft_start;
    A.seqs = seqs;
    A.drafts = drafts;
    A.max_drafts = max_drafts;
    A.parts = (int)((vocab + kPart - 1) / kPart);
    A.vocab = vocab;
    A.cap = cap;
    A.inv_t = greedy ? 1.0 : 1.0 / (double)temperature;
    A.greedy = greedy;
    A.u = u;
    A.u_next = u_next;
    A.stats = static_cast<PartStat *>(workspace);
    A.weights = reinterpret_cast<double *>(A.stats + verify_rows(seqs, drafts) * A.parts);
    A.norms = A.weights + (int64_t)seqs * A.parts;
    A.chosen = reinterpret_cast<int *>(A.norms + 4 * (int64_t)seqs);
    A.tokens = tokens;
    A.accepted = accepted;
    A.logprobs = logprobs;
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL(verify_stats_kernel, dim3(A.parts, (unsigned)rows), dim3(kVerThreads), 0, s, A);
    G4_LAUNCHED("verify_stats_kernel");
    if (greedy) {
        hipLaunchKernelGGL(verify_greedy_kernel, dim3(seqs), dim3(kVerThreads), 0, s, A);
        G4_LAUNCHED("verify_greedy_kernel");
        return G4_OK;
    }
    hipLaunchKernelGGL(verify_weights_kernel, dim3(A.parts, seqs), dim3(kVerThreads), 0, s, A);
    G4_LAUNCHED("verify_weights_kernel");
    hipLaunchKernelGGL(verify_pick_kernel, dim3(seqs), dim3(kVerThreads), 0, s, A);
    G4_LAUNCHED("verify_pick_kernel");
    return G4_OK;
}

}  // extern "C"
