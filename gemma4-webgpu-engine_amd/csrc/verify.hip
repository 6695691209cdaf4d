// Verification of drafted tokens against the target's logits (include/g4serve.h): the speculative
// sampling rule with given random numbers, or the greedy one.
//
// Launches: (1) every row's maximum and sum of exp, by parts of kPart logits; (2) a block per sequence
// joins its rows' parts, judges the drafts and writes all outputs but the drawn token (greedy: that too, and
// no more launches); (3) the weights that the token is drawn from, summed by units of kUnit logits; (4) a
// block per sequence finds the unit and then the logit where the running sum passes u_next of the total.
//
// A drawn token is the one of up to 262144 whose running sum passes a given point: sums that are 1e-7 off
// would often name its neighbour. So exponents and sums are held in 64 bits and 2^f is good to 1e-12.
//
// What bounds it: (1) issue, about 55 vector operations a logit with the softcap, 29 of them 64-bit, and 37 and 18
// without (264 rows of 262144, with: 98 us, what 55 take at 16 lanes a cycle and SIMD, for a read of 43; 160 rows
// 60; without, 9 rows 7, latency); (3) reading the drawn rows again (32 sequences, 26 us, two rows each); (2) and
// (4) a chain of loads, 4-8 and 8-13 us. Parts of 8192 give 4 waves 32 logits a thread, loaded at once; units of
// 1024 keep the last step one block's work and its code short (2048: 2.4 us more).
#include "g4_logits.h"
#include "../../include/g4serve.h"
#include <cmath>

namespace g4 {

constexpr int kPart = 8192, kVerThreads = 256, kPerThread = kPart / kVerThreads;
constexpr int kUnit = 1024, kUnitPer = kUnit / kVerThreads;
constexpr int kJudgeWaves = 16;
constexpr int kMaxDrafts = 63;

struct PartStat {
    double sum;  // of exp((y - y(max)) / T)
    float max;   // of the logits as given
    int index;   // of the first maximum
};

// What the draw of a sequence needs.
struct Draw {
    double p_top, p_sum, q_top, p_inv, q_inv;  // y(max), sum of exp((y - top) / T) and 1 over it (no weight: 0)
    int taken, refused;                 // drafts taken; whether the next one was refused
};

struct VerifyArgs {
    const float *logits, *draft_logits;
    const int32_t *draft_tokens, *draft_start;
    int seqs, drafts, max_drafts, parts, units;
    int64_t vocab;
    double cap, inv_t;
    double inv_cap2;
    float half_cap;  // a little less than half the cap
    int greedy, vec;  // vec: rows may be read 16 bytes at a time
    const float *u, *u_next;
    PartStat *stats;  // [drafts + seqs (+ drafts)][parts]
    double *weights;  // [seqs][units]
    Draw *draws;      // [seqs]
    int32_t *tokens, *accepted;
    float *logprobs;
};

// The weight of the bulk of a row, 2^((y - top) slope): 16 64-bit operations a logit.
struct RowScale {
    double top, slope;  // 2^((y - top) slope)
};
__device__ __forceinline__ RowScale row_scale(double top, const VerifyArgs &A) {
    return {top, A.inv_t * 1.4426950408889634074};
}
// exp((y - top) / T), 1 at the maximum itself (both infinite included).
__device__ __forceinline__ double weight(float x, double top, const VerifyArgs &A) {
    const double y = softcap64(x, A);
    return y == top ? 1.0 : exp((y - top) * A.inv_t);
}
template <bool CAP>
__device__ __forceinline__ double bulk_weight(float x, const RowScale &S, const VerifyArgs &A) {
    double y = x;
    if (CAP) {
        y = near_cap(y, A);
        if (is_far(x, A)) y = far_cap(x, A.cap);
    }
    const double z = (y - S.top) * S.slope;
    const double e = z > -1000.0 ? pow2(z) : 0.0;  // under 2^-1000 of the largest: none
    return !CAP && x == INFINITY ? 1.0 : e;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

__device__ __forceinline__ void first_max(float &m, int &at, float om, int oat) {
    if (om > m || (om == m && oat < at)) {
        m = om;
        at = oat;
    }
}

// N values of a thread from a row's range of `n` logits at x (past its end: no weight): 16 bytes at a time
// (element j is 1024 (j / 4) + 4 t + j % 4 of the range) or one (256 j + t).
__device__ __forceinline__ int element(int j, int vec) {
    return vec ? (j / 4) * 4 * kVerThreads + 4 * (int)threadIdx.x + j % 4 : j * kVerThreads + (int)threadIdx.x;
}
template <int N>
__device__ __forceinline__ void load_range(const float *x, int n, int vec, float (&v)[N]) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const int i = element(j, 1);
            float4 y = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (i < n) y = *reinterpret_cast<const float4 *>(x + i);  // n is a multiple of 4 here
            v[j] = y.x;
            v[j + 1] = y.y;
            v[j + 2] = y.z;
            v[j + 3] = y.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = element(j, 0);
            v[j] = i < n ? x[i] : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = clean(v[j]);
}

// Grid (parts, rows): part blockIdx.x of row blockIdx.y, the target's rows first.
template <bool CAP>
__global__ __launch_bounds__(kVerThreads) void verify_stats_kernel(VerifyArgs A) {
    __shared__ float ms[4];
    __shared__ double ss[4];
    __shared__ int first;
    const int t = threadIdx.x, part = blockIdx.x, row = blockIdx.y, targets = A.drafts + A.seqs;
    const float *x = row < targets ? A.logits + row * A.vocab : A.draft_logits + (int64_t)(row - targets) * A.vocab;
    const int64_t base = (int64_t)part * kPart;
    const int n = (int)(A.vocab - base < kPart ? A.vocab - base : kPart);
    float v[kPerThread];
    load_range(x + base, n, A.vec, v);
    float mine = v[0];
#pragma unroll
    for (int j = 1; j < kPerThread; ++j) mine = fmaxf(mine, v[j]);
    float m = mine;
#pragma unroll
    for (int s = 32; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
    if ((t & 63) == 0) ms[t >> 6] = m;
    if (t == 0) first = INT32_MAX;
    __syncthreads();
    m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    double sum = 0.0;
    if (m > -INFINITY) {
        if (mine == m) {  // few threads: the first of the maximum's places
            int at = INT32_MAX;
#pragma unroll
            for (int j = kPerThread - 1; j >= 0; --j) at = v[j] == m ? element(j, A.vec) : at;
            atomicMin(&first, at);
        }
        if (!CAP && m == INFINITY) {
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) sum += v[j] == m ? 1.0 : 0.0;
        } else {
            const RowScale S = row_scale(softcap64(m, A), A);
            uint32_t far = 0;  // elements left out here
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) {
                double z = ((CAP ? near_cap(v[j], A) : (double)v[j]) - S.top) * S.slope;
                if (CAP) {
                    const bool f = is_far(v[j], A);
                    far |= f ? 1u << j : 0u;
                    z = f ? -1000.0 : z;
                }
                sum += pow2(z);
            }
            for (; far; far &= far - 1) sum += weight(x[base + element(__ffs(far) - 1, A.vec)], S.top, A);
        }
    }
    sum = wave_sum64(sum);
    if ((t & 63) == 0) ss[t >> 6] = sum;
    __syncthreads();
    if (t == 0)
        A.stats[(int64_t)row * A.parts + part] = {(ss[0] + ss[1]) + (ss[2] + ss[3]), m,
                                                  first == INT32_MAX ? -1 : (int)(base + first)};
}

struct RowStat {
    double top, sum;
    int index;
};

// A row's statistics from its parts, by one wave (the same in every lane).
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &A, int row) {
    const PartStat *p = A.stats + (int64_t)row * A.parts;
    const int lane = threadIdx.x & 63;
    const PartStat mine = p[min(lane, A.parts - 1)];  // the first 64 parts are read once
    float m = -INFINITY;
    int at = INT32_MAX;
    for (int c = lane; c < A.parts; c += 64) {
        const PartStat s = c == lane ? mine : p[c];
        first_max(m, at, s.max, s.index < 0 ? INT32_MAX : s.index);
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) first_max(m, at, __shfl_xor(m, s), __shfl_xor(at, s));
    if (!(m > -INFINITY)) return {0.0, 0.0, -1};
    const double top = softcap64(m, A);
    double sum = 0.0;
    for (int c = lane; c < A.parts; c += 64) {
        const PartStat s = c == lane ? mine : p[c];
        if (s.max > -INFINITY) sum += s.sum * weight(s.max, top, A);
    }
    return {top, wave_sum64(sum), at};
}

__device__ __forceinline__ void draft_span(const VerifyArgs &A, int seq, int *start, int *count) {
    const int a = min(max(A.draft_start[seq], 0), A.drafts);
    const int b = min(max(A.draft_start[seq + 1], a), A.drafts);
    *start = a;
    *count = min(b - a, A.max_drafts);
}

// log p of a token of target row `row`.
__device__ __forceinline__ float log_p(const VerifyArgs &A, int row, int token, const RowStat &P) {
    const double y = softcap64(A.logits[row * A.vocab + token], A);
    return (float)((y == P.top ? 0.0 : (y - P.top) * A.inv_t) - log(P.sum));
}

// One block per sequence: a wave joins one row's parts at a time, then lane i of the first wave judges
// draft i.
__global__ __launch_bounds__(64 * kJudgeWaves) void verify_judge_kernel(VerifyArgs A) {
    __shared__ RowStat ps[kMaxDrafts + 1], qs[kMaxDrafts + 1];
    const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int start, count;
    draft_span(A, seq, &start, &count);
    const int tasks = count + 1 + (A.draft_logits ? count : 0);
    for (int i = wave; i < tasks; i += kJudgeWaves) {
        const bool target = i <= count;
        const int r = target ? i : i - count - 1;
        const RowStat S = row_stat(A, target ? start + seq + r : A.drafts + A.seqs + start + r);
        if (lane == 0) (target ? ps : qs)[r] = S;
    }
    __syncthreads();
    if (wave) return;
    const int row = start + seq + lane;
    int token = -1;
    bool ok = false;
    RowStat P{0.0, 0.0, -1};
    if (lane < count) {
        token = A.draft_tokens[start + lane];
        P = ps[lane];
        if (token >= 0 && token < A.vocab && P.sum > 0.0) {
            if (A.greedy) {
                ok = P.index == token;
            } else {
                const float xp = clean(A.logits[row * A.vocab + token]);
                const double p = xp > -INFINITY ? weight(xp, P.top, A) / P.sum : 0.0;
                double q = 1.0;
                if (A.draft_logits) {
                    const RowStat Q = qs[lane];
                    const float xq = clean(A.draft_logits[(int64_t)(start + lane) * A.vocab + token]);
                    q = Q.sum > 0.0 && xq > -INFINITY ? weight(xq, Q.top, A) / Q.sum : 0.0;
                }
                ok = (double)A.u[start + lane] * q < p;
            }
        }
    }
    const unsigned long long good = __ballot(ok);
    const int taken = min(__ffsll((long long)~good) - 1, count);  // bit 63 of good is never set: count <= 63
    int32_t *out = A.tokens + (int64_t)seq * (A.max_drafts + 1);
    float *lp = A.logprobs ? A.logprobs + (int64_t)seq * (A.max_drafts + 1) : nullptr;
    if (lane <= A.max_drafts && lane != taken) {
        out[lane] = lane < taken ? token : -1;
        if (lp) lp[lane] = lane < taken ? log_p(A, row, token, P) : 0.0f;
    }
    if (lane) return;
    const bool refused = taken < count;
    const RowStat S = ps[taken];
    A.accepted[seq] = taken;
    if (A.greedy) {
        out[taken] = S.index;
        if (lp) lp[taken] = S.index >= 0 ? log_p(A, start + seq + taken, S.index, S) : 0.0f;
        return;
    }
    const RowStat Q = refused && A.draft_logits ? qs[taken] : RowStat{0.0, 0.0, -1};
    A.draws[seq] = {S.top, S.sum, Q.top, S.sum > 0.0 ? 1.0 / S.sum : 0.0, Q.sum > 0.0 ? 1.0 / Q.sum : 0.0, taken,
                    refused};
}

// The distribution that the next token comes from: max(p - q, 0), with q a row, one token, or nothing.
struct Source {
    const float *p, *q;
    RowScale ps, qs;
    double p_inv, q_inv;
    int64_t point;  // q is 1 here (-1: nowhere)
};

__device__ __forceinline__ Source source_of(const VerifyArgs &A, int seq, int start, const Draw &D, bool less) {
    Source S;
    S.p = A.logits + (int64_t)(start + seq + D.taken) * A.vocab;
    S.q = less && A.draft_logits ? A.draft_logits + (int64_t)(start + D.taken) * A.vocab : nullptr;
    S.ps = row_scale(D.p_top, A);
    S.qs = row_scale(D.q_top, A);
    S.p_inv = D.p_inv;
    S.q_inv = D.q_inv;
    S.point = less && !A.draft_logits ? A.draft_tokens[start + D.taken] : -1;
    return S;
}

template <bool CAP>
__device__ __forceinline__ double source_weight(const VerifyArgs &A, const Source &S, int64_t i, float xp, float xq) {
    double w = xp > -INFINITY ? bulk_weight<CAP>(xp, S.ps, A) * S.p_inv : 0.0;
    if (S.q) {
        if (xq > -INFINITY) w -= bulk_weight<CAP>(xq, S.qs, A) * S.q_inv;
    } else if (i == S.point) {
        w -= 1.0;
    }
    return w > 0.0 ? w : 0.0;
}

// The block's thread's weights of a unit, in the element order of load_range; returns their sum.
template <bool CAP>
__device__ __forceinline__ double unit_weights(const VerifyArgs &A, const Source &S, int64_t base,
                                               double (&w)[kUnitPer]) {
    float xp[kUnitPer], xq[kUnitPer] = {};
    const int n = (int)(A.vocab - base < kUnit ? A.vocab - base : kUnit);
    load_range(S.p + base, n, A.vec, xp);
    if (S.q) load_range(S.q + base, n, A.vec, xq);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kUnitPer; ++j) {
        w[j] = source_weight<CAP>(A, S, base + element(j, A.vec), xp[j], xq[j]);
        sum += w[j];
    }
    return sum;
}

__device__ __forceinline__ double block_sum64(double sum, double *lds) {
    sum = wave_sum64(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Grid (units, seqs): unit blockIdx.x's sum of the weights to draw from.
template <bool CAP>
__global__ __launch_bounds__(kVerThreads) void verify_weights_kernel(VerifyArgs A) {
    __shared__ double ss[4];
    const int seq = blockIdx.y;
    int start, count;
    draft_span(A, seq, &start, &count);
    const Draw D = A.draws[seq];
    const Source S = source_of(A, seq, start, D, D.refused);
    double w[kUnitPer];
    const double sum = block_sum64(unit_weights<CAP>(A, S, (int64_t)blockIdx.x * kUnit, w), ss);
    if (threadIdx.x == 0) A.weights[(int64_t)seq * A.units + blockIdx.x] = sum;
}

// The first weight of the unit at `base` whose running sum exceeds `target`; the last one with any weight
// where rounding leaves none (-1: no weight at all). Same in every thread.
template <bool CAP>
__device__ __forceinline__ int64_t pick(const VerifyArgs &A, const Source &S, int64_t base, double target, double *w_lds,
                                        double *ws, int *first, int *last) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    double w[kUnitPer];
    unit_weights<CAP>(A, S, base, w);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kUnitPer; ++j) w_lds[element(j, A.vec)] = w[j];  // to token order
    if (t == 0) {
        *first = INT32_MAX;
        *last = -1;
    }
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kUnitPer; ++j) {
        w[j] = w_lds[t * kUnitPer + j];
        sum += w[j];
    }
    double run = sum;  // of the threads up to this one
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double o = __shfl_up(run, s);
        if (lane >= s) run += o;
    }
    if (lane == 63) ws[wave] = run;
    __syncthreads();
    for (int v = 0; v < wave; ++v) run += ws[v];
    double before = run - sum;
    int hit = INT32_MAX, any = -1;
#pragma unroll
    for (int j = 0; j < kUnitPer; ++j) {
        before += w[j];
        if (w[j] > 0.0) {
            any = t * kUnitPer + j;
            if (hit == INT32_MAX && before > target) hit = any;
        }
    }
    if (hit != INT32_MAX) atomicMin(first, hit);
    if (any >= 0) atomicMax(last, any);
    __syncthreads();
    const int f = *first, l = *last;
    return f != INT32_MAX ? base + f : (l >= 0 ? base + l : -1);
}

// One block per sequence: the unit where the running sum of the units passes the target, then the logit.
template <bool CAP>
__global__ __launch_bounds__(kVerThreads) void verify_pick_kernel(VerifyArgs A) {
    __shared__ double w_lds[kUnit], ws[4];
    __shared__ int first, last;
    const int seq = blockIdx.x, lane = threadIdx.x & 63;
    int start, count;
    draft_span(A, seq, &start, &count);
    const Draw D = A.draws[seq];
    const double *w = A.weights + (int64_t)seq * A.units;
    const double u = A.u_next[seq];
    // every wave by itself: the total, then the first unit that takes the running sum past u of it; the first 256
    // units' sums (a vocabulary of 262144) are read once, all at once
    double total = 0.0, kept[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) kept[i] = 64 * i + lane < A.units ? w[64 * i + lane] : 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) total += kept[i];
    for (int c0 = 256; c0 < A.units; c0 += 64) total += c0 + lane < A.units ? w[c0 + lane] : 0.0;
    total = wave_sum64(total);
    int64_t token = -1;
    if (total > 0.0) {
        const double target = u * total;
        double before = 0.0, unit_before = 0.0;
        int unit = -1;
        for (int c0 = 0; c0 < A.units; c0 += 64) {
            const double x = c0 == 0 ? kept[0] : c0 == 64 ? kept[1] : c0 == 128 ? kept[2] : c0 == 192 ? kept[3]
                             : c0 + lane < A.units ? w[c0 + lane] : 0.0;
            double run = x;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const double o = __shfl_up(run, s);
                if (lane >= s) run += o;
            }
            const unsigned long long some = __ballot(x > 0.0), past = __ballot(x > 0.0 && before + run > target);
            if (some) {  // the first past the target, or the last with any weight so far
                const int at = past ? __ffsll((long long)past) - 1 : 63 - __clzll((long long)some);
                unit = c0 + at;
                unit_before = before + __shfl(run - x, at);
            }
            if (past) break;
            before += __shfl(run, 63);
        }
        token = pick<CAP>(A, source_of(A, seq, start, D, D.refused), (int64_t)unit * kUnit, target - unit_before, w_lds, ws,
                     &first, &last);
    } else if (D.refused && D.p_sum > 0.0) {
        // p and q are the same everywhere: the draw is from p, whose sum of weights is 1
        const Source S = source_of(A, seq, start, D, false);
        double before = 0.0;
        for (int c = 0; c < A.units; ++c) {
            double x[kUnitPer];
            const double sum = block_sum64(unit_weights<CAP>(A, S, (int64_t)c * kUnit, x), ws);
            if (sum > 0.0) token = pick<CAP>(A, S, (int64_t)c * kUnit, u - before, w_lds, ws, &first, &last);
            if (before + sum > u) break;
            before += sum;
        }
    }
    if (threadIdx.x) return;
    A.tokens[(int64_t)seq * (A.max_drafts + 1) + D.taken] = (int)token;
    if (A.logprobs)
        A.logprobs[(int64_t)seq * (A.max_drafts + 1) + D.taken] =
            token >= 0 ? log_p(A, start + seq + D.taken, (int)token, RowStat{D.p_top, D.p_sum, -1}) : 0.0f;
}

template <bool CAP>
static int launch_verify(const VerifyArgs &A, unsigned rows, hipStream_t s) {
    hipLaunchKernelGGL(verify_stats_kernel<CAP>, dim3(A.parts, rows), dim3(kVerThreads), 0, s, A);
    G4_LAUNCHED("verify_stats_kernel");
    hipLaunchKernelGGL(verify_judge_kernel, dim3(A.seqs), dim3(64 * kJudgeWaves), 0, s, A);
    G4_LAUNCHED("verify_judge_kernel");
    if (A.greedy) return G4_OK;
    hipLaunchKernelGGL(verify_weights_kernel<CAP>, dim3(A.units, A.seqs), dim3(kVerThreads), 0, s, A);
    G4_LAUNCHED("verify_weights_kernel");
    hipLaunchKernelGGL(verify_pick_kernel<CAP>, dim3(A.seqs), dim3(kVerThreads), 0, s, A);
    G4_LAUNCHED("verify_pick_kernel");
    return G4_OK;
}

static int64_t verify_rows(int seqs, int drafts) { return 2 * (int64_t)drafts + seqs; }

}  // namespace g4

using namespace g4;

extern "C" {

size_t g4_verify_workspace_bytes(int seqs, int drafts, int64_t vocab) {
    if (seqs <= 0 || drafts < 0 || vocab <= 0 || vocab > INT32_MAX) return 0;
    const size_t parts = (size_t)((vocab + kPart - 1) / kPart);
    const size_t units = (size_t)((vocab + kUnit - 1) / kUnit);
    return (size_t)verify_rows(seqs, drafts) * parts * sizeof(PartStat) + (size_t)seqs * (units * sizeof(double) + sizeof(Draw));
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
    A.units = (int)((vocab + kUnit - 1) / kUnit);
    A.vocab = vocab;
    A.cap = cap;
    A.inv_cap2 = cap > 0.0f ? 1.0 / ((double)cap * cap) : 0.0;
    A.half_cap = 0.4999999f * cap;
    A.vec = vocab % 4 == 0 && (((uintptr_t)logits | (uintptr_t)draft_logits) & 15) == 0;
    A.inv_t = greedy ? 1.0 : 1.0 / (double)temperature;
    A.greedy = greedy;
    A.u = u;
    A.u_next = u_next;
    A.stats = static_cast<PartStat *>(workspace);
    A.weights = reinterpret_cast<double *>(A.stats + verify_rows(seqs, drafts) * A.parts);
    A.draws = reinterpret_cast<Draw *>(A.weights + (int64_t)seqs * A.units);
    A.tokens = tokens;
    A.accepted = accepted;
    A.logprobs = logprobs;
    hipStream_t s = as_stream(stream);
    return cap > 0.0f ? launch_verify<true>(A, (unsigned)rows, s) : launch_verify<false>(A, (unsigned)rows, s);
}

}  // extern "C"
