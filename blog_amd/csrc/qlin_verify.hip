// qlin_verify.hip -- drafted tokens checked against the target's probabilities, and the next token drawn from given random
// numbers (qlin_launch_verify_drafts, qlin_decoder.h), gfx950.
//
// Mathematics: p = softmax(target / T), q = softmax(draft / T); x_i is accepted while u_i q_i(x_i) < p_i(x_i); the next token
// comes from max(p_m - q_m, 0) at the first rejection, else from p_n, by the running sum of the weights against u times
// their total.  All of it in f64: with f32 sums a border between two of 150 thousand tokens would move by some 1e-8 for each
// token before it, and one draw in about a thousand would come out otherwise in another order of the sum.
//
// 1. verify_stats_kernel: a workgroup takes a slice of a row, its logits in registers: the largest one, and the sum of
//    exp((l - largest) / T).  This is the only pass over all logits.
// 2. verify_decide_kernel: a workgroup a sequence joins the slices of each row, accepts or rejects, and draws from the
//    target's own weights where that is what is due: the slice by the slices' sums, then the token inside the slice.
// 3. With draft logits, where a draft was rejected: verify_rest_kernel sums max(p - q, 0) over each slice of the one row,
//    verify_draw_kernel draws.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_decoder.h"
#include "qlin_device.hpp"
#include "qlin_f64.hpp"
#include "qlin_internal.hpp"

namespace qlin {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMostDrafts = 63;

typedef float f32x4v __attribute__((ext_vector_type(4)));

// One row's statistics over a slice, or over the row.
struct Stat {
    double sum;  // of exp((l - top) / T)
    float top;
    int at;      // of top, the first one
};
// What is left to do for a sequence after verify_decide_kernel.
struct Rest {
    double inv_p, inv_q;  // one over the sums
    double heat;          // 1 / T
    float top_p, top_q;
    int row;              // -1: nothing is left
};

struct VerifyArgs {
    const float *target, *draft;
    size_t target_stride, draft_stride;
    const int *drafts, *n_drafts;
    const float *temperature, *uniform;
    int *tokens, *accepted;
    float *logprobs, *rates;
    int n_seqs, max_drafts, vocab, slice, slices;
    Stat *stats;  // [n_seqs][2 max_drafts + 1][slices]: target rows, then draft rows
    double *rest_sums;  // [n_seqs][slices]
    Rest *rests;  // [n_seqs]
};

__device__ __forceinline__ int drafts_of(const VerifyArgs &a, int seq) {
    return a.n_drafts ? min(max(a.n_drafts[seq], 0), a.max_drafts) : a.max_drafts;
}
__device__ __forceinline__ double heat_of(const VerifyArgs &a, int seq) {
    const float t = a.temperature ? a.temperature[seq] : 1.0f;
    return t > 0.0f ? 1.0 / static_cast<double>(t) : 0.0;  // 0: the largest takes all
}
__device__ __forceinline__ bool greedy_of(const VerifyArgs &a, int seq) { return a.temperature && !(a.temperature[seq] > 0.0f); }
__device__ __forceinline__ const float *target_row(const VerifyArgs &a, int seq, int i) {
    return a.target + (static_cast<size_t>(seq) * (a.max_drafts + 1) + i) * a.target_stride;
}
__device__ __forceinline__ const float *draft_row(const VerifyArgs &a, int seq, int i) {
    return a.draft + (static_cast<size_t>(seq) * a.max_drafts + i) * a.draft_stride;
}
// exp((l - top) / T) of a logit l of a row whose largest is top; 0 for what is not above -inf (NaN among it), 1 at top
__device__ __forceinline__ double weight(float l, float top, double heat) {
    return l == top && l > -INFINITY ? 1.0 : l > -INFINITY ? exp_f64((static_cast<double>(l) - static_cast<double>(top)) * heat) : 0.0;
}
__device__ __forceinline__ float uniform_at(const float *p) { return fminf(fmaxf(*p, 0.0f), 0x1.fffffep-1f); }

// the larger of two (value, index) pairs, the lower index among equals; NaN never
__device__ __forceinline__ void better(float &v, int &i, float w, int j) {
    const bool take = w > v || (w == v && j < i);
    v = take ? w : v;
    i = take ? j : i;
}
__device__ __forceinline__ void wave_best(float &v, int &i) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
}

// U runs of 4 tokens a thread.
template <int U>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
    __shared__ float s_v[kWaves];
    __shared__ int s_i[kWaves];
    __shared__ double s_sum[kWaves];
    const int rows = a.max_drafts + 1 + (a.draft ? a.max_drafts : 0);
    const int slice = blockIdx.x % a.slices, r = blockIdx.x / a.slices % rows, seq = blockIdx.x / a.slices / rows;
    const int n_drafts = drafts_of(a, seq);
    if (r <= a.max_drafts ? r > n_drafts : r - a.max_drafts - 1 >= n_drafts) return;  // uniform: a row that is not there
    const int v0 = slice * a.slice, n = min(a.slice, a.vocab - v0), tid = threadIdx.x;
    const float *src = (r <= a.max_drafts ? target_row(a, seq, r) : draft_row(a, seq, r - a.max_drafts - 1)) + v0;
    f32x4v x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = 4 * (u * kThreads + tid);
        x[u] = f32x4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 4 <= n) {
            __builtin_memcpy(&x[u], __builtin_assume_aligned(src + i, 4), 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) x[u][e] = src[i + e];
        }
    }
    const double heat = heat_of(a, seq);
    float top = -INFINITY;
    int at = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) better(top, at, x[u][e], v0 + 4 * (u * kThreads + tid) + e);
    wave_best(top, at);
    if ((tid & 63) == 0) {
        s_v[tid >> 6] = top;
        s_i[tid >> 6] = at;
    }
    __syncthreads();
    top = s_v[0];
    at = s_i[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) better(top, at, s_v[w], s_i[w]);
    double sum = 0.0;
    if (!greedy_of(a, seq)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += weight(x[u][e], top, heat);
        sum = wave_sum_f64(sum);
    }
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += s_sum[w];
        a.stats[(static_cast<size_t>(seq) * (2 * a.max_drafts + 1) + r) * a.slices + slice] = Stat{sum, top, at};
    }
}

// The running sum of one value a thread over the workgroup, in thread order: what stands before this thread's, and the total.
__device__ __forceinline__ double before(double v, double &total, double *s_part) {
    double run = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(run, o, 64);
        if ((threadIdx.x & 63) >= static_cast<unsigned>(o)) run += up;
    }
    __syncthreads();  // (s_part's readers of before are done)
    if ((threadIdx.x & 63) == 63) s_part[threadIdx.x >> 6] = run;
    __syncthreads();
    double base = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < static_cast<int>(threadIdx.x >> 6)) base += s_part[w];
        total += s_part[w];
    }
    return base + (run - v);
}

// The workgroup's draw: the first index i of 0 .. n - 1 at which the running sum of weight(i) (>= 0) is above goal(total); where
// rounding leaves none, the last one with a weight; -1 where there is no weight at all.  base: the running sum before i.
// Each thread takes consecutive indices.  A thread's sum and its walk add the same numbers from another start, so a goal
// can lie beyond the walk's end by a rounding: then its last index with a weight.
struct Pick {
    int at;
    double base;
};
template <class Weight, class Goal>
__device__ __forceinline__ Pick draw(int n, Weight weight_of, Goal goal_of, double *s_part, int *s_found, double *s_base) {
    const int each = (n + kThreads - 1) / kThreads, from = min(n, static_cast<int>(threadIdx.x) * each), to = min(n, from + each);
    double mine = 0.0;
    for (int i = from; i < to; ++i) mine += weight_of(i);
    double total;
    const double start = before(mine, total, s_part), goal = goal_of(total);
    if (threadIdx.x == 0) {
        s_found[0] = 0x7fffffff;  // the first thread whose range passes the goal
        s_found[1] = -1;          // the last thread with a weight
        s_found[2] = -1;
    }
    __syncthreads();
    if (mine > 0.0) {
        if (start + mine > goal) atomicMin(&s_found[0], static_cast<int>(threadIdx.x));
        atomicMax(&s_found[1], static_cast<int>(threadIdx.x));
    }
    __syncthreads();
    const int who = s_found[0] != 0x7fffffff ? s_found[0] : s_found[1];
    if (who == static_cast<int>(threadIdx.x)) {
        double run = start;
        for (int i = from; i < to; ++i) {
            const double w = weight_of(i);
            if (w > 0.0) {
                s_found[2] = i;
                *s_base = run;
                if (run + w > goal) break;
            }
            run += w;
        }
    }
    __syncthreads();
    return Pick{s_found[2], *s_base};
}

struct Shared {
    double part[kWaves], base;
    int found[3];
};

// A workgroup a sequence.
__global__ __launch_bounds__(kThreads) void verify_decide_kernel(VerifyArgs a) {
    __shared__ Stat s_row[2 * kMostDrafts + 1];
    __shared__ Shared sh;
    __shared__ int s_accepted;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = drafts_of(a, seq), D = a.max_drafts;
    const double heat = heat_of(a, seq);
    const bool greedy = greedy_of(a, seq);
    const Stat *stats = a.stats + static_cast<size_t>(seq) * (2 * D + 1) * a.slices;
    const int rows = 2 * n + 1;  // the target's n + 1, then the drafts'
    for (int r = wave; r < (a.draft ? rows : n + 1); r += kWaves) {
        const Stat *of = stats + static_cast<size_t>(r <= n ? r : D + r - n) * a.slices;
        float top = -INFINITY;
        int at = 0;
        for (int k = lane; k < a.slices; k += 64) better(top, at, of[k].top, of[k].at);
        wave_best(top, at);
        double sum = 0.0;
        if (!greedy) {
            for (int k = lane; k < a.slices; k += 64) sum += of[k].sum * weight(of[k].top, top, heat);
            sum = wave_sum_f64(sum);
        }
        if (lane == 0) s_row[r] = Stat{sum, top, at};
    }
    __syncthreads();
    if (wave == 0) {  // a draft a lane
        const float inf = INFINITY;
        bool ok = false;
        double px = 0.0, log_px = 0.0;
        int x = 0;
        if (lane < n) {
            x = a.drafts[static_cast<size_t>(seq) * D + lane];
            const bool token = x >= 0 && x < a.vocab;
            const Stat p = s_row[lane];
            double qx = token ? 1.0 : 0.0;
            if (token && p.top > -inf) {
                const float l = target_row(a, seq, lane)[x];
                if (greedy) {
                    px = x == p.at ? 1.0 : 0.0;
                } else {
                    px = weight(l, p.top, heat) / p.sum;
                    log_px = (l == p.top ? 0.0 : (static_cast<double>(l) - static_cast<double>(p.top)) * heat) - log(p.sum);
                }
            }
            if (token && a.draft) {
                const Stat q = s_row[n + 1 + lane];
                qx = !(q.top > -inf) ? 0.0
                     : greedy        ? (x == q.at ? 1.0 : 0.0)
                                     : weight(draft_row(a, seq, lane)[x], q.top, heat) / q.sum;
            }
            ok = static_cast<double>(uniform_at(a.uniform + static_cast<size_t>(seq) * (D + 1) + lane)) * qx < px;
            if (a.rates) a.rates[static_cast<size_t>(seq) * D + lane] = static_cast<float>(qx > px ? px / qx : px > 0.0 ? 1.0 : 0.0);
        } else if (lane < D && a.rates) {
            a.rates[static_cast<size_t>(seq) * D + lane] = 0.0f;
        }
        const int m = static_cast<int>(__ffsll(static_cast<long long>(~__ballot(ok)))) - 1;  // (lane 63 has no draft)
        if (lane <= D && lane != m) {
            a.tokens[static_cast<size_t>(seq) * (D + 1) + lane] = lane < m ? x : -1;
            if (a.logprobs) a.logprobs[static_cast<size_t>(seq) * (D + 1) + lane] = lane < m ? static_cast<float>(log_px) : 0.0f;
        }
        if (lane == 0) {
            a.accepted[seq] = m;
            s_accepted = m;
        }
    }
    __syncthreads();
    const int m = s_accepted;
    const Stat p = s_row[m];
    const float *row = target_row(a, seq, m);
    const int x = m < n ? a.drafts[static_cast<size_t>(seq) * D + m] : -1;  // rejected
    const double u = static_cast<double>(uniform_at(a.uniform + static_cast<size_t>(seq) * (D + 1) + D));
    Rest rest = {0.0, 0.0, heat, p.top, 0.0f, -1};
    int token = p.at;  // (0 where the row has nothing)
    const bool some = p.top > -INFINITY;
    if (some && !greedy) {
        if (a.draft && m < n && s_row[n + 1 + m].top > -INFINITY) {
            const Stat q = s_row[n + 1 + m];
            rest = Rest{1.0 / p.sum, 1.0 / q.sum, heat, p.top, q.top, m};
        } else {
            // the target's own weights, without the rejected token of a draft by lookup
            const Stat *of = stats + static_cast<size_t>(m) * a.slices;
            const int out = a.draft ? -1 : x;
            auto slice_sum = [&](int k) {
                double w = of[k].sum * weight(of[k].top, p.top, heat);
                if (out >= 0 && out < a.vocab && out / a.slice == k) w = fmax(w - weight(row[out], p.top, heat), 0.0);
                return w;
            };
            double goal = 0.0;
            Pick k = draw(a.slices, slice_sum, [&](double total) { return goal = u * total; }, sh.part, sh.found, &sh.base);
            bool all = out < 0;
            if (k.at < 0) {  // uniform: nothing but the rejected token has a weight
                all = true;
                k = draw(a.slices, [&](int i) { return of[i].sum * weight(of[i].top, p.top, heat); },
                         [&](double total) { return goal = u * total; }, sh.part, sh.found, &sh.base);
            }
            const int v0 = k.at * a.slice, size = min(a.slice, a.vocab - v0);
            const Pick v = draw(size, [&](int i) { return !all && v0 + i == out ? 0.0 : weight(row[v0 + i], p.top, heat); },
                                [&](double) { return goal - k.base; }, sh.part, sh.found, &sh.base);
            token = v0 + max(v.at, 0);
        }
    }
    if (tid == 0) {
        if (a.draft) a.rests[seq] = rest;
        if (rest.row < 0) {
            a.tokens[static_cast<size_t>(seq) * (D + 1) + m] = token;
            if (a.logprobs) {
                const double t = row[token] == p.top ? 0.0 : (static_cast<double>(row[token]) - static_cast<double>(p.top)) * heat;
                a.logprobs[static_cast<size_t>(seq) * (D + 1) + m] = !some ? -INFINITY : greedy ? 0.0f : static_cast<float>(t - log(p.sum));
            }
        }
    }
}

__device__ __forceinline__ double rest_weight(const Rest &r, float p, float q) {
    return fmax(weight(p, r.top_p, r.heat) * r.inv_p - weight(q, r.top_q, r.heat) * r.inv_q, 0.0);
}

template <int U>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs a) {
    __shared__ double s_sum[kWaves];
    const int slice = blockIdx.x % a.slices, seq = blockIdx.x / a.slices, tid = threadIdx.x;
    const Rest r = a.rests[seq];
    if (r.row < 0) return;  // uniform
    const int v0 = slice * a.slice, n = min(a.slice, a.vocab - v0);
    const float *p = target_row(a, seq, r.row) + v0, *q = draft_row(a, seq, r.row) + v0;
    f32x4v x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = 4 * (u * kThreads + tid);
        x[u] = y[u] = f32x4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 4 <= n) {
            __builtin_memcpy(&x[u], __builtin_assume_aligned(p + i, 4), 16);
            __builtin_memcpy(&y[u], __builtin_assume_aligned(q + i, 4), 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) {
                    x[u][e] = p[i + e];
                    y[u][e] = q[i + e];
                }
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += rest_weight(r, x[u][e], y[u][e]);
    sum = wave_sum_f64(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += s_sum[w];
        a.rest_sums[static_cast<size_t>(seq) * a.slices + slice] = sum;
    }
}

__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    const int seq = blockIdx.x, D = a.max_drafts;
    const Rest r = a.rests[seq];
    if (r.row < 0) return;  // uniform
    const float *p = target_row(a, seq, r.row), *q = draft_row(a, seq, r.row);
    const double *sums = a.rest_sums + static_cast<size_t>(seq) * a.slices;
    const double u = static_cast<double>(uniform_at(a.uniform + static_cast<size_t>(seq) * (D + 1) + D));
    const Stat *of = a.stats + (static_cast<size_t>(seq) * (2 * D + 1) + r.row) * a.slices;
    double goal = 0.0;
    bool rest = true;
    Pick k = draw(a.slices, [&](int i) { return sums[i]; }, [&](double total) { return goal = u * total; }, sh.part, sh.found, &sh.base);
    if (k.at < 0) {  // uniform: p is nowhere above q
        rest = false;
        k = draw(a.slices, [&](int i) { return of[i].sum * weight(of[i].top, r.top_p, r.heat); },
                 [&](double total) { return goal = u * total; }, sh.part, sh.found, &sh.base);
    }
    const int v0 = max(k.at, 0) * a.slice, size = min(a.slice, a.vocab - v0);
    const Pick v = draw(size, [&](int i) { return rest ? rest_weight(r, p[v0 + i], q[v0 + i]) : weight(p[v0 + i], r.top_p, r.heat); },
                        [&](double) { return goal - k.base; }, sh.part, sh.found, &sh.base);
    if (threadIdx.x == 0) {
        const int token = v0 + max(v.at, 0);
        a.tokens[static_cast<size_t>(seq) * (D + 1) + r.row] = token;
        const double t = p[token] == r.top_p ? 0.0 : (static_cast<double>(p[token]) - static_cast<double>(r.top_p)) * r.heat;
        if (a.logprobs) a.logprobs[static_cast<size_t>(seq) * (D + 1) + r.row] = static_cast<float>(t + log(r.inv_p));
    }
}

constexpr int kMinSlice = 4 * kThreads;
int slices_of(int vocab, int slice) { return (vocab + slice - 1) / slice; }
// Runs per thread.
int runs_of(int64_t rows, int vocab) {
    for (int u = 4; u > 1; u /= 2)
        if (rows * slices_of(vocab, u * kMinSlice) >= 1024) return u;
    return 1;
}
struct Layout {
    int runs, slices;
    size_t stats, rests, sums, bytes;
};
// (the same for calls with and without draft logits)
Layout layout_of(int n_seqs, int max_drafts, int vocab) {
    Layout l;
    const int64_t rows = static_cast<int64_t>(n_seqs) * (2 * max_drafts + 1);
    l.runs = runs_of(static_cast<int64_t>(n_seqs) * (max_drafts + 1), vocab);
    l.slices = slices_of(vocab, l.runs * kMinSlice);
    l.stats = 0;
    l.rests = l.stats + rows * l.slices * sizeof(Stat);
    l.sums = l.rests + static_cast<size_t>(n_seqs) * ((sizeof(Rest) + 15) / 16 * 16);
    l.bytes = l.sums + static_cast<size_t>(n_seqs) * l.slices * 8;
    return l;
}

bool al4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace
}  // namespace qlin

extern "C" {

size_t qlin_verify_drafts_workspace_bytes(int n_seqs, int max_drafts, int vocab) {
    if (n_seqs <= 0 || max_drafts < 0 || max_drafts > qlin::kMostDrafts || vocab <= 0 || vocab > 1 << 28) return 0;
    return qlin::layout_of(n_seqs, max_drafts, vocab).bytes;
}

int qlin_launch_verify_drafts(const float *target, size_t target_stride, const float *draft, size_t draft_stride,
                              const int *drafts, const int *n_drafts, const float *temperature, const float *uniform,
                              int *tokens, int *accepted, float *logprobs, float *rates, int n_seqs, int max_drafts,
                              int vocab, void *workspace, size_t workspace_bytes) {
    if (n_seqs < 0 || max_drafts < 0 || vocab < 0) return QLIN_ERR_SHAPE;
    if (vocab > (1 << 28) || max_drafts > qlin::kMostDrafts) return QLIN_ERR_LIMIT;
    if (n_seqs == 0) return QLIN_OK;
    if (vocab == 0) return QLIN_ERR_SHAPE;  // (there is no token to draw)
    if (target_stride < static_cast<size_t>(vocab) || (draft && max_drafts > 0 && draft_stride < static_cast<size_t>(vocab))) return QLIN_ERR_SHAPE;
    if (!target || !uniform || !tokens || !accepted || (max_drafts > 0 && !drafts)) return QLIN_ERR_NULL;
    for (const void *p : {static_cast<const void *>(target), static_cast<const void *>(draft), static_cast<const void *>(drafts),
                          static_cast<const void *>(n_drafts), static_cast<const void *>(temperature), static_cast<const void *>(uniform),
                          static_cast<const void *>(tokens), static_cast<const void *>(accepted), static_cast<const void *>(logprobs),
                          static_cast<const void *>(rates)})
        if (!qlin::al4(p)) return QLIN_ERR_ALIGN;
    if (max_drafts == 0) draft = nullptr;
    const qlin::Layout l = qlin::layout_of(n_seqs, max_drafts, vocab);
    const int64_t grid = static_cast<int64_t>(n_seqs) * (max_drafts + 1 + (draft ? max_drafts : 0)) * l.slices;
    if (grid > (1 << 23)) return QLIN_ERR_LIMIT;
    if (!workspace) return QLIN_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return QLIN_ERR_ALIGN;
    if (workspace_bytes < l.bytes) return QLIN_ERR_LIMIT;
    char *ws = static_cast<char *>(workspace);
    const qlin::VerifyArgs a = {target, draft, target_stride, draft_stride, drafts, n_drafts, temperature, uniform, tokens, accepted,
                                logprobs, rates, n_seqs, max_drafts, vocab, l.runs * qlin::kMinSlice, l.slices,
                                reinterpret_cast<qlin::Stat *>(ws + l.stats), reinterpret_cast<double *>(ws + l.sums),
                                reinterpret_cast<qlin::Rest *>(ws + l.rests)};
    const hipStream_t s = static_cast<hipStream_t>(qlin_get_stream());
    auto go = [&](auto stats, auto rest) {
        hipLaunchKernelGGL(stats, dim3(static_cast<unsigned>(grid)), dim3(qlin::kThreads), 0, s, a);
        hipLaunchKernelGGL(qlin::verify_decide_kernel, dim3(n_seqs), dim3(qlin::kThreads), 0, s, a);
        if (draft) {
            hipLaunchKernelGGL(rest, dim3(static_cast<unsigned>(n_seqs) * l.slices), dim3(qlin::kThreads), 0, s, a);
            hipLaunchKernelGGL(qlin::verify_draw_kernel, dim3(n_seqs), dim3(qlin::kThreads), 0, s, a);
        }
        return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
    };
    switch (l.runs) {
        case 4: return go(qlin::verify_stats_kernel<4>, qlin::verify_rest_kernel<4>);
        case 2: return go(qlin::verify_stats_kernel<2>, qlin::verify_rest_kernel<2>);
        default: return go(qlin::verify_stats_kernel<1>, qlin::verify_rest_kernel<1>);
    }
}

}  // extern "C"
