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
// 2. verify_decide_kernel: a workgroup a sequence joins the slices of each row, accepts or rejects, and without draft logits
//    draws from the target's own weights: the slice by the slices' sums, then the token inside the slice.
// 3. With draft logits: verify_rest_kernel sums max(p - q, 0) over each slice of the one row where a draft was rejected,
//    verify_draw_kernel draws, also from p alone (in 2., a draw that a few sequences wait for cost all of them 4 us).
//
// 24 sequences of 4 drafts with their logits, 216 rows of 151936, take 51 us in a graph: 30.8 of the first launch, bound by
// its vector work (25 instructions a logit, which issue in 85% of its busy cycles; 131 MB at 4.3 TB/s beside), and 5.1, 8.7 and 6.2
// of chains of dependent loads, sums and barriers.  One sequence of 4
// drafts by lookup takes 9.8 us, 40 draws of 102400 without drafts 13.4: latency but for 3.2 us.
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
constexpr int kDecideThreads = 1024;  // a wave a row of a sequence's
constexpr int kDrawThreads = 512;
constexpr int kMostVocab = 1 << 21;    // a slice a thread of the draws
constexpr int kMostDrafts = 63;

typedef float f32x4v __attribute__((ext_vector_type(4)));

// One row's statistics over a slice, or over the row.
struct Stat {
    double sum;  // of exp((l - top) / T)
    float top;
    int at;      // of top, the first one; only at T = 0
};
// What is left to do for a sequence after verify_decide_kernel.
struct Rest {
    double inv_p, inv_q;  // one over the sums
    double heat;          // 32 / (T ln 2)
    double log_p;         // of p's sum
    float top_p, top_q;
    int row;              // -1: nothing is left
    int whole;            // drawn from p alone
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
constexpr double kSteps = 0x1.71547652b82fep+5;  // 32 / ln 2
__device__ __forceinline__ double heat_of(float t) { return t > 0.0f ? kSteps / static_cast<double>(t) : 0.0; }
__device__ __forceinline__ float temperature_of(const VerifyArgs &a, int seq) { return a.temperature ? a.temperature[seq] : 1.0f; }
__device__ __forceinline__ const float *target_row(const VerifyArgs &a, int seq, int i) {
    return a.target + (static_cast<size_t>(seq) * (a.max_drafts + 1) + i) * a.target_stride;
}
__device__ __forceinline__ const float *draft_row(const VerifyArgs &a, int seq, int i) {
    return a.draft + (static_cast<size_t>(seq) * a.max_drafts + i) * a.draft_stride;
}
__device__ __forceinline__ float uniform_at(float u) { return fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f); }
__device__ __forceinline__ float number(float l) { return fmaxf(l, -INFINITY); }  // -inf for NaN

// exp((l - top) / T), heat = 32 / (T ln 2): 2^(n / 32) from a table of 32 values in LDS, 2^(r / 32) for the rest |r| <= 1/2 by
// its Taylor polynomial of degree 5 (the first term left out is below 2e-15 of it).  16 operations; the polynomial of degree
// 13 alone (exp_f64) took 28 with what is around it, and the pass over 216 rows of 151936 took 44.7 us, so 29.1 (4.5 TB/s).
// l is not NaN.  0 for l = -inf, 1 at top, also where both are infinite; a row whose top is -inf is not asked.
__device__ __forceinline__ double step_of(int j) { return exp_f64(j * 0x1.62e42fefa39efp-6); }  // 2^(j / 32)
__device__ __forceinline__ double weight(float l, double top, double heat, const double *steps) {
    const double d = fmin(static_cast<double>(l) - top, 0.0);    // (0 for inf - inf)
    const double t = fmax(d * heat, -35200.0);                   // (and this for -inf * 0)
    const double m = t + 0x1.8p52;
    const int n = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, m)));
    const double r = t - (m - 0x1.8p52);
    constexpr double c = 0x1.62e42fefa39efp-6;  // ln 2 / 32
    double p = __builtin_fma(c * c * c * c * c / 120.0, r, c * c * c * c / 24.0);
    p = __builtin_fma(p, r, c * c * c / 6.0);
    p = __builtin_fma(p, r, c * c / 2.0);
    p = __builtin_fma(p, r, c);
    const double s = steps[n & 31];
    return __builtin_ldexp(__builtin_fma(s * r, p, s), n >> 5);
}

// log exp((l - top) / T)
__device__ __forceinline__ double log_of(float l, float top, float t) {
    return l == top ? 0.0 : (static_cast<double>(l) - static_cast<double>(top)) / static_cast<double>(t);
}

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

// logits i .. i + 3 of the n at p, NaN and what is past them as -inf
__device__ __forceinline__ f32x4v logits_at(const float *p, int i, int n) {
    f32x4v v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (i + 4 <= n) {
        __builtin_memcpy(&v, __builtin_assume_aligned(p + i, 4), 16);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) v[e] = p[i + e];
    }
    return v;
}

// U runs of 4 tokens a thread.
template <int U>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
    __shared__ float s_v[kWaves];
    __shared__ int s_i[kWaves];
    __shared__ double s_sum[kWaves], s_steps[32];
    const int rows = a.max_drafts + 1 + (a.draft ? a.max_drafts : 0);
    const int slice = blockIdx.x % a.slices, r = blockIdx.x / a.slices % rows, seq = blockIdx.x / a.slices / rows;
    const int n_drafts = drafts_of(a, seq);
    if (r <= a.max_drafts ? r > n_drafts : r - a.max_drafts - 1 >= n_drafts) return;  // uniform: a row that is not there
    const int v0 = slice * a.slice, n = min(a.slice, a.vocab - v0), tid = threadIdx.x;
    const float *src = (r <= a.max_drafts ? target_row(a, seq, r) : draft_row(a, seq, r - a.max_drafts - 1)) + v0;
    f32x4v x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = logits_at(src, 4 * (u * kThreads + tid), n);
    const float t = temperature_of(a, seq);
    if (tid < 32) s_steps[tid] = step_of(tid);
    float top = -INFINITY;
    int at = 0;
    if (t > 0.0f) {  // uniform
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[u][e] = number(x[u][e]);
                top = fmaxf(top, x[u][e]);
            }
        top = wave_max_dpp(top);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) better(top, at, x[u][e], v0 + 4 * (u * kThreads + tid) + e);
        wave_best(top, at);
    }
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
    if (t > 0.0f) {
        const double heat = heat_of(t), top64 = top;
        double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[e] += weight(x[u][e], top64, heat, s_steps);
        sum = wave_sum_f64((part[0] + part[1]) + (part[2] + part[3]));
        if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
        __syncthreads();
        sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    }
    if (tid == 0) a.stats[(static_cast<size_t>(seq) * (2 * a.max_drafts + 1) + r) * a.slices + slice] = Stat{sum, top, at};
}

template <int N>
struct Shared {
    double steps[32], part[2][N / 64], base[2];
    int found[2];
};
__device__ __forceinline__ double of_lane(double v, int lane) {  // (uniform)
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return halves(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane)),
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), lane)));
}

// A draw by N threads: from the slices of a row, then from the tokens of a slice.  Thread t has the weights w (>= 0) of the
// items t U .. t U + U - 1 (of a slice each one item, in w[0]).  The first item at which the running sum is above goal(total); where
// rounding leaves none, the last one with a weight; -1 where there is no weight at all.  base: the running sum before it.
// Every wave finds the wave that has the item, from the waves' sums, and that wave finds the item: two barriers (a search by
// all threads between four took 1 us more).  turn: draws that follow one another take the halves of sh in turn.
// (A wave's, a thread's and a walk's sums add the same numbers from other starts, so that a goal can lie beyond the last one by a
// rounding: then the last item with a weight.)
struct Pick {
    int at;
    double base, total;
};
template <int N, int U, class Goal>
__device__ __forceinline__ Pick draw(const double (&w)[U], int each, Goal goal_of, Shared<N> &sh, int turn) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    double mine = 0.0;
#pragma unroll
    for (int e = 0; e < U; ++e) mine += w[e];
    const double run = wave_scan_f64(mine);
    if (lane == 63) sh.part[turn][wave] = run;
    __syncthreads();
    const double part = lane < N / 64 ? sh.part[turn][lane] : 0.0;
    const double upto = wave_scan_f64(part);
    const double total = of_lane(upto, 63), goal = goal_of(total);
    const uint64_t some = __ballot(part > 0.0), past = __ballot(part > 0.0 && upto > goal);
    if (!some) return Pick{-1, 0.0, total};  // (the same in every wave)
    if (wave == (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some))) {
        const double before = wave > 0 ? of_lane(upto, wave - 1) : 0.0;
        const uint64_t some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && before + run > goal);
        if (lane == (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some))) {
            double at = before + (run - mine);
            bool done = false;
#pragma unroll
            for (int e = 0; e < U; ++e) {
                if (w[e] > 0.0 && !done) {
                    sh.found[turn] = tid * each + e;
                    sh.base[turn] = at;
                    done = at + w[e] > goal;
                }
                at += w[e];
            }
        }
    }
    __syncthreads();
    return Pick{sh.found[turn], sh.base[turn], total};
}

// The whole draw of a row from given sums of its slices: slice_weight(k, all) and token_weights(first, i, n, all, w).  all: not
// without what is taken out, where nothing else has a weight.
template <int N, int U, class Slice, class Tokens>
__device__ __forceinline__ int draw_row(const VerifyArgs &a, double u, Slice slice_weight, Tokens token_weights, Shared<N> &sh, bool all = false) {
    int slice = -1;
    double goal = 0.0;
#pragma unroll 1
    for (int turn = 0;; turn ^= 1) {  // (in one piece of code: instructions that are met once cost more time than the arithmetic)
        double w[U];
        if (slice < 0) {
#pragma unroll
            for (int e = 0; e < U; ++e) w[e] = 0.0;
            if (static_cast<int>(threadIdx.x) < a.slices) w[0] = slice_weight(threadIdx.x, all);
        } else {
            token_weights(slice * a.slice, static_cast<int>(threadIdx.x) * U, min(a.slice, a.vocab - slice * a.slice), all, w);
        }
        const Pick k = draw<N, U>(w, slice < 0 ? 1 : U, [&](double total) { return slice < 0 ? u * total : goal; }, sh, turn);
        if (slice >= 0) return slice * a.slice + max(k.at, 0);
        if (k.at < 0) {  // uniform
            if (all) return 0;
            all = true;
            continue;
        }
        slice = k.at;
        goal = u * k.total - k.base;
    }
}
template <int U>
__device__ __forceinline__ void logits_of(const float *p, int i, int n, float (&v)[U]) {
    if constexpr (U % 4 == 0) {
#pragma unroll
        for (int e = 0; e < U; e += 4) {
            const f32x4v x = logits_at(p, i + e, n);
            v[e] = x[0], v[e + 1] = x[1], v[e + 2] = x[2], v[e + 3] = x[3];
        }
    } else {
#pragma unroll
        for (int e = 0; e < U; ++e) v[e] = i + e < n ? p[i + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < U; ++e) v[e] = number(v[e]);
}

// A workgroup a sequence.  What does not wait for the statistics is requested first.
template <int U, bool DRAFT>
__global__ __launch_bounds__(kDecideThreads) void verify_decide_kernel(VerifyArgs a) {
    __shared__ Stat s_row[2 * kMostDrafts + 1];
    __shared__ Shared<kDecideThreads> sh;
    __shared__ double s_log[kMostDrafts + 1];  // of the sums
    __shared__ int s_accepted, s_rejected;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = drafts_of(a, seq), D = a.max_drafts;
    const float t = temperature_of(a, seq);
    const bool greedy = !(t > 0.0f);
    const double heat = heat_of(t);
    int x = -1;
    float u_x = 0.0f, l_p = -INFINITY, l_q = -INFINITY;
    double log_px = 0.0;
    if (wave < 2 && lane < D) {  // a draft a lane, also those that n_drafts leaves out: it is still on its way
        x = a.drafts[static_cast<size_t>(seq) * D + lane];
        u_x = uniform_at(a.uniform[static_cast<size_t>(seq) * (D + 1) + lane]);
        if (x >= 0 && x < a.vocab) {
            l_p = number(target_row(a, seq, lane)[x]);
            if (DRAFT) l_q = number(draft_row(a, seq, lane)[x]);
        }
    }
    const double u = static_cast<double>(uniform_at(a.uniform[static_cast<size_t>(seq) * (D + 1) + D]));
    const Stat *stats = a.stats + static_cast<size_t>(seq) * (2 * D + 1) * a.slices;
    const int rows = DRAFT ? 2 * D + 1 : D + 1;
    constexpr int kAhead = U == 1 ? 3 : 1;  // slices of a row a lane; more are read one after the other
    Stat next[kAhead];
    auto load = [&](int r) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            next[i] = stats[static_cast<size_t>(min(r, rows - 1)) * a.slices + min(lane + 64 * i, a.slices - 1)];
            if (lane + 64 * i >= a.slices) next[i] = Stat{0.0, -INFINITY, 0};
        }
    };
    load(wave);
    if (tid < 32) sh.steps[tid] = step_of(tid);
    __syncthreads();
    // the target's rows, then the drafts' (of rows that are not there: anything, which is not used)
#pragma unroll 1
    for (int r = wave; r < rows;) {
        const Stat *of = stats + static_cast<size_t>(r) * a.slices;
        float top = next[0].top;
        int at = next[0].at;
        double sum = 0.0;
        if (greedy) {
#pragma unroll
            for (int i = 1; i < kAhead; ++i) better(top, at, next[i].top, next[i].at);
#pragma unroll 1
            for (int k = lane + 64 * kAhead; k < a.slices; k += 64) better(top, at, of[k].top, of[k].at);
            wave_best(top, at);
        } else {
#pragma unroll
            for (int i = 1; i < kAhead; ++i) top = fmaxf(top, next[i].top);
#pragma unroll 1
            for (int k = lane + 64 * kAhead; k < a.slices; k += 64) top = fmaxf(top, of[k].top);
            top = wave_max_dpp(top);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) sum += next[i].sum * weight(next[i].top, top, heat, sh.steps);
#pragma unroll 1
            for (int k = lane + 64 * kAhead; k < a.slices; k += 64) sum += of[k].sum * weight(of[k].top, top, heat, sh.steps);
            sum = wave_sum_f64(sum);
        }
        if (lane == 0) s_row[r] = Stat{sum, top, at};
        r += kDecideThreads / 64;
        load(r);
    }
    __syncthreads();
    if (wave == 0) {
        const float inf = INFINITY;
        bool ok = false;
        double px = 0.0;
        if (lane < n) {
            const bool token = x >= 0 && x < a.vocab;
            const Stat p = s_row[lane];
            double qx = token ? 1.0 : 0.0;
            if (token && p.top > -inf) px = greedy ? (x == p.at ? 1.0 : 0.0) : weight(l_p, p.top, heat, sh.steps) / p.sum;
            if (DRAFT && token) {
                const Stat q = s_row[D + 1 + lane];
                qx = !(q.top > -inf) ? 0.0 : greedy ? (x == q.at ? 1.0 : 0.0) : weight(l_q, q.top, heat, sh.steps) / q.sum;
            }
            ok = static_cast<double>(u_x) * qx < px;
            if (a.rates) a.rates[static_cast<size_t>(seq) * D + lane] = static_cast<float>(qx > px ? px / qx : px > 0.0 ? 1.0 : 0.0);
        } else if (lane < D && a.rates) {
            a.rates[static_cast<size_t>(seq) * D + lane] = 0.0f;
        }
        const int m = static_cast<int>(__ffsll(static_cast<long long>(~__ballot(ok)))) - 1;  // (lane 63 has no draft)
        if (lane <= D && lane != m) a.tokens[static_cast<size_t>(seq) * (D + 1) + lane] = lane < m ? x : -1;
        const int rejected = __shfl(x, m, 64);  // (not used where all were accepted)
        if (lane == 0) {
            a.accepted[seq] = m;
            s_accepted = m;
            s_rejected = rejected;
        }
    } else if (wave == 1 && a.logprobs && !greedy) {  // (beside the above, which it would hold up)
        if (lane <= n) {
            const Stat p = s_row[lane];
            const double log_sum = log(p.sum);
            s_log[lane] = log_sum;
            if (lane < n) log_px = log_of(l_p, p.top, t) - log_sum;  // (of an accepted draft, which p has)
        }
    }
    __syncthreads();
    const int m = s_accepted;
    if (wave == 1 && a.logprobs && lane <= D && lane != m)
        a.logprobs[static_cast<size_t>(seq) * (D + 1) + lane] = lane < m ? static_cast<float>(log_px) : 0.0f;
    const Stat p = s_row[m];
    const bool some = p.top > -INFINITY;
    if (DRAFT) {
        const bool due = some && !greedy, rest = m < n && s_row[D + 1 + m].top > -INFINITY;
        if (tid == 0) {
            const Stat q = s_row[rest ? D + 1 + m : m];
            a.rests[seq] = Rest{1.0 / p.sum, 1.0 / q.sum, heat, s_log[m], p.top, q.top, due ? m : -1, !rest};
        }
        if (due) return;  // uniform
    }
    const float *row = target_row(a, seq, m);
    int token = p.at;  // (0 where the row has nothing)
    if constexpr (!DRAFT) {
        if (some && !greedy) {
            // the target's own weights, without the rejected token of a draft by lookup
            const Stat *of = stats + static_cast<size_t>(m) * a.slices;
            const int out = m < n && s_rejected < a.vocab ? s_rejected : -1;
            const double taken = out >= 0 ? weight(number(row[out]), p.top, heat, sh.steps) : 0.0;
            token = draw_row<kDecideThreads, U>(a, u, [&](int k, bool all) {
                const double w = of[k].sum * weight(of[k].top, p.top, heat, sh.steps);
                return !all && out >= 0 && out / a.slice == k ? fmax(w - taken, 0.0) : w;
            }, [&](int v0, int i, int size, bool all, double (&w)[U]) {
                float l[U];
                logits_of(row + v0, i, size, l);
#pragma unroll
                for (int e = 0; e < U; ++e) w[e] = !all && v0 + i + e == out ? 0.0 : weight(l[e], p.top, heat, sh.steps);
            }, sh);
        }
    }
    if (tid == 0) {
        a.tokens[static_cast<size_t>(seq) * (D + 1) + m] = token;
        if (a.logprobs) {
            const float log_p = static_cast<float>(log_of(number(row[token]), p.top, t) - s_log[m]);
            a.logprobs[static_cast<size_t>(seq) * (D + 1) + m] = !some ? -INFINITY : greedy ? 0.0f : log_p;
        }
    }
}

__device__ __forceinline__ double rest_weight(const Rest &r, float p, float q, const double *steps) {
    return fmax(weight(p, r.top_p, r.heat, steps) * r.inv_p - weight(q, r.top_q, r.heat, steps) * r.inv_q, 0.0);
}

template <int U>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs a) {
    __shared__ double s_sum[kWaves], s_steps[32];
    const int slice = blockIdx.x % a.slices, seq = blockIdx.x / a.slices, tid = threadIdx.x;
    const Rest r = a.rests[seq];
    if (r.row < 0 || r.whole) return;  // uniform
    const int v0 = slice * a.slice, n = min(a.slice, a.vocab - v0);
    const float *p = target_row(a, seq, r.row) + v0, *q = draft_row(a, seq, r.row) + v0;
    f32x4v x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        x[u] = logits_at(p, 4 * (u * kThreads + tid), n);
        y[u] = logits_at(q, 4 * (u * kThreads + tid), n);
    }
    if (tid < 32) s_steps[tid] = step_of(tid);
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += rest_weight(r, number(x[u][e]), number(y[u][e]), s_steps);
    sum = wave_sum_f64(sum);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) a.rest_sums[static_cast<size_t>(seq) * a.slices + slice] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

template <int U>  // tokens a thread
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs a) {
    __shared__ Shared<kDrawThreads> sh;
    const int seq = blockIdx.x, D = a.max_drafts;
    const Rest r = a.rests[seq];
    // (requested before it is known whether there is anything to draw)
    const double sum = static_cast<int>(threadIdx.x) < a.slices ? a.rest_sums[static_cast<size_t>(seq) * a.slices + threadIdx.x] : 0.0;
    if (r.row < 0) return;  // uniform
    if (threadIdx.x < 32) sh.steps[threadIdx.x] = step_of(threadIdx.x);
    const float *p = target_row(a, seq, r.row), *q = draft_row(a, seq, r.row);
    const double u = static_cast<double>(uniform_at(a.uniform[static_cast<size_t>(seq) * (D + 1) + D]));
    const float t = temperature_of(a, seq);
    const Stat *of = a.stats + (static_cast<size_t>(seq) * (2 * D + 1) + r.row) * a.slices;
    __syncthreads();
    // all: from p, as where p is nowhere above q
    const int token = draw_row<kDrawThreads, U>(a, u, [&](int k, bool all) {
        return all ? of[k].sum * weight(of[k].top, r.top_p, r.heat, sh.steps) : sum;
    }, [&](int v0, int i, int size, bool all, double (&w)[U]) {
        float x[U], y[U];
        logits_of(p + v0, i, size, x);
        if (!all) logits_of(q + v0, i, size, y);  // uniform
#pragma unroll
        for (int e = 0; e < U; ++e) w[e] = all ? weight(x[e], r.top_p, r.heat, sh.steps) : rest_weight(r, x[e], y[e], sh.steps);
    }, sh, r.whole != 0);
    if (threadIdx.x == 0) {
        a.tokens[static_cast<size_t>(seq) * (D + 1) + r.row] = token;
        if (a.logprobs) a.logprobs[static_cast<size_t>(seq) * (D + 1) + r.row] = static_cast<float>(log_of(number(p[token]), r.top_p, t) - r.log_p);
    }
}

constexpr int kMinSlice = 4 * kThreads;
int slices_of(int vocab, int slice) { return (vocab + slice - 1) / slice; }
// Runs per thread.
int runs_of(int64_t rows, int vocab) {
    for (int u = 4; u > 1; u /= 2)
        if (slices_of(vocab, u / 2 * kMinSlice) > kDrawThreads || rows * slices_of(vocab, u * kMinSlice) >= 1024) return u;
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
    if (n_seqs <= 0 || max_drafts < 0 || max_drafts > qlin::kMostDrafts || vocab <= 0 || vocab > qlin::kMostVocab) return 0;
    return qlin::layout_of(n_seqs, max_drafts, vocab).bytes;
}

int qlin_launch_verify_drafts(const float *target, size_t target_stride, const float *draft, size_t draft_stride,
                              const int *drafts, const int *n_drafts, const float *temperature, const float *uniform,
                              int *tokens, int *accepted, float *logprobs, float *rates, int n_seqs, int max_drafts,
                              int vocab, void *workspace, size_t workspace_bytes) {
    if (n_seqs < 0 || max_drafts < 0 || vocab < 0) return QLIN_ERR_SHAPE;
    if (vocab > qlin::kMostVocab || max_drafts > qlin::kMostDrafts) return QLIN_ERR_LIMIT;
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
    if (grid > (1 << 23) || static_cast<int64_t>(n_seqs) * qlin::kDecideThreads > UINT32_MAX) return QLIN_ERR_LIMIT;
    if (!workspace) return QLIN_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return QLIN_ERR_ALIGN;
    if (workspace_bytes < l.bytes) return QLIN_ERR_LIMIT;
    char *ws = static_cast<char *>(workspace);
    const qlin::VerifyArgs a = {target, draft, target_stride, draft_stride, drafts, n_drafts, temperature, uniform, tokens, accepted,
                                logprobs, rates, n_seqs, max_drafts, vocab, l.runs * qlin::kMinSlice, l.slices,
                                reinterpret_cast<qlin::Stat *>(ws + l.stats), reinterpret_cast<double *>(ws + l.sums),
                                reinterpret_cast<qlin::Rest *>(ws + l.rests)};
    const hipStream_t s = static_cast<hipStream_t>(qlin_get_stream());
    auto go = [&](auto stats, auto decide, auto decide_drafts, auto rest, auto draw) {
        hipLaunchKernelGGL(stats, dim3(static_cast<unsigned>(grid)), dim3(qlin::kThreads), 0, s, a);
        if (!draft) {
            hipLaunchKernelGGL(decide, dim3(n_seqs), dim3(qlin::kDecideThreads), 0, s, a);
        } else {
            hipLaunchKernelGGL(decide_drafts, dim3(n_seqs), dim3(qlin::kDecideThreads), 0, s, a);
            hipLaunchKernelGGL(rest, dim3(static_cast<unsigned>(n_seqs) * l.slices), dim3(qlin::kThreads), 0, s, a);
            hipLaunchKernelGGL(draw, dim3(n_seqs), dim3(qlin::kDrawThreads), 0, s, a);
        }
        return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
    };
    using namespace qlin;
    switch (l.runs) {
        case 4: return go(verify_stats_kernel<4>, verify_decide_kernel<4, false>, verify_decide_kernel<4, true>, verify_rest_kernel<4>, verify_draw_kernel<8>);
        case 2: return go(verify_stats_kernel<2>, verify_decide_kernel<2, false>, verify_decide_kernel<2, true>, verify_rest_kernel<2>, verify_draw_kernel<4>);
        default: return go(verify_stats_kernel<1>, verify_decide_kernel<1, false>, verify_decide_kernel<1, true>, verify_rest_kernel<1>, verify_draw_kernel<2>);
    }
}

}  // extern "C"
