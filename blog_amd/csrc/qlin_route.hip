// qlin_route.hip -- the choice of experts by softmax or sigmoid scores, with a bias for the choice, groups, the k best and
// renormalised weights (qlin_launch_moe_route, qlin.h), gfx950.
//
// A wave a token, J consecutive experts a lane (64 J >= n_experts), so that the lowest lane that holds a maximum has the
// lowest expert.  Scores are computed in f64 and rounded to f32 once: which of two experts goes first then does not hang on
// the last bit of an exponential.  Groups are scored from the choice scores in LDS, by as many lanes each as there are; a pick is a
// wave maximum and a ballot.  Bound by latency: one wave's chain of k maxima.  2011 tokens of 256 experts in 8 groups take 7.6 us in
// a graph (a lane a group 7.9; loops over a lane's experts not unrolled, for fewer instructions to fetch, 8.8), one token of 64
// experts 3.0.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_device.hpp"
#include "qlin_f64.hpp"
#include "qlin_internal.hpp"

namespace qlin {
namespace {

constexpr int kWaves = 4;  // tokens a workgroup

template <int J>
__global__ __launch_bounds__(64 * kWaves) void route_kernel(qlin_moe_routing how, const float *__restrict__ logits,
                                                            size_t stride, int *__restrict__ ids, float *__restrict__ weights,
                                                            int tokens, int ne, int k) {
    __shared__ float s_choice[kWaves][64 * J];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, token = blockIdx.x * kWaves + wave;
    if (token >= tokens) return;  // (no barrier follows)
    const float *row = logits + token * stride;
    float l[J], s[J], c[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = lane * J + j;
        l[j] = e < ne ? row[e] : -INFINITY;
        if (!isfinite(l[j])) l[j] = -INFINITY;
    }
    if (how.sigmoid) {
#pragma unroll
        for (int j = 0; j < J; ++j) s[j] = l[j] == -INFINITY ? 0.0f : static_cast<float>(1.0 / (1.0 + exp_f64(-static_cast<double>(l[j]))));
    } else {
        float m = l[0];
#pragma unroll
        for (int j = 1; j < J; ++j) m = fmaxf(m, l[j]);
        m = wave_max_dpp(m);
        double p[J], sum = 0.0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            p[j] = l[j] == -INFINITY ? 0.0 : exp_f64(static_cast<double>(l[j]) - static_cast<double>(m));
            sum += p[j];
        }
        sum = wave_sum_f64(sum);
#pragma unroll
        for (int j = 0; j < J; ++j) s[j] = l[j] == -INFINITY ? 0.0f : static_cast<float>(p[j] / sum);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = lane * J + j;
        c[j] = how.bias && e < ne ? s[j] + how.bias[e] : s[j];
        if (l[j] == -INFINITY || !(c[j] > -INFINITY)) c[j] = -INFINITY;
    }
    if (how.n_groups > 1) {
        const int size = ne / how.n_groups;
#pragma unroll
        for (int j = 0; j < J; ++j) s_choice[wave][lane * J + j] = c[j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (a wave's LDS accesses run in program order)
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // 64 / n_groups lanes a group, as many as a power of two has
        const int shift = 31 - __builtin_clz(64 / how.n_groups), lanes = 1 << shift, group = lane >> shift;
        float first = -INFINITY, second = -INFINITY;
        auto meet = [&](float f, float s) {  // the two largest of both
            second = fmaxf(fmaxf(second, s), fminf(first, f));
            first = fmaxf(first, f);
        };
        if (group < how.n_groups) {
            for (int i = lane & (lanes - 1); i < size; i += lanes) meet(s_choice[wave][group * size + i], -INFINITY);
        }
        for (int o = 1; o < lanes; o <<= 1) meet(__shfl_xor(first, o, 64), __shfl_xor(second, o, 64));
        if (how.group_pairs && second > -INFINITY) first = first + second;
        // a group's place among the groups: those of a larger score, and of an equal one before it
        int place = 0;
        for (int g = 0; g < how.n_groups; ++g) {
            const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, first), g << shift));
            place += other > first || (other == first && g < group);
        }
        const uint64_t kept = __ballot(group < how.n_groups && place < how.top_groups);
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (!(kept >> (min(lane * J + j, ne - 1) / size << shift) & 1)) c[j] = -INFINITY;
    }
    float best = -INFINITY;
    int at = 0;
    auto look = [&]() {
        best = c[0];
        at = 0;
#pragma unroll
        for (int j = 1; j < J; ++j)
            if (c[j] > best) {
                best = c[j];
                at = j;
            }
    };
    look();
    int mine = -1;       // lane r: pick r
    float mine_s = 0.0f;
    double sum = 0.0;
    for (int r = 0; r < k; ++r) {
        const float m = wave_max_dpp(best);
        if (m == -INFINITY) break;  // uniform
        const int p = static_cast<int>(__ffsll(static_cast<long long>(__ballot(best == m)))) - 1;
        float score = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) score = at == j ? s[j] : score;
        const int e = __builtin_amdgcn_readlane(lane * J + at, p);
        score = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, score), p));
        sum += score;
        if (lane == r) {
            mine = e;
            mine_s = score;
        }
        if (lane == p) {
#pragma unroll
            for (int j = 0; j < J; ++j) c[j] = at == j ? -INFINITY : c[j];
            look();
        }
    }
    if (lane < k) {
        double w = mine_s;
        if (how.renormalise) w = w / (sum + 1e-20);
        ids[static_cast<size_t>(token) * k + lane] = mine;
        weights[static_cast<size_t>(token) * k + lane] = mine < 0 ? 0.0f : static_cast<float>(w * static_cast<double>(how.scaling));
    }
}

bool al4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace
}  // namespace qlin

extern "C" int qlin_launch_moe_route(const qlin_moe_routing *how, const float *router_logits, size_t logits_stride,
                                     int *expert_ids, float *weights, int tokens, int n_experts, int k) {
    if (!how) return QLIN_ERR_NULL;
    const qlin_moe_routing &h = *how;
    if (tokens < 0 || n_experts <= 0 || k < 0 || h.n_groups < 1 || h.top_groups < 1) return QLIN_ERR_SHAPE;
    if (n_experts > 1024 || h.n_groups > 64 || k > 64) return QLIN_ERR_LIMIT;
    if (n_experts % h.n_groups || h.top_groups > h.n_groups || k > n_experts / h.n_groups * h.top_groups) return QLIN_ERR_SHAPE;
    if (tokens == 0 || k == 0) return QLIN_OK;
    if (logits_stride < static_cast<size_t>(n_experts)) return QLIN_ERR_SHAPE;
    if (!router_logits || !expert_ids || !weights) return QLIN_ERR_NULL;
    for (const void *p : {static_cast<const void *>(h.bias), static_cast<const void *>(router_logits),
                          static_cast<const void *>(expert_ids), static_cast<const void *>(weights)})
        if (!qlin::al4(p)) return QLIN_ERR_ALIGN;
    const int64_t groups = (static_cast<int64_t>(tokens) + qlin::kWaves - 1) / qlin::kWaves;
    if (groups * 64 * qlin::kWaves > UINT32_MAX) return QLIN_ERR_LIMIT;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(64 * qlin::kWaves), 0,
                           static_cast<hipStream_t>(qlin_get_stream()), h, router_logits, logits_stride, expert_ids, weights,
                           tokens, n_experts, k);
        return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
    };
    if (n_experts <= 64) return go(qlin::route_kernel<1>);
    if (n_experts <= 128) return go(qlin::route_kernel<2>);
    if (n_experts <= 256) return go(qlin::route_kernel<4>);
    if (n_experts <= 512) return go(qlin::route_kernel<8>);
    return go(qlin::route_kernel<16>);
}
