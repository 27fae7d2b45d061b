// qlin_logits.hip -- penalties for repeated tokens, biases and a mask on logits, and the greedy pick of the result
// (qlin_launch_logits_controls, qlin_decoder.h), gfx950.
//
// One pass over the logits: a workgroup takes a slice of a row's vocabulary, its logits in registers; it counts the
// history's tokens of its slice in LDS (integers, so the order of the atomics does not matter), applies penalties and
// mask, and leaves its best (value, token) for a second small launch.  Biased tokens are few: a bit each in LDS takes
// them out of the pass, and the thread that holds a token's first list entry computes that token alone, the sum of its
// entries in list order.  Bound by bytes: each workgroup reads the history again (from L2).  48 rows of 151936 with
// histories of 4000, biases and masks 16.2 to 20.5 us in a kernel trace, 2.9 to 3.7 TB/s; one row 4.5; the second launch
// 1.9 to 4.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_decoder.h"
#include "qlin_internal.hpp"

namespace qlin {
namespace {

constexpr int kThreads = 256;

typedef float f32x4v __attribute__((ext_vector_type(4)));
// (the logits leave as streaming stores: what lies dirty in the L2s at the kernel's end is written back then, 48 rows of
// 151936 18.3 us, so 16.2)
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// the larger of two (value, index) pairs, the lower index among equals; NaN never
__device__ __forceinline__ void better(float &v, int &i, float w, int j) {
    const bool take = w > v || (w == v && j < i);
    v = take ? w : v;
    i = take ? j : i;
}
// over the wave, in every lane
__device__ __forceinline__ void wave_best(float &v, int &i) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(v, i, __shfl_xor(v, o, 64), __shfl_xor(i, o, 64));
}
// over the workgroup, in thread 0
__device__ __forceinline__ void block_best(float &v, int &i, float *s_v, int *s_i) {
    wave_best(v, i);
    if ((threadIdx.x & 63) == 0) {
        s_v[threadIdx.x >> 6] = v;
        s_i[threadIdx.x >> 6] = i;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < kThreads / 64; ++w) better(v, i, s_v[w], s_i[w]);
}

// entries i .. i + 3 of the n at p, -1 past them
__device__ __forceinline__ int4 ids_at(const int *p, int i, int n) {
    int4 v = make_int4(-1, -1, -1, -1);
    if (i + 4 <= n) {
        __builtin_memcpy(&v, __builtin_assume_aligned(p + i, 4), 16);
    } else {
        if (i < n) v.x = p[i];
        if (i + 1 < n) v.y = p[i + 1];
        if (i + 2 < n) v.z = p[i + 2];
    }
    return v;
}

// U runs of 4 tokens a thread: slices of 1024 U tokens.  Everything that does not wait for another load is requested
// before the first barrier: the logits, the mask, the first 2048 tokens of the history (whose length is then not known
// yet) and the first 256 biases.
template <int U>
__global__ __launch_bounds__(kThreads) void logits_controls_kernel(qlin_logits_controls c, const float *logits,
                                                                   size_t logits_stride, float *out, size_t out_stride,
                                                                   int vocab, int slices, float *__restrict__ best_v,
                                                                   int *__restrict__ best_i, int *__restrict__ picks) {
    constexpr int S = 4 * kThreads * U;
    __shared__ __attribute__((aligned(16))) int s_count[S];
    __shared__ uint32_t s_biased[S / 32];
    __shared__ float s_v[kThreads / 64];
    __shared__ int s_i[kThreads / 64], s_twice;
    const int row = blockIdx.x / slices, slice = blockIdx.x % slices, v0 = slice * S, tid = threadIdx.x;
    const int n = min(S, vocab - v0);
    const float *src = logits + static_cast<size_t>(row) * logits_stride + v0;
    float *dst = out + static_cast<size_t>(row) * out_stride + v0;
    const uint32_t *mask = c.mask ? c.mask + static_cast<size_t>(row) * c.mask_stride + v0 / 32 : nullptr;

    f32x4v x[U];
    uint32_t allow[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = 4 * (u * kThreads + tid);
        x[u] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
        allow[u] = ~0u;
        if (i + 4 <= n) {
            __builtin_memcpy(&x[u], __builtin_assume_aligned(src + i, 4), 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) x[u][e] = src[i + e];
        }
        if (mask && i < n) allow[u] = mask[i / 32] >> (i % 32);
    }
    const int *hist = c.history ? c.history + static_cast<size_t>(row) * c.max_history : nullptr;
    const int most = hist ? c.max_history : 0;
    int4 h0 = ids_at(hist, 4 * tid, most), h1 = ids_at(hist, 4 * (kThreads + tid), most);
    const bool biased = c.bias_ids != nullptr && c.max_bias > 0;
    const int *ids = c.bias_ids + static_cast<size_t>(row) * c.max_bias;
    const float *add = c.bias_values + static_cast<size_t>(row) * c.max_bias;
    const int id0 = biased && tid < c.max_bias ? ids[tid] : -1;
    const float add0 = biased && tid < c.max_bias ? add[tid] : 0.0f;
    const float rep = c.repetition ? c.repetition[row] : 1.0f;
    const float freq = c.frequency ? c.frequency[row] : 0.0f, pres = c.presence ? c.presence[row] : 0.0f;
    const int h = most && c.history_lens ? min(max(c.history_lens[row], 0), most) : most;
    const bool counted = h > 0 && !(rep == 1.0f && freq == 0.0f && pres == 0.0f);  // uniform
    if (counted) {
#pragma unroll
        for (int u = 0; u < U; ++u) reinterpret_cast<int4 *>(s_count)[u * kThreads + tid] = make_int4(0, 0, 0, 0);
    }
    if (biased) {
        for (int i = tid; i < S / 32; i += kThreads) s_biased[i] = 0;
        if (tid == 0) s_twice = 0;
    }
    __syncthreads();
    if (counted) {
        auto count = [&](int t) {  // (as unsigned, what is below the slice is above it too: ids < 0 among them)
            const unsigned at = static_cast<unsigned>(t) - static_cast<unsigned>(v0);
            if (at < static_cast<unsigned>(n)) atomicAdd(&s_count[at], 1);
        };
        auto count4 = [&](int4 t, int i) {
            count(i < h ? t.x : -1);
            count(i + 1 < h ? t.y : -1);
            count(i + 2 < h ? t.z : -1);
            count(i + 3 < h ? t.w : -1);
        };
        count4(h0, 4 * tid);
        count4(h1, 4 * (kThreads + tid));
        for (int i0 = 8 * kThreads; i0 < h; i0 += 8 * kThreads) {
            h0 = ids_at(hist, i0 + 4 * tid, h);
            h1 = ids_at(hist, i0 + 4 * (kThreads + tid), h);
            count(h0.x);
            count(h0.y);
            count(h0.z);
            count(h0.w);
            count(h1.x);
            count(h1.y);
            count(h1.z);
            count(h1.w);
        }
    }
    if (biased) {
        for (int e = tid; e < c.max_bias; e += kThreads) {
            const int t = e == tid ? id0 : ids[e];
            const unsigned at = static_cast<unsigned>(t) - static_cast<unsigned>(v0);
            if (t >= 0 && at < static_cast<unsigned>(n)) {
                const uint32_t bit = 1u << (at % 32);
                if (atomicOr(&s_biased[at / 32], bit) & bit) s_twice = 1;
            }
        }
    }
    __syncthreads();
    auto penalized = [&](float l, int count) {
        if (count > 0) {
            l = l > 0.0f ? l / rep : l * rep;
            l = l - freq * static_cast<float>(count);
            l = l - pres;
        }
        return l;
    };
    float bv = -INFINITY;
    int bi = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = 4 * (u * kThreads + tid);
        if (i >= n) continue;
        uint32_t skip = 0;
        if (biased) skip = s_biased[i / 32] >> (i % 32) & 15u;
        if (counted) {
            const int4 k = reinterpret_cast<const int4 *>(s_count)[u * kThreads + tid];
            x[u][0] = penalized(x[u][0], k.x);
            x[u][1] = penalized(x[u][1], k.y);
            x[u][2] = penalized(x[u][2], k.z);
            x[u][3] = penalized(x[u][3], k.w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(allow[u] >> e & 1u)) x[u][e] = -INFINITY;
        if (i + 4 <= n && skip == 0) {
            __builtin_nontemporal_store(x[u], reinterpret_cast<f32x4u *>(dst + i));
#pragma unroll
            for (int e = 0; e < 4; ++e) better(bv, bi, x[u][e], v0 + i + e);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n && !(skip >> e & 1u)) {
                    dst[i + e] = x[u][e];
                    better(bv, bi, x[u][e], v0 + i + e);
                }
        }
    }
    if (biased) {
        const bool twice = s_twice != 0;  // uniform
        for (int e = tid; e < c.max_bias; e += kThreads) {
            const int t = e == tid ? id0 : ids[e];
            const unsigned at = static_cast<unsigned>(t) - static_cast<unsigned>(v0);
            if (t < 0 || at >= static_cast<unsigned>(n)) continue;
            float sum = e == tid ? add0 : add[e];
            if (twice) {
                bool first = true;
                for (int k = 0; k < e; ++k) first &= ids[k] != t;
                if (!first) continue;
                for (int k = e + 1; k < c.max_bias; ++k)
                    if (ids[k] == t) sum += add[k];
            }
            float l = penalized(src[at], counted ? s_count[at] : 0) + sum;
            if (mask && !(mask[at / 32] >> (at % 32) & 1u)) l = -INFINITY;
            dst[at] = l;
            better(bv, bi, l, t);
        }
    }
    if (!picks) return;
    block_best(bv, bi, s_v, s_i);
    if (tid == 0) {
        if (slices == 1) {
            picks[row] = bi;
        } else {
            best_v[blockIdx.x] = bv;
            best_i[blockIdx.x] = bi;
        }
    }
}

// A wave per row: the best of its slices'.
__global__ __launch_bounds__(64) void logits_pick_kernel(const float *__restrict__ best_v, const int *__restrict__ best_i,
                                                         int slices, int *__restrict__ picks) {
    const size_t at = static_cast<size_t>(blockIdx.x) * slices;
    float v = -INFINITY;
    int i = 0;
#pragma unroll 4
    for (int k = threadIdx.x; k < slices; k += 64) better(v, i, best_v[at + k], best_i[at + k]);
    wave_best(v, i);
    if (threadIdx.x == 0) picks[blockIdx.x] = i;
}

constexpr int kMinSlice = 4 * kThreads;
int slices_of(int vocab, int slice) { return (vocab + slice - 1) / slice; }
// Runs per thread.
int runs_of(int rows, int vocab) {
    for (int u = 8; u > 1; u /= 2)
        if (static_cast<int64_t>(rows) * slices_of(vocab, u * kMinSlice) >= 1024) return u;
    return 1;
}

hipStream_t current_stream() { return static_cast<hipStream_t>(qlin_get_stream()); }
bool al4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace
}  // namespace qlin

extern "C" {

size_t qlin_logits_controls_scratch_bytes(int rows, int vocab) {
    if (rows <= 0 || vocab <= 0 || vocab > 1 << 28) return 0;
    const int s = qlin::slices_of(vocab, qlin::runs_of(rows, vocab) * qlin::kMinSlice);
    return s <= 1 ? 0 : static_cast<size_t>(rows) * s * 8;
}

int qlin_launch_logits_controls(const qlin_logits_controls *controls, const float *logits, size_t logits_stride,
                                float *out, size_t out_stride, int rows, int vocab, int *picks, void *scratch,
                                size_t scratch_bytes) {
    if (!controls) return QLIN_ERR_NULL;
    const qlin_logits_controls &c = *controls;
    if (rows < 0 || vocab < 0 || c.max_history < 0 || c.max_bias < 0) return QLIN_ERR_SHAPE;
    if (vocab > (1 << 28) || c.max_history > 1 << 20 || c.max_bias > 4096) return QLIN_ERR_LIMIT;
    if (rows == 0 || vocab == 0) return QLIN_OK;
    if (logits_stride < static_cast<size_t>(vocab) || out_stride < static_cast<size_t>(vocab)) return QLIN_ERR_SHAPE;
    if (logits == out && logits_stride != out_stride) return QLIN_ERR_SHAPE;
    if (c.mask && c.mask_stride < (static_cast<size_t>(vocab) + 31) / 32) return QLIN_ERR_SHAPE;
    if (!logits || !out || (c.bias_ids && c.max_bias > 0 && !c.bias_values)) return QLIN_ERR_NULL;
    for (const void *p : {static_cast<const void *>(logits), static_cast<const void *>(out), static_cast<const void *>(c.history),
                          static_cast<const void *>(c.history_lens), static_cast<const void *>(c.repetition),
                          static_cast<const void *>(c.frequency), static_cast<const void *>(c.presence),
                          static_cast<const void *>(c.bias_ids), static_cast<const void *>(c.bias_values),
                          static_cast<const void *>(c.mask), static_cast<const void *>(picks), static_cast<const void *>(scratch)})
        if (!qlin::al4(p)) return QLIN_ERR_ALIGN;
    const int u = qlin::runs_of(rows, vocab), slices = qlin::slices_of(vocab, u * qlin::kMinSlice);
    const int64_t grid = static_cast<int64_t>(rows) * slices;
    if (grid > (1 << 23)) return QLIN_ERR_LIMIT;
    const size_t need = picks ? qlin_logits_controls_scratch_bytes(rows, vocab) : 0;
    if (need > 0 && !scratch) return QLIN_ERR_NULL;
    if (scratch_bytes < need) return QLIN_ERR_LIMIT;
    float *bv = static_cast<float *>(scratch);
    int *bi = bv ? reinterpret_cast<int *>(bv + grid) : nullptr;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(qlin::kThreads), 0, qlin::current_stream(), c,
                           logits, logits_stride, out, out_stride, vocab, slices, bv, bi, picks);
        if (hipGetLastError() != hipSuccess) return QLIN_ERR_LAUNCH;
        if (!picks || slices == 1) return QLIN_OK;
        hipLaunchKernelGGL(qlin::logits_pick_kernel, dim3(rows), dim3(64), 0, qlin::current_stream(), bv, bi,
                           slices, picks);
        return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
    };
    switch (u) {
        case 8: return go(qlin::logits_controls_kernel<8>);
        case 4: return go(qlin::logits_controls_kernel<4>);
        case 2: return go(qlin::logits_controls_kernel<2>);
        default: return go(qlin::logits_controls_kernel<1>);
    }
}

}  // extern "C"
