// qlin_norm.hip -- the residual's addition, the RMSNorm and its result in f32 and in Q8_1 blocks in one pass, and Q8_1
// blocks read back as the values they stand for (qlin_launch_add_rms_norm, qlin_launch_dequantize_q8_1), gfx950.
//
// Mathematics (qlin_decoder.h): s = x + delta, y = s (mean s^2 + eps)^(-1/2) w, blocks of 32 values as codes rint(y (1 / d)),
// d = amax (1 / 127).  The sum of squares, the root and the product are in f64: y then is the same f32 value whatever the order of
// the sum, and so are the codes (an f64 operation takes an f32 one's time here).
//
// A row is taken by W waves, 4 consecutive values a lane and U such runs in registers, so that x is read once; 8 lanes hold
// one Q8_1 block.  Rows that do not fit (U = 0) are read a second time, each value by the lane that wrote or read it before, so
// that outputs may take the inputs' place.  Many rows are bound by HBM: 2011 rows of 4096 with their sum and blocks of 128 and
// the blocks read back, 150 MB, take 35.1 us in a graph (4.3 TB/s; 8 waves of 2 runs 35.5, 16 of one 37.3), 42 with f32 results
// through the caches: from 16 MB on they leave as streaming stores.  Few rows are bound by latency: 16 waves take a row of 3584 in
// 4.4 us, 4 waves in 6.4; 48 rows of 2048 with f32 results and blocks take 4.0 by 8 waves each, 5.0 by 4.  Wider rows take 16
// waves however many they are: 2011 rows of 8192 49 us in a graph, by 8 waves of 4 runs 53; of 16384 95, by 8 of 8 runs 102.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_decoder.h"
#include "qlin_f64.hpp"
#include "qlin_internal.hpp"
#include "qlin_q8_1.hpp"

namespace qlin {
namespace {

typedef float f32x4v __attribute__((ext_vector_type(4)));

struct NormArgs {
    const float *x, *delta;
    float *sum, *normed;
    uint8_t *q8;
    const uint16_t *w;
    size_t x_stride, delta_stride, sum_stride, normed_stride;
    int norm_type, one_plus, rows, hidden, padded, mmq, raw;  // padded: the values that the row's blocks hold, or hidden
    float eps;
};

// values i .. i + 3 of the n at p, 0 past them
__device__ __forceinline__ f32x4v values_at(const float *p, int i, int n) {
    f32x4v v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i + 4 <= n) {
        __builtin_memcpy(&v, __builtin_assume_aligned(p + i, 4), 16);
    } else {
        if (i < n) v[0] = p[i];
        if (i + 1 < n) v[1] = p[i + 1];
        if (i + 2 < n) v[2] = p[i + 2];
    }
    return v;
}
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
template <bool STREAM>  // (a choice while it runs would be one plain store to the compiler)
__device__ __forceinline__ void store_values(float *p, int i, int n, const f32x4v &v) {
    if (i + 4 <= n) {
        if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<f32x4u *>(p + i));
        else *reinterpret_cast<f32x4u *>(p + i) = v;
    } else {
        if (i < n) p[i] = v[0];
        if (i + 1 < n) p[i + 1] = v[1];
        if (i + 2 < n) p[i + 2] = v[2];
    }
}
// weights i .. i + 3 as 16-bit patterns, one load where w is 8-byte aligned
__device__ __forceinline__ uint2 weights_at(const uint16_t *w, int i, int n) {
    uint2 v = make_uint2(0u, 0u);
    if (i + 4 <= n && (reinterpret_cast<uintptr_t>(w) & 7u) == 0) {
        v = *reinterpret_cast<const uint2 *>(w + i);
    } else {
        if (i < n) v.x = w[i];
        if (i + 1 < n) v.x |= static_cast<uint32_t>(w[i + 1]) << 16;
        if (i + 2 < n) v.y = w[i + 2];
        if (i + 3 < n) v.y |= static_cast<uint32_t>(w[i + 3]) << 16;
    }
    return v;
}
__device__ __forceinline__ double weight_of(uint2 w, int e, int type, int one_plus) {
    const uint32_t u = (e < 2 ? w.x : w.y) >> (16 * (e & 1)) & 0xffffu;
    const float v = type == 0 ? __builtin_bit_cast(float, u << 16)
                              : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u)));
    return one_plus ? static_cast<double>(v) + 1.0 : static_cast<double>(v);
}

template <int W, int U, bool STREAM>
__global__ __launch_bounds__(W < 4 ? 256 : 64 * W) void add_rms_norm_kernel(NormArgs a) {
    constexpr int R = W < 4 ? 4 / W : 1, N = 64 * W;  // rows a workgroup, lanes a row
    __shared__ double red[W > 1 ? R * W : 1];
    const int group = threadIdx.x / N, t = threadIdx.x % N;
    const int row = blockIdx.x * R + group;
    if (W == 1 && row >= a.rows) return;  // (whole waves; with more waves a row, a workgroup has one)
    const float *x = a.x + row * a.x_stride, *delta = a.delta ? a.delta + row * a.delta_stride : nullptr;
    float *sum = a.sum ? a.sum + row * a.sum_stride : nullptr;
    float *normed = a.normed ? a.normed + row * a.normed_stride : nullptr;
    double ss = 0.0;
    auto take = [&](int i) {  // s of values i .. i + 3
        f32x4v s = values_at(x, i, a.hidden);
        if (delta) s += values_at(delta, i, a.hidden);
        return s;
    };
    auto count = [&](int i, const f32x4v &s) {  // stored and squared
        if (sum) store_values<STREAM>(sum, i, a.hidden, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) ss += static_cast<double>(s[e]) * static_cast<double>(s[e]);
    };
    constexpr int K = U > 0 ? U : 1;
    f32x4v s[K];
    uint2 w[K];
    if constexpr (U > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = values_at(x, 4 * (t + N * u), a.hidden);
        if (delta) {  // uniform; asked for all at once, as x
            f32x4v d[K];
#pragma unroll
            for (int u = 0; u < U; ++u) d[u] = values_at(delta, 4 * (t + N * u), a.hidden);
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] += d[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = weights_at(a.w, 4 * (t + N * u), a.hidden);
#pragma unroll
        for (int u = 0; u < U; ++u) count(4 * (t + N * u), s[u]);
    } else {
        for (int i = 4 * t; i < a.hidden; i += 4 * N) count(i, take(i));
    }
    ss = wave_sum_f64(ss);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int v = 0; v < W; ++v) ss += red[group * W + v];
    }
    const double inv = 1.0 / sqrt(ss / a.hidden + static_cast<double>(a.eps));
    auto put = [&](int i, const f32x4v &v, uint2 wv) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[e] = i + e < a.hidden ? static_cast<float>(static_cast<double>(v[e]) * inv * weight_of(wv, e, a.norm_type, a.one_plus)) : 0.0f;
        if (normed) store_values<STREAM>(normed, i, a.hidden, f32x4v{y[0], y[1], y[2], y[3]});
        if (a.q8) {
            const int b = i / 32, j = t & 7;
            if (a.mmq) {
                uint8_t *at = a.q8 + (static_cast<size_t>(b >> 2) * a.rows + row) * 144;
                quantize_normed_lanes(y, j, reinterpret_cast<uint32_t *>(at) + (b & 3),
                                           reinterpret_cast<uint32_t *>(at + 16 + 32 * (b & 3)), a.raw != 0);
            } else {
                uint32_t *at = reinterpret_cast<uint32_t *>(a.q8 + (static_cast<size_t>(row) * (a.padded / 32) + b) * 36);
                quantize_normed_lanes(y, j, at, at + 1, a.raw != 0);
            }
        }
    };
    if constexpr (U > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (4 * (t + N * u) < a.padded) put(4 * (t + N * u), s[u], w[u]);  // (whole groups of 8 lanes, with blocks)
    } else {
        for (int i = 4 * t; i < a.padded; i += 4 * N)
            put(i, sum ? values_at(sum, i, a.hidden) : take(i), weights_at(a.w, i, a.hidden));
    }
}

// 4 values a lane; a lane past the row's end has none.
template <bool STREAM>
__global__ __launch_bounds__(256) void dequantize_q8_1_kernel(const uint8_t *__restrict__ xq, float *__restrict__ x,
                                                              int in_dim, int m, int quads, int64_t total, int mmq) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < total; q += stride) {
        const int64_t r = q / quads;
        const int i = 4 * static_cast<int>(q - r * quads), b = i / 32, j = i / 4 & 7;
        uint32_t scale, codes;
        if (mmq) {
            const uint8_t *at = xq + (static_cast<size_t>(b >> 2) * m + r) * 144;
            scale = reinterpret_cast<const uint32_t *>(at)[b & 3];
            codes = reinterpret_cast<const uint32_t *>(at + 16 + 32 * (b & 3))[j];
        } else {
            const uint32_t *at = reinterpret_cast<const uint32_t *>(xq + (r * ((quads + 7) / 8) + b) * 36);
            scale = at[0];
            codes = at[1 + j];
        }
        const float d = f16_bits_to_f32(scale & 0xffffu);
        f32x4v v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = d * static_cast<float>(static_cast<int8_t>(codes >> (8 * e)));
        store_values<STREAM>(x + r * in_dim, i, in_dim, v);
    }
}

// results of so many values are not kept in the caches
bool streamed(int64_t values) { return values * 4 >= 16 << 20; }

hipStream_t current_stream() { return static_cast<hipStream_t>(qlin_get_stream()); }
bool al(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <int W, int U>
int launch(const NormArgs &a) {
    constexpr int R = W < 4 ? 4 / W : 1;
    const dim3 block(W < 4 ? 256 : 64 * W);
    const int64_t groups = (static_cast<int64_t>(a.rows) + R - 1) / R;
    if (groups * block.x > UINT32_MAX) return QLIN_ERR_LIMIT;
    const dim3 grid(static_cast<unsigned>(groups));
    if (streamed(static_cast<int64_t>(a.rows) * a.hidden)) hipLaunchKernelGGL((add_rms_norm_kernel<W, U, true>), grid, block, 0, current_stream(), a);
    else hipLaunchKernelGGL((add_rms_norm_kernel<W, U, false>), grid, block, 0, current_stream(), a);
    return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
}

}  // namespace
}  // namespace qlin

extern "C" {

int qlin_launch_add_rms_norm(const float *x, size_t x_stride, const float *delta, size_t delta_stride, float *sum,
                             size_t sum_stride, const uint16_t *weight, int norm_type, float eps, int one_plus,
                             float *normed, size_t normed_stride, uint8_t *q8_1, int mmq, int raw_sum, int rows, int hidden) {
    if (norm_type != 0 && norm_type != 1) return QLIN_ERR_UNSUPPORTED_TYPE;
    if (rows < 0 || hidden < 0) return QLIN_ERR_SHAPE;
    if (hidden > 1 << 24) return QLIN_ERR_LIMIT;
    if (rows == 0 || hidden == 0) return QLIN_OK;
    const size_t h = static_cast<size_t>(hidden);
    if (x_stride < h || (delta && delta_stride < h) || (sum && sum_stride < h) || (normed && normed_stride < h)) return QLIN_ERR_SHAPE;
    if (!x || !weight || (!normed && !q8_1)) return QLIN_ERR_NULL;
    // in place, an output stands where the input does
    if ((sum == x && sum_stride != x_stride) || (delta && sum == delta && sum_stride != delta_stride) ||
        (normed && ((normed == x && normed_stride != x_stride) || (normed == delta && normed_stride != delta_stride) || normed == sum)))
        return QLIN_ERR_SHAPE;
    if (!qlin::al(weight, 2)) return QLIN_ERR_ALIGN;
    for (const void *p : {static_cast<const void *>(x), static_cast<const void *>(delta), static_cast<const void *>(sum),
                          static_cast<const void *>(normed), static_cast<const void *>(q8_1)})
        if (!qlin::al(p, 4)) return QLIN_ERR_ALIGN;
    const int unit = !q8_1 ? 1 : mmq ? 128 : 32;
    qlin::NormArgs a = {x, delta, sum, normed, q8_1, weight, x_stride, delta_stride, sum_stride, normed_stride, norm_type,
                        one_plus, rows, hidden, (hidden + unit - 1) / unit * unit, mmq != 0, raw_sum != 0, eps};
    if (a.padded <= 256) return qlin::launch<1, 1>(a);
    if (a.padded <= 1024) return qlin::launch<4, 1>(a);
    if (a.padded <= 2048 && rows < 512) return qlin::launch<8, 1>(a);
    if (a.padded <= 2048) return qlin::launch<4, 2>(a);
    if (a.padded <= 4096 && rows < 512) return qlin::launch<16, 1>(a);
    if (a.padded <= 4096) return qlin::launch<4, 4>(a);
    if (a.padded <= 8192) return qlin::launch<16, 2>(a);
    if (a.padded <= 16384) return qlin::launch<16, 4>(a);
    return qlin::launch<16, 0>(a);
}

int qlin_launch_dequantize_q8_1(const uint8_t *x_q8_1, float *x, int in_dim, int m, int mmq) {
    if (in_dim < 0 || m < 0) return QLIN_ERR_SHAPE;
    if (in_dim == 0 || m == 0) return QLIN_OK;
    if (!x_q8_1 || !x) return QLIN_ERR_NULL;
    if (!qlin::al(x_q8_1, 4) || !qlin::al(x, 4)) return QLIN_ERR_ALIGN;
    if (in_dim > (1 << 30)) return QLIN_ERR_LIMIT;
    const int quads = (in_dim + 3) / 4;
    const int64_t total = static_cast<int64_t>(m) * quads;
    const int64_t groups = (total + 255) / 256;
    const dim3 grid(static_cast<unsigned>(groups < 8192 ? groups : 8192));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, qlin::current_stream(), x_q8_1, x, in_dim, m, quads, total, mmq != 0);
    };
    if (qlin::streamed(total * 4)) go(qlin::dequantize_q8_1_kernel<true>);
    else go(qlin::dequantize_q8_1_kernel<false>);
    return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
}

}  // extern "C"
