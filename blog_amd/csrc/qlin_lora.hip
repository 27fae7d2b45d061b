// qlin_lora.hip -- low-rank adapters of many requests beside a shared projection (qlin_launch_lora_add, qlin_decoder.h),
// gfx950.
//
// Mathematics: z = A x, y = base + B (scale z), A and B those of the row's adapter.
//
// 1. lora_down_kernel: a wave a value of z.
// 2. lora_up_kernel: a thread a value of y.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_decoder.h"
#include "qlin_device.hpp"
#include "qlin_internal.hpp"

namespace qlin {
namespace {

constexpr int kMostMats = 4;

struct LoraArgs {
    qlin_lora mats[kMostMats];
    const int *ranks, *ids;
    const float *scales, *x;
    float *z;  // [n_mats][rows][max_rank]
    size_t x_stride;
    int n_mats, n_adapters, max_rank, in_dim, rows;
};

template <int T>
__device__ __forceinline__ float weight_at(const void *p, size_t i) {
    if constexpr (T == 0) return __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t *>(p)[i]) << 16);
    else if constexpr (T == 1) return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
    else return static_cast<const float *>(p)[i];
}
__device__ __forceinline__ int adapter_of(const LoraArgs &a, int row) {
    const int id = a.ids[row];
    return id >= 0 && id < a.n_adapters ? id : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs &a, int id) { return a.ranks ? min(max(a.ranks[id], 0), a.max_rank) : a.max_rank; }

template <int T>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    const int row = blockIdx.x, k = blockIdx.y * 4 + (threadIdx.x >> 6), mat = blockIdx.z, lane = threadIdx.x & 63;
    const int id = adapter_of(a, row);
    if (id < 0 || k >= rank_of(a, id)) return;
    const float *x = a.x + row * a.x_stride;
    const size_t w = (static_cast<size_t>(id) * a.max_rank + k) * a.in_dim;
    float sum = 0.0f;
    for (int i = lane; i < a.in_dim; i += 64) sum = fmaf(weight_at<T>(a.mats[mat].a, w + i), x[i], sum);
    sum = wave_sum(sum);
    if (lane == 0) a.z[(static_cast<size_t>(mat) * a.rows + row) * a.max_rank + k] = sum;
}

template <int T>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    const int row = blockIdx.x, o = blockIdx.y * 256 + threadIdx.x, mat = blockIdx.z;
    const qlin_lora &m = a.mats[mat];
    if (o >= m.out_dim) return;
    const int id = adapter_of(a, row);
    const float was = m.base[row * m.base_stride + o];
    float sum = 0.0f;
    if (id >= 0) {
        const int rank = rank_of(a, id);
        const float scale = a.scales ? a.scales[id] : 1.0f;
        const float *z = a.z + (static_cast<size_t>(mat) * a.rows + row) * a.max_rank;
        const size_t w = (static_cast<size_t>(id) * m.out_dim + o) * a.max_rank;
        for (int k = 0; k < rank; ++k) sum = fmaf(weight_at<T>(m.b, w + k), z[k] * scale, sum);
    } else if (m.y == m.base) {
        return;
    }
    m.y[row * m.y_stride + o] = id >= 0 ? was + sum : was;
}

bool al(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace qlin

extern "C" {

size_t qlin_lora_workspace_bytes(int rows, int n_mats, int n_adapters, int max_rank, int in_dim) {
    if (rows <= 0 || n_mats <= 0 || n_adapters <= 0 || max_rank <= 0 || in_dim <= 0) return 0;
    return static_cast<size_t>(rows) * n_mats * max_rank * 4;
}

int qlin_launch_lora_add(const qlin_lora *mats, int n_mats, int weight_type, int n_adapters, int max_rank, int in_dim,
                         const int *ranks, const float *scales, const float *x, size_t x_stride, const int *adapter_ids,
                         int rows, void *workspace, size_t workspace_bytes) {
    if (weight_type < 0 || weight_type > 2) return QLIN_ERR_UNSUPPORTED_TYPE;
    if (n_mats < 0 || n_adapters < 0 || max_rank < 0 || in_dim < 0 || rows < 0 || max_rank % 8 || in_dim % 8) return QLIN_ERR_SHAPE;
    if (n_mats > qlin::kMostMats || max_rank > 256 || n_adapters > 1024 || rows > 65536) return QLIN_ERR_LIMIT;
    if (n_mats == 0 || rows == 0) return QLIN_OK;
    if (!mats || !adapter_ids) return QLIN_ERR_NULL;
    if (!qlin::al(adapter_ids, 4) || !qlin::al(ranks, 4) || !qlin::al(scales, 4) || !qlin::al(x, 4)) return QLIN_ERR_ALIGN;
    const bool work = n_adapters > 0 && max_rank > 0 && in_dim > 0;
    int widest = 0;
    for (int i = 0; i < n_mats; ++i) {
        const qlin_lora &m = mats[i];
        if (m.out_dim < 0) return QLIN_ERR_SHAPE;
        if (m.out_dim == 0) continue;
        const size_t out = static_cast<size_t>(m.out_dim);
        if (m.base_stride < out || m.y_stride < out || (m.y == m.base && m.y_stride != m.base_stride)) return QLIN_ERR_SHAPE;
        if (!m.base || !m.y || (work && (!m.a || !m.b))) return QLIN_ERR_NULL;
        if (!qlin::al(m.a, 16) || !qlin::al(m.b, 16) || !qlin::al(m.base, 4) || !qlin::al(m.y, 4)) return QLIN_ERR_ALIGN;
        widest = m.out_dim > widest ? m.out_dim : widest;
    }
    if (widest == 0) return QLIN_OK;
    if (work && x_stride < static_cast<size_t>(in_dim)) return QLIN_ERR_SHAPE;
    if (work && (!x || !workspace)) return QLIN_ERR_NULL;
    if (!qlin::al(workspace, 16)) return QLIN_ERR_ALIGN;
    if (work && workspace_bytes < qlin_lora_workspace_bytes(rows, n_mats, n_adapters, max_rank, in_dim)) return QLIN_ERR_LIMIT;
    qlin::LoraArgs a = {};
    for (int i = 0; i < n_mats; ++i) a.mats[i] = mats[i];
    a.ranks = ranks, a.ids = adapter_ids, a.scales = scales, a.x = x, a.z = static_cast<float *>(workspace), a.x_stride = x_stride;
    a.n_mats = n_mats, a.n_adapters = work ? n_adapters : 0, a.max_rank = max_rank, a.in_dim = in_dim, a.rows = rows;
    const hipStream_t s = static_cast<hipStream_t>(qlin_get_stream());
    auto go = [&](auto down, auto up) {
        if (work) hipLaunchKernelGGL(down, dim3(rows, (max_rank + 3) / 4, n_mats), dim3(256), 0, s, a);
        hipLaunchKernelGGL(up, dim3(rows, (widest + 255) / 256, n_mats), dim3(256), 0, s, a);
        return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
    };
    switch (weight_type) {
        case 0: return go(qlin::lora_down_kernel<0>, qlin::lora_up_kernel<0>);
        case 1: return go(qlin::lora_down_kernel<1>, qlin::lora_up_kernel<1>);
        default: return go(qlin::lora_down_kernel<2>, qlin::lora_up_kernel<2>);
    }
}

}  // extern "C"
