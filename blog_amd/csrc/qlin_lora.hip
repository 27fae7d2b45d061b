// qlin_lora.hip -- low-rank adapters of many requests beside a shared projection (qlin_launch_lora_add, qlin_decoder.h),
// gfx950.
//
// Mathematics: z = A x, y = base + B (scale z), A and B those of the row's adapter.
//
// Rows of one adapter stand in tiles, of 16 rows (up to 256 rows in all, where each workgroup of the first launch groups the
// ids by itself) or of 64 (a launch of one workgroup before it).  Weights are the A operand of the matrix cores, rows of x and
// z the B operand; a lane loads 8 consecutive values of both, so that nothing goes through LDS on the way in.
// 1. lora_down_kernel: z of a tile, up to 64 ranks and a slice of x: 4 waves take parts of the slice and meet in LDS.  Slices
//    are stored apart and added up by the second launch, in order: no atomics.
// 2. lora_up_kernel: a tile and a run of outputs, scale z in LDS.
// Everything is multiplied on v_mfma_f32_16x16x4_f32: f32's products and sums, whatever the values are.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_decoder.h"
#include "qlin_device.hpp"
#include "qlin_internal.hpp"

namespace qlin {
namespace {

constexpr int kMostMats = 4;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kFewRows = 256;   // grouped by each workgroup; with more, a launch groups them
constexpr int kTile = 64;       // the most rows of a tile
constexpr int kRanks = 64;      // of a workgroup of lora_down_kernel
constexpr int kMostAdapters = 1024;

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Rows that have one adapter (-1: none), in the workspace.
struct Tile {
    int adapter, count, pad[2];
    int rows[kTile];
};

struct LoraArgs {
    qlin_lora mats[kMostMats];
    const int *ranks, *ids;
    const float *scales, *x;
    Tile *tiles;
    int *n_tiles;
    float *z;  // [splits][n_mats][rows][max_rank]
    size_t x_stride;
    int n_mats, n_adapters, max_rank, in_dim, rows, splits;
    int copies;  // whether rows without an adapter are copied (somewhere y is not base)
    int chunk, chunks[kMostMats];  // outputs of a workgroup of lora_up_kernel, and their runs up to and with each projection
};

// the adapter's slot; n_adapters for none; -1 for a row with nothing to do
__device__ __forceinline__ int slot_of(const LoraArgs &a, int row) {
    const int id = a.ids[row];
    return id >= 0 && id < a.n_adapters ? id : a.copies ? a.n_adapters : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs &a, int id) { return a.ranks ? min(max(a.ranks[id], 0), a.max_rank) : a.max_rank; }

// 8 weights of a type (0 bf16, 1 f16, 2 f32) as loaded, and as f32 values
template <int T>
struct Weights {
    u32x4 v[T == 2 ? 2 : 1];
    __device__ __forceinline__ void load(const void *p, size_t i, bool there) {
        const u32x4 zero = {0u, 0u, 0u, 0u};
        const u32x4 *q = reinterpret_cast<const u32x4 *>(static_cast<const char *>(p) + i * (T == 2 ? 4 : 2));
#pragma unroll
        for (int h = 0; h < (T == 2 ? 2 : 1); ++h) v[h] = there ? q[h] : zero;
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (T == 2) {
            return __builtin_bit_cast(float, static_cast<uint32_t>(v[j >> 2][j & 3]));
        } else {
            const uint32_t w = v[0][j >> 1];
            if constexpr (T == 0) return __builtin_bit_cast(float, j & 1 ? w & 0xffff0000u : w << 16);
            else return f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xffffu);
        }
    }
    // only the first n count
    __device__ __forceinline__ void keep(int n) {
#pragma unroll
        for (int h = 0; h < (T == 2 ? 2 : 1); ++h)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                if constexpr (T == 2) {
                    if (4 * h + d >= n) v[h][d] = 0u;
                } else {
                    if (2 * d >= n) v[h][d] = 0u;
                    else if (2 * d + 1 >= n) v[h][d] &= 0xffffu;
                }
            }
    }
};

struct Values {  // 8 values of x
    f32x4 v[2];
    __device__ __forceinline__ void load(const float *p, bool there) {
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        v[0] = v[1] = zero;
        if (there) {
            __builtin_memcpy(&v[0], __builtin_assume_aligned(p, 4), 16);
            __builtin_memcpy(&v[1], __builtin_assume_aligned(p + 4, 4), 16);
        }
    }
};

// The tile of number `tile` among up to 256 rows, a row a thread: tiles are numbered by their first rows, and a tile's rows are in
// order, so that every workgroup finds the same.  Gives the number of tiles.
__device__ __forceinline__ int group_rows(const LoraArgs &a, int tile, Tile &t, int *s_ids, int *s_first, int *s_chunk) {
    const int r = threadIdx.x;
    const int mine = r < a.rows ? slot_of(a, r) : -1;
    s_ids[r] = mine;
    if (r == 0) {
        t.count = 0;
        t.adapter = -1;
        *s_chunk = -1;
    }
    __syncthreads();
    int before = 0;  // rows before this one that have its adapter
    for (int i = 0; i < (r & ~63) + 64; i += 4) {  // (uniform in a wave)
        const int4 v = *reinterpret_cast<const int4 *>(s_ids + i);
        before += (v.x == mine && i < r) + (v.y == mine && i + 1 < r) + (v.z == mine && i + 2 < r) + (v.w == mine && i + 3 < r);
    }
    const bool first = mine >= 0 && before % 16 == 0;
    const uint64_t firsts = __ballot(first);
    if ((r & 63) == 0) s_first[r >> 6] = static_cast<int>(__popcll(firsts));
    __syncthreads();
    int at = static_cast<int>(__popcll(firsts & ((1ull << (r & 63)) - 1))), n = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < (r >> 6)) at += s_first[w];
        n += s_first[w];
    }
    if (first && at == tile) {
        t.adapter = mine;
        *s_chunk = before / 16;
    }
    __syncthreads();
    if (mine >= 0 && mine == t.adapter && before / 16 == *s_chunk) {
        t.rows[before % 16] = r;
        atomicMax(&t.count, before % 16 + 1);
    }
    __syncthreads();
    if (r == 0 && t.adapter == a.n_adapters) t.adapter = -1;
    __syncthreads();
    return n;
}

// More rows: one workgroup counts each adapter's rows, gives it its tiles and puts the rows into them.  (In what order does
// not matter: a row's results do not depend on its tile.)
constexpr int kGroupThreads = 1024;
__global__ __launch_bounds__(kGroupThreads) void lora_group_kernel(LoraArgs a) {
    __shared__ int s_count[kMostAdapters + 1], s_tile[kMostAdapters + 1], s_wave[kGroupThreads / 64], s_total;
    const int tid = threadIdx.x, lane = tid & 63;
    for (int i = tid; i <= kMostAdapters; i += kGroupThreads) s_count[i] = 0;
    if (tid == 0) s_total = 0;
    __syncthreads();
    for (int r = tid; r < a.rows; r += kGroupThreads) {
        const int id = slot_of(a, r);
        if (id >= 0) atomicAdd(&s_count[id], 1);
    }
    __syncthreads();
    for (int base = 0; base <= a.n_adapters; base += kGroupThreads) {
        const int id = base + tid;
        const int n = id <= a.n_adapters ? (s_count[id] + kTile - 1) / kTile : 0;
        int run = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(run, o, 64);
            if (lane >= o) run += up;
        }
        if (lane == 63) s_wave[tid >> 6] = run;
        __syncthreads();
        int start = s_total + run - n;
        for (int w = 0; w < (tid >> 6); ++w) start += s_wave[w];
        if (id <= a.n_adapters) s_tile[id] = start;
        for (int t = 0; t < n; ++t) {
            a.tiles[start + t].adapter = id == a.n_adapters ? -1 : id;
            a.tiles[start + t].count = min(kTile, s_count[id] - t * kTile);
        }
        __syncthreads();
        if (tid == kGroupThreads - 1) s_total = start + n;
        if (id <= a.n_adapters) s_count[id] = 0;
        __syncthreads();
    }
    for (int r = tid; r < a.rows; r += kGroupThreads) {
        const int id = slot_of(a, r);
        if (id < 0) continue;
        const int at = atomicAdd(&s_count[id], 1);
        a.tiles[s_tile[id] + at / kTile].rows[at % kTile] = r;
    }
    if (tid == 0) *a.n_tiles = s_total;
}

// z of one tile, one projection, one group of ranks and one slice of x.  NT: tiles of 16 rows.
template <int T, int NT>
__device__ __forceinline__ void down(const LoraArgs &a, const Tile &t, int mat, int group, int split, f32x4 *s_z) {
    constexpr int RT = kRanks / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int rank = rank_of(a, t.adapter) - group * kRanks;
    if (rank <= 0) return;  // uniform
    const int tiles = min((rank + 15) / 16, RT);
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = zero;
    // (rows past the tile's or the rank's end are others again; what comes of them is not stored)
    const float *x[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) x[j] = a.x + t.rows[min(16 * j + n, t.count - 1)] * a.x_stride;
    size_t w[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
        w[i] = (static_cast<size_t>(t.adapter) * a.max_rank + group * kRanks + min(16 * i + n, rank - 1)) * a.in_dim;
    const void *weights = a.mats[mat].a;
    const int steps = (a.in_dim + 31) / 32, parts = a.splits * kWaves, part = split * kWaves + wave;
    const int from = static_cast<int>(static_cast<int64_t>(steps) * part / parts), to = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / parts);
    struct Step {
        Weights<T> w[RT];
        Values x[NT];
    };
    auto load = [&](Step &s, int at) {
        const int k = 32 * at + 8 * g;
        const bool there = at < to && k < a.in_dim;
#pragma unroll
        for (int j = 0; j < NT; ++j) s.x[j].load(x[j] + k, there);
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (i < tiles) s.w[i].load(weights, w[i] + k, there);
    };
    auto multiply = [&](const Step &s) {
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (i < tiles) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(s.w[i].at(e), s.x[j].v[e >> 2][e & 3], acc[i][j], 0, 0, 0);
            }
    };
    constexpr int U = NT == 1 ? 4 : 2;  // steps in flight
    Step s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(s[u], from + u);
    for (int at = from; at < to; at += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Step now = s[u];
            load(s[u], at + U + u);
            multiply(now);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (i < tiles) s_z[((wave * RT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // a lane's 4 values are ranks 4 g .. 4 g + 3 of row n
#pragma unroll
    for (int i = 0; i < RT * NT; i += kWaves) {
        const int at = i + wave, rt = at / NT, j = at % NT;
        if (rt >= tiles) continue;
        f32x4 sum = s_z[at * 64 + lane];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += s_z[(v * RT * NT + at) * 64 + lane];
        const int row = 16 * j + n, k = group * kRanks + 16 * rt + 4 * g;
        if (row < t.count && k < a.max_rank)
            *reinterpret_cast<f32x4 *>(a.z + ((static_cast<size_t>(split) * a.n_mats + mat) * a.rows + t.rows[row]) * a.max_rank + k) = sum;
    }
}

// FEW: at most 256 rows in tiles of 16, a workgroup for each tile that there can be; else the tiles that there are in turn.
template <int T, bool FEW>
__global__ __launch_bounds__(kThreads) void lora_down_kernel(LoraArgs a) {
    __shared__ Tile t;
    __shared__ __attribute__((aligned(16))) f32x4 s_z[kWaves * (kRanks / 16) * (FEW ? 1 : kTile / 16) * 64];
    const int groups = (a.max_rank + kRanks - 1) / kRanks, units = a.n_mats * groups * a.splits;
    if constexpr (FEW) {
        __shared__ __attribute__((aligned(16))) int s_ids[kFewRows];
        __shared__ int s_first[kWaves], s_chunk;
        const int tile = blockIdx.x / units, unit = blockIdx.x % units;
        const int n = group_rows(a, tile, t, s_ids, s_first, &s_chunk);
        if (unit == 0) {  // for lora_up_kernel
            if (tile < n) {
                if (threadIdx.x < 16) a.tiles[tile].rows[threadIdx.x] = t.rows[threadIdx.x];
                if (threadIdx.x == 0) {
                    a.tiles[tile].adapter = t.adapter;
                    a.tiles[tile].count = t.count;
                }
            }
            if (tile == 0 && threadIdx.x == 0) *a.n_tiles = n;
        }
        if (tile >= n || t.adapter < 0) return;  // uniform
        const int split = unit % a.splits, rest = unit / a.splits;
        down<T, 1>(a, t, rest % a.n_mats, rest / a.n_mats, split, s_z);
    } else {
        const int total = *a.n_tiles * units;
        for (int item = blockIdx.x; item < total; item += gridDim.x) {
            const int tile = item / units, unit = item % units;
            __syncthreads();  // (the tile and the sums of before are read)
            if (threadIdx.x < kTile) t.rows[threadIdx.x] = a.tiles[tile].rows[threadIdx.x];
            if (threadIdx.x == 0) {
                t.adapter = a.tiles[tile].adapter;
                t.count = a.tiles[tile].count;
            }
            __syncthreads();
            if (t.adapter < 0) continue;  // uniform
            const int split = unit % a.splits, rest = unit / a.splits;
            if (t.count <= 16) down<T, 1>(a, t, rest % a.n_mats, rest / a.n_mats, split, s_z);
            else down<T, kTile / 16>(a, t, rest % a.n_mats, rest / a.n_mats, split, s_z);
        }
    }
}

__device__ __forceinline__ f32x4 values_at(const float *p, int i, int n) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i + 4 <= n) {
        __builtin_memcpy(&v, __builtin_assume_aligned(p + i, 4), 16);
    } else {
        if (i < n) v[0] = p[i];
        if (i + 1 < n) v[1] = p[i + 1];
        if (i + 2 < n) v[2] = p[i + 2];
    }
    return v;
}
__device__ __forceinline__ void store_values(float *p, int i, int n, const f32x4 &v) {
    if (i + 4 <= n) {
        __builtin_memcpy(__builtin_assume_aligned(p + i, 4), &v, 16);
    } else {
        if (i < n) p[i] = v[0];
        if (i + 1 < n) p[i + 1] = v[1];
        if (i + 2 < n) p[i + 2] = v[2];
    }
}

// y of one tile and one run of outputs.  s_z: [16 NT][stride] scale z, 0 past the rank.
template <int T, int NT>
__device__ __forceinline__ void up(const LoraArgs &a, const Tile &t, int mat, int first, const float *s_z, int stride, int rank) {
    const qlin_lora &m = a.mats[mat];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int last = min(first + a.chunk, m.out_dim);
    const float *base[NT];
    float *y[NT];
    bool there[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int row = t.rows[min(16 * j + n, t.count - 1)];
        there[j] = 16 * j + n < t.count;
        base[j] = m.base + row * m.base_stride;
        y[j] = m.y + row * m.y_stride;
    }
    const size_t w = static_cast<size_t>(max(t.adapter, 0)) * m.out_dim;
    const int chunks = (rank + 31) / 32;  // 0 without an adapter
    // 32 outputs at a time, so that a row's 128 bytes are met together
    for (int o = first + 32 * wave; o < last; o += 32 * kWaves) {
        f32x4 acc[2][NT];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[h][j] = values_at(base[j], o + 16 * h + 4 * g, there[j] ? last : 0);
        f32x4 sum[2][NT];
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j) sum[h][j] = zero;
        for (int c = 0; c < chunks; ++c) {
            const int k = 32 * c + 8 * g;
            Weights<T> b[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                b[h].load(m.b, (w + min(o + 16 * h + n, m.out_dim - 1)) * a.max_rank + k, k < rank);
                if (32 * c + 32 > rank) b[h].keep(rank - k);  // uniform
            }
            f32x4 z[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const f32x4 *p = reinterpret_cast<const f32x4 *>(s_z + (16 * j + n) * stride + k);
                z[j][0] = p[0];
                z[j][1] = p[1];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        sum[h][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[h].at(e), z[j][e >> 2][e & 3], sum[h][j], 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                store_values(y[j], o + 16 * h + 4 * g, there[j] ? last : 0, chunks ? acc[h][j] + sum[h][j] : acc[h][j]);
    }
}

template <int T, bool FEW>
__global__ __launch_bounds__(kThreads) void lora_up_kernel(LoraArgs a) {
    constexpr int M = FEW ? 16 : kTile;
    extern __shared__ __attribute__((aligned(16))) float s_z[];  // [M][stride]
    __shared__ Tile t;
    const int stride = (a.max_rank + 31) / 32 * 32 + 4;  // (rows 4 banks apart)
    const int runs = a.chunks[a.n_mats - 1], total = *a.n_tiles * runs;
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
        const int tile = item / runs;
        int run = item % runs, mat = 0;
        while (run >= a.chunks[mat]) ++mat;
        if (mat > 0) run -= a.chunks[mat - 1];
        __syncthreads();  // (the tile of before is read)
        if (threadIdx.x < M) t.rows[threadIdx.x] = a.tiles[tile].rows[threadIdx.x];
        if (threadIdx.x == 0) {
            t.adapter = a.tiles[tile].adapter;
            t.count = a.tiles[tile].count;
        }
        __syncthreads();
        if (t.adapter < 0 && a.mats[mat].y == a.mats[mat].base) continue;  // uniform
        const int rank = t.adapter < 0 ? 0 : rank_of(a, t.adapter);
        const int quads = (rank + 31) / 32 * 8;  // of a row
        const float scale = t.adapter >= 0 && a.scales ? a.scales[t.adapter] : 1.0f;
        const int rows = (t.count + 15) / 16 * 16;
        for (int i = threadIdx.x; i < rows * quads; i += kThreads) {
            const int r = i / quads, k = 4 * (i % quads);
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            if (r < t.count && k < rank) {
                const float *p = a.z + (static_cast<size_t>(mat) * a.rows + t.rows[r]) * a.max_rank + k;
                for (int s = 0; s < a.splits; ++s) sum += *reinterpret_cast<const f32x4 *>(p + static_cast<size_t>(s) * a.n_mats * a.rows * a.max_rank);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = k + e < rank ? sum[e] * scale : 0.0f;
            }
            *reinterpret_cast<f32x4 *>(s_z + r * stride + k) = sum;
        }
        __syncthreads();
        if (FEW || t.count <= 16) up<T, 1>(a, t, mat, run * a.chunk, s_z, stride, rank);
        else up<T, M / 16>(a, t, mat, run * a.chunk, s_z, stride, rank);
    }
}

bool al(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Layout {
    int most_tiles, groups, splits;
    size_t tiles, z, bytes;
};
Layout layout_of(int rows, int n_mats, int n_adapters, int max_rank, int in_dim) {
    Layout l;
    const bool few = rows <= kFewRows;
    const int m = few ? 16 : kTile, kinds = rows < n_adapters + 1 ? rows : n_adapters + 1;
    l.most_tiles = rows / m + kinds;
    if (l.most_tiles > rows) l.most_tiles = rows;
    l.groups = (max_rank + kRanks - 1) / kRanks;
    // slices of x: as many as give about 512 workgroups, each wave 2 steps of 32 at least
    const int steps = (in_dim + 31) / 32;
    int64_t tiles = few ? l.most_tiles : (rows + m - 1) / m;
    l.splits = static_cast<int>(512 / (tiles * n_mats * l.groups));
    if (l.splits > steps / (2 * kWaves)) l.splits = steps / (2 * kWaves);
    if (l.splits > 8) l.splits = 8;
    if (l.splits < 1) l.splits = 1;
    l.tiles = 16;
    l.z = l.tiles + sizeof(Tile) * l.most_tiles;
    l.bytes = l.z + sizeof(float) * l.splits * n_mats * static_cast<size_t>(rows) * max_rank;
    return l;
}

}  // namespace
}  // namespace qlin

extern "C" {

size_t qlin_lora_workspace_bytes(int rows, int n_mats, int n_adapters, int max_rank, int in_dim) {
    if (rows <= 0 || n_mats <= 0 || n_adapters <= 0 || max_rank <= 0 || in_dim <= 0 || rows > 65536 || n_mats > qlin::kMostMats ||
        max_rank > 256 || n_adapters > qlin::kMostAdapters)
        return 0;
    return qlin::layout_of(rows, n_mats, n_adapters, max_rank, in_dim).bytes;
}

int qlin_launch_lora_add(const qlin_lora *mats, int n_mats, int weight_type, int n_adapters, int max_rank, int in_dim,
                         const int *ranks, const float *scales, const float *x, size_t x_stride, const int *adapter_ids,
                         int rows, void *workspace, size_t workspace_bytes) {
    if (weight_type < 0 || weight_type > 2) return QLIN_ERR_UNSUPPORTED_TYPE;
    if (n_mats < 0 || n_adapters < 0 || max_rank < 0 || in_dim < 0 || rows < 0 || max_rank % 8 || in_dim % 8) return QLIN_ERR_SHAPE;
    if (n_mats > qlin::kMostMats || max_rank > 256 || n_adapters > qlin::kMostAdapters || rows > 65536) return QLIN_ERR_LIMIT;
    if (n_mats == 0 || rows == 0) return QLIN_OK;
    if (n_adapters == 0 || max_rank == 0 || in_dim == 0) return QLIN_ERR_SHAPE;
    if (!mats || !adapter_ids || !x) return QLIN_ERR_NULL;
    if (!qlin::al(adapter_ids, 4) || !qlin::al(ranks, 4) || !qlin::al(scales, 4) || !qlin::al(x, 4)) return QLIN_ERR_ALIGN;
    if (x_stride < static_cast<size_t>(in_dim)) return QLIN_ERR_SHAPE;
    qlin::LoraArgs a = {};
    for (int i = 0; i < n_mats; ++i) {
        const qlin_lora &m = mats[i];
        if (m.out_dim < 0) return QLIN_ERR_SHAPE;
        if (m.out_dim > 1 << 24) return QLIN_ERR_LIMIT;
        a.mats[i] = m;
        if (m.out_dim == 0) continue;
        const size_t out = static_cast<size_t>(m.out_dim);
        if (m.base_stride < out || m.y_stride < out || (m.y == m.base && m.y_stride != m.base_stride)) return QLIN_ERR_SHAPE;
        if (!m.base || !m.y || !m.a || !m.b) return QLIN_ERR_NULL;
        if (!qlin::al(m.a, 16) || !qlin::al(m.b, 16) || !qlin::al(m.base, 4) || !qlin::al(m.y, 4)) return QLIN_ERR_ALIGN;
        if (m.y != m.base) a.copies = 1;
    }
    // projections without outputs have nothing to do
    int kept = 0;
    for (int i = 0; i < n_mats; ++i)
        if (a.mats[i].out_dim > 0) a.mats[kept++] = a.mats[i];
    if (kept == 0) return QLIN_OK;
    if (!workspace) return QLIN_ERR_NULL;
    if (!qlin::al(workspace, 16)) return QLIN_ERR_ALIGN;
    if (workspace_bytes < qlin_lora_workspace_bytes(rows, n_mats, n_adapters, max_rank, in_dim)) return QLIN_ERR_LIMIT;
    const qlin::Layout l = qlin::layout_of(rows, n_mats, n_adapters, max_rank, in_dim);
    char *ws = static_cast<char *>(workspace);
    a.ranks = ranks, a.ids = adapter_ids, a.scales = scales, a.x = x, a.x_stride = x_stride;
    a.n_tiles = reinterpret_cast<int *>(ws), a.tiles = reinterpret_cast<qlin::Tile *>(ws + l.tiles), a.z = reinterpret_cast<float *>(ws + l.z);
    a.n_mats = kept, a.n_adapters = n_adapters, a.max_rank = max_rank, a.in_dim = in_dim, a.rows = rows, a.splits = l.splits;
    const bool few = rows <= qlin::kFewRows;
    a.chunk = few ? 256 : 1024;
    int runs = 0;
    for (int i = 0; i < kept; ++i) a.chunks[i] = runs += (a.mats[i].out_dim + a.chunk - 1) / a.chunk;
    const int64_t downs = static_cast<int64_t>(l.most_tiles) * kept * l.groups * l.splits, ups = static_cast<int64_t>(l.most_tiles) * runs;
    const hipStream_t s = static_cast<hipStream_t>(qlin_get_stream());
    const size_t lds = sizeof(float) * (few ? 16 : qlin::kTile) * ((max_rank + 31) / 32 * 32 + 4);
    auto go = [&](auto down, auto up) {
        if (!few) hipLaunchKernelGGL(qlin::lora_group_kernel, dim3(1), dim3(qlin::kGroupThreads), 0, s, a);
        hipLaunchKernelGGL(down, dim3(static_cast<unsigned>(few ? downs : downs < 2048 ? downs : 2048)), dim3(qlin::kThreads), 0, s, a);
        hipLaunchKernelGGL(up, dim3(static_cast<unsigned>(ups < 2048 ? ups : 2048)), dim3(qlin::kThreads), lds, s, a);
        return hipGetLastError() == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH;
    };
    using namespace qlin;
    switch (weight_type) {
        case 0: return few ? go(lora_down_kernel<0, true>, lora_up_kernel<0, true>) : go(lora_down_kernel<0, false>, lora_up_kernel<0, false>);
        case 1: return few ? go(lora_down_kernel<1, true>, lora_up_kernel<1, true>) : go(lora_down_kernel<1, false>, lora_up_kernel<1, false>);
        default: return few ? go(lora_down_kernel<2, true>, lora_up_kernel<2, true>) : go(lora_down_kernel<2, false>, lora_up_kernel<2, false>);
    }
}

}  // extern "C"
