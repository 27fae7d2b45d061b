// qlin_lora.hip -- low-rank adapters of many requests beside a shared projection (qlin_launch_lora_add, qlin_decoder.h),
// gfx950.
//
// Mathematics: z = A x, y = base + B (scale z), A and B those of the row's adapter.
//
// Rows of one adapter stand in tiles, of 16 rows (up to 256 rows in all, where each wave groups the ids by itself) or of 64 (a
// launch of one workgroup before the others).  Weights are the A operand of the matrix cores, rows of x and
// z the B operand.
// 1. lora_down_kernel: z of a tile, up to 64 ranks and a slice of x: 4 waves take parts of the slice and meet in LDS.  Slices
//    are stored apart and added up by the second launch, in order: no atomics.
// 2. lora_up_kernel: a tile and a run of outputs, scale z in LDS.
//
// Products are exact.  bf16 and f16 weights go to v_mfma_f32_16x16x32_bf16: an f16 weight is the sum of two bf16 values, and
// 2^26 v of an f32 value v is the sum of three (8 bits each; with the factor, which leaves with the sum, all parts of any v are
// normal numbers).  Where a |v| is 2^60 or more (or infinite) these would overflow: such values of x, and the rows of z that have
// one, go to v_mfma_f32_16x16x4_f32 after the others, a uniform and rare branch, so that no row's result depends on the rows beside
// it; f32 weights go there always: 613 rows of 18944 to 3584 with 8 adapters of rank 64 51 us in a graph, of f16 42 and of bf16
// 35; 2011 of 4096 to 14336 with 3 97, 76 and 68.
//
// Few rows are bound by latency: one row of 896 to 896, 128 and 128 at rank 16 takes 9.7 us in a graph, 48 rows of 3584 to 3584,
// 512 and 512 with 15 adapters of rank 32 15.8.  Many are bound by memory in the second launch (2011 rows of 4096 to 14336 at rank
// 64: 230 MB of base and y, 55.7 us, 4.1 TB/s, 77.2 in all) and in the first by what a wave has to do between its loads: x into
// three parts and f16 weights into two take the vector unit 40 of 100 cycles, the products the matrix unit 20.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "qlin.h"
#include "qlin_decoder.h"
#include "qlin_bf16x3.hpp"
#include "qlin_device.hpp"
#include "qlin_internal.hpp"

namespace qlin {
namespace {

constexpr int kMostMats = 4;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kFewRows = 256;   // grouped by each wave; with more, a launch groups them
constexpr int kTile = 64;       // the most rows of a tile
constexpr int kUpThreads = 512;  // of lora_up_kernel over tiles of 64 rows
constexpr int kPart = 32;       // of a workgroup of lora_down_kernel
constexpr int kRanks = 64;      // of a workgroup of lora_down_kernel
constexpr int kMostAdapters = 1024;

// Rows that have one adapter (-1: none), with its rank and scale; no rows: no such tile.
struct Group {
    int adapter, count, rank;
    float scale;
};
struct Tile {  // in the workspace
    Group group;
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
    int n_mats, n_adapters, max_rank, in_dim, rows, splits, most_tiles;
    int copies;  // whether rows without an adapter are copied (somewhere y is not base)
    int chunk, chunks[kMostMats];  // outputs of a workgroup of lora_up_kernel, and their runs up to and with each projection
};

// the adapter's slot; n_adapters for none; -1 for a row with nothing to do
__device__ __forceinline__ int slot_of(const LoraArgs &a, int row) {
    const int id = a.ids[row];
    return id >= 0 && id < a.n_adapters ? id : a.copies ? a.n_adapters : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs &a, int id) { return a.ranks ? min(max(a.ranks[id], 0), a.max_rank) : a.max_rank; }
__device__ __forceinline__ Group group_of(const LoraArgs &a, int id, int count) {
    return id < a.n_adapters ? Group{id, count, rank_of(a, id), a.scales ? a.scales[id] : 1.0f} : Group{-1, count, 0, 1.0f};
}

// Loads and stores.  Eight lanes take a line of 128 bytes, a wave 8 rows, so that no line is met by two instructions: the second
// would wait in the first level cache for the first one's miss, with all that comes after it.  (The lanes as the matrix cores
// take them, row l % 16 and the values 8 (l / 16) .., 2011 rows of 4096 to 14336 at rank 64 took 19.5 and 78.6 us, with the cache
// stalled for two thirds of it; four lanes to half a line 20.1 and 73.3; so 16.9 and 61.)  What is loaded changes lanes through LDS of the
// wave's own, rows 144 bytes apart, so that 16 lanes with 16 bytes of 16 rows meet all banks.
constexpr int kLine = 128, kRowBytes = kLine + 16;

// what the wave has written to LDS is read by other lanes of it, or the other way round
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// rows 8 i + lane / 8, 16 bytes each lane
template <int N, class V>
__device__ __forceinline__ void put_rows(char *lds, const V (&v)[N], int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<V *>(lds + (8 * i + (lane >> 3)) * kRowBytes + 16 * (lane & 7)) = v[i];
}

constexpr float kUp = 0x1p26f, kDown = 0x1p-26f, kWide = 0x1p60f;

// 8 weights of a type (0 bf16, 1 f16, 2 f32), and as f32 values
template <int T>
struct Weights {
    static constexpr int kBytes = T == 2 ? 4 : 2, kValues = kLine / kBytes;  // of a line
    u32x4 v[T == 2 ? 2 : 1];
    // values 8 i .. of a row in LDS
    __device__ __forceinline__ void get(const char *row, int i) {
#pragma unroll
        for (int h = 0; h < (T == 2 ? 2 : 1); ++h) v[h] = *reinterpret_cast<const u32x4 *>(row + 8 * kBytes * i + 16 * h);
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
};
// only the first n values of the 16 bytes at v count (no choice that would be a branch: a wait would come with it)
template <int T>
__device__ __forceinline__ void keep_weights(u32x4 &v, int n) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        if constexpr (T == 2) v[d] &= static_cast<uint32_t>((d - n) >> 31);
        else v[d] &= (static_cast<uint32_t>((2 * d - n) >> 31) & 0xffffu) | (static_cast<uint32_t>((2 * d + 1 - n) >> 31) & 0xffff0000u);
    }
}

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// The bf16 operands of 8 bf16 or f16 weights: the weights, or what their 8 leading bits are and the rest.
template <int T>
struct Operands {
    u32x4 hi, lo;
    __device__ __forceinline__ explicit Operands(const Weights<T> &w) {
        if constexpr (T == 0) {
            hi = w.v[0];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = w.at(2 * i), b = w.at(2 * i + 1);
                hi[i] = bf16_tops(a, b);
                lo[i] = bf16_tops(a - bf16_hi_val(__builtin_bit_cast(uint32_t, a)), b - bf16_hi_val(__builtin_bit_cast(uint32_t, b)));
            }
        }
    }
    // acc += weights times the three parts of 8 values; the large products first
    __device__ __forceinline__ f32x4 times(const u32x4 &h, const u32x4 &m, const u32x4 &l, f32x4 acc) const {
        acc = mfma_bf16(hi, h, acc);
        acc = mfma_bf16(hi, m, acc);
        if constexpr (T == 1) acc = mfma_bf16(lo, h, acc);
        acc = mfma_bf16(hi, l, acc);
        if constexpr (T == 1) {
            acc = mfma_bf16(lo, m, acc);
            acc = mfma_bf16(lo, l, acc);
        }
        return acc;
    }
};
template <int T>
__device__ __forceinline__ f32x4 mfma_f32(const Weights<T> &w, const f32x4 (&v)[2], f32x4 acc) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.at(e), v[e >> 2][e & 3], acc, 0, 0, 0);
    return acc;
}

// A tile's rows: in LDS, or of up to 16 in lanes 0 .. 15 of each wave.
struct TileRows {
    const int *rows;
    __device__ __forceinline__ int operator()(int i) const { return rows[i]; }
};
struct LaneRows {
    int row;
    __device__ __forceinline__ int operator()(int i) const { return __builtin_amdgcn_ds_bpermute(4 * i, row); }
};
// The tile of number `tile` among up to 256 rows, by each wave for itself, 64 rows at a time: adapters in the order of their
// first rows, an adapter's rows in order, so that every wave finds the same.  No LDS, no barrier: with both and a row a
// thread one row of 896 to 896, 128 and 128 took 15.3 us in the two launches, so 9.6.
__device__ __forceinline__ Group find_tile(const LoraArgs &a, int tile, LaneRows &rows) {
    constexpr int I = kFewRows / 64;
    const int lane = threadIdx.x & 63;
    const uint64_t below = (1ull << lane) - 1;
    int slot[I];
    uint64_t todo[I], mine[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
        slot[i] = -1;
        if (64 * i < a.rows && 64 * i + lane < a.rows) slot[i] = slot_of(a, 64 * i + lane);
    }
#pragma unroll
    for (int i = 0; i < I; ++i) todo[i] = __ballot(slot[i] >= 0);
    int id = 0, count = 0;
#pragma unroll 1
    for (;;) {  // uniform
        if (todo[0]) id = __builtin_amdgcn_readlane(slot[0], __builtin_ctzll(todo[0]));
        else if (todo[1]) id = __builtin_amdgcn_readlane(slot[1], __builtin_ctzll(todo[1]));
        else if (todo[2]) id = __builtin_amdgcn_readlane(slot[2], __builtin_ctzll(todo[2]));
        else if (todo[3]) id = __builtin_amdgcn_readlane(slot[3], __builtin_ctzll(todo[3]));
        else return Group{-1, 0, 0, 1.0f};
        count = 0;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            mine[i] = __ballot(slot[i] == id);
            todo[i] &= ~mine[i];
            count += static_cast<int>(__popcll(mine[i]));
        }
        const int n = (count + 15) / 16;
        if (tile < n) break;
        tile -= n;
    }
    // each row to the lane of its place, plus one; lanes that nothing comes to get 0
    int before = -16 * tile, row = 0;
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const int place = before + static_cast<int>(__popcll(mine[i] & below));
        const bool in = (mine[i] >> lane & 1) && place >= 0 && place < 16;
        row = max(row, __builtin_amdgcn_ds_permute(4 * (in ? place : 63), in ? 64 * i + lane + 1 : 0));
        before += static_cast<int>(__popcll(mine[i]));
    }
    rows.row = max(row - 1, 0);  // (lanes past the last row: another)
    return group_of(a, id, min(16, count - 16 * tile));
}
static_assert(kFewRows == 256, "find_tile has four registers of rows");

// More rows: one workgroup counts each adapter's rows, gives it its tiles and puts the rows into them.  (In what order does
// not matter: a row's results do not depend on its place.)
constexpr int kGroupThreads = 1024, kKept = 4;  // rows a thread whose places are kept in registers
__global__ __launch_bounds__(kGroupThreads) void lora_group_kernel(LoraArgs a) {
    __shared__ int s_count[kMostAdapters + 1], s_tile[kMostAdapters + 1], s_wave[kGroupThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, kinds = a.n_adapters + 1;
    int slot[kKept], place[kKept];
    const Group mine = group_of(a, tid, 0);
#pragma unroll
    for (int i = 0; i < kKept; ++i) slot[i] = tid + i * kGroupThreads < a.rows ? slot_of(a, tid + i * kGroupThreads) : -1;
    for (int i = tid; i < kinds; i += kGroupThreads) s_count[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
        place[i] = 0;
        const int first = __builtin_amdgcn_readfirstlane(slot[i]);
        if (__all(slot[i] == first)) {  // a run: one addition for 64 rows, where 64 would come one after the other
            if (first < 0) continue;
            if (lane == 0) place[i] = atomicAdd(&s_count[first], 64);
            place[i] = __builtin_amdgcn_readfirstlane(place[i]) + lane;
        } else if (slot[i] >= 0) {
            place[i] = atomicAdd(&s_count[slot[i]], 1);
        }
    }
    __syncthreads();  // (the kept rows' places are the first ones, those of the rest come after them all)
    const int rest = tid + kKept * kGroupThreads;
    for (int r = rest; r < a.rows; r += kGroupThreads) {
        const int id = slot_of(a, r);
        if (id >= 0) atomicAdd(&s_count[id], 1);
    }
    __syncthreads();
    // (kinds <= 1025: the last one, the rows without an adapter, is thread 1023's second)
    const int count = tid < kinds ? s_count[tid] : 0, last = kinds > kGroupThreads ? s_count[kGroupThreads] : 0;
    const int n = (count + kTile - 1) / kTile;
    int run = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(run, o, 64);
        if (lane >= o) run += up;
    }
    if (lane == 63) s_wave[tid >> 6] = run;
    __syncthreads();
    int start = run - n, total = 0;
#pragma unroll
    for (int w = 0; w < kGroupThreads / 64; ++w) {
        const int v = s_wave[w];
        if (w < (tid >> 6)) start += v;
        total += v;
    }
    auto head = [&](int id, Group of, int at, int rows) {
        s_tile[id] = at;
        for (int t = 0; t * kTile < rows; ++t) {
            of.count = min(kTile, rows - t * kTile);
            a.tiles[at + t].group = of;
        }
    };
    if (tid < kinds) head(tid, mine, start, count);
    if (last > 0 && tid == 0) head(kGroupThreads, Group{-1, 0, 0, 1.0f}, total, last);
    if (tid == 0) *a.n_tiles = total + (last + kTile - 1) / kTile;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept; ++i)
        if (slot[i] >= 0) a.tiles[s_tile[slot[i]] + place[i] / kTile].rows[place[i] % kTile] = tid + i * kGroupThreads;
    if (a.rows > kKept * kGroupThreads) {  // uniform; the rest are counted again, downwards
        for (int r = rest; r < a.rows; r += kGroupThreads) {
            const int id = slot_of(a, r);
            if (id < 0) continue;
            const int at = atomicSub(&s_count[id], 1) - 1;
            a.tiles[s_tile[id] + at / kTile].rows[at % kTile] = r;
        }
    }
}

// Tile number `tile`, its rows into LDS; no rows where there is no such tile.  (All of it is asked for at once: there is room for
// most_tiles of them, of which the first n_tiles are filled.)
__device__ __forceinline__ Group tile_at(const LoraArgs &a, int tile, int *s_rows) {
    const int n = *a.n_tiles, t = min(tile, a.most_tiles - 1);
    Group of = a.tiles[t].group;
    if (threadIdx.x < kTile) s_rows[threadIdx.x] = a.tiles[t].rows[threadIdx.x];
    if (tile >= n) of.count = 0;
    return of;
}

// z of 16 NT rows of a tile from its row `first` on, one projection, one group of ranks and one slice of x.  lds: at least
// kDownBytes for the workgroup.
constexpr int kDownRows = 64;  // of LDS a wave: two lines of 32 rows of x, or a line of 64 rows of weights
constexpr int kDownBytes = kWaves * kDownRows * kRowBytes;
static_assert(kDownBytes >= kWaves * (kRanks / 16) * (kPart / 16) * 64 * 16, "the waves' sums");
template <int T, int NT, class R>
__device__ __forceinline__ void down(const LoraArgs &a, const Group &t, const R &rows, int first, int mat, int group, int split, char *lds) {
    constexpr int RT = kRanks / 16, K = Weights<T>::kValues, H = K / 32;  // a step: a line of weights, H lines of x
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rank = t.rank - group * kRanks;
    if (rank <= 0) return;  // uniform
    const int tiles = min((rank + 15) / 16, RT);
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = zero;
    // (rows past the tile's or the rank's end are others again; what comes of them is not stored)
    const float *x[2 * NT];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) x[j] = a.x + rows(min(first + 8 * j + (lane >> 3), t.count - 1)) * a.x_stride;
    const char *w[2 * RT];
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i)
        w[i] = static_cast<const char *>(a.mats[mat].a) +
               (static_cast<size_t>(t.adapter) * a.max_rank + group * kRanks + min(8 * i + (lane >> 3), rank - 1)) * a.in_dim * Weights<T>::kBytes;
    const int steps = (a.in_dim + K - 1) / K, parts = a.splits * kWaves, part = split * kWaves + wave;
    const int from = static_cast<int>(static_cast<int64_t>(steps) * part / parts), to = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / parts);
    struct Step {
        u32x4 w[RT][2];
        f32x4 x[H][2 * NT];
    };
    // (past the end of x: its last values once more, as zeros)
    auto load = [&](Step &s, int at) {
        const int kx = K * at + 4 * (lane & 7), kw = min(K * at + (16 / Weights<T>::kBytes) * (lane & 7), a.in_dim - 16 / Weights<T>::kBytes);
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int j = 0; j < 2 * NT; ++j) __builtin_memcpy(&s.x[h][j], __builtin_assume_aligned(x[j] + min(kx + 32 * h, a.in_dim - 4), 4), 16);
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (i < tiles) {
#pragma unroll
                for (int h = 0; h < 2; ++h) s.w[i][h] = *reinterpret_cast<const u32x4 *>(w[2 * i + h] + kw * Weights<T>::kBytes);
            }
    };
    // A lane's operands: row n of 16, the values 8 g .. of 32.
    static_assert(H * 16 * NT <= kDownRows && 16 * RT <= kDownRows, "");
    char *mine = lds + wave * (kDownRows * kRowBytes);
    const int n = lane & 15, g = lane >> 4;
    // How a step is taken: on bf16 products all values (not done, and false, where one is kWide or more) or those below kWide; on f32
    // products the other ones, of f32 weights all.
    constexpr int kAll = 0, kSmall = 1, kLarge = 2;
    auto multiply = [&](Step &s, int at, auto how) {
        constexpr int HOW = decltype(how)::value;
        if (K * at + K > a.in_dim) {  // uniform
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s.x[h][j][e] = K * at + 32 * h + 4 * (lane & 7) < a.in_dim ? s.x[h][j][e] : 0.0f;
        }
        f32x4 v[H][NT][2];
        wave_sync();
#pragma unroll
        for (int h = 0; h < H; ++h) put_rows(mine + h * 16 * NT * kRowBytes, s.x[h], lane);
        wave_sync();
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    v[h][j][i] = *reinterpret_cast<const f32x4 *>(mine + (16 * (h * NT + j) + n) * kRowBytes + 32 * g + 16 * i);
        wave_sync();
#pragma unroll
        for (int i = 0; i < RT; ++i)
            if (i < tiles) put_rows(mine + 16 * i * kRowBytes, s.w[i], lane);
        wave_sync();
        if constexpr (HOW != kAll && T != 2) {
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float f = v[h][j][e >> 2][e & 3];
                        v[h][j][e >> 2][e & 3] = (fabsf(f) < kWide) == (HOW == kSmall) ? f : 0.0f;
                    }
        }
        if constexpr (HOW == kLarge) {
#pragma unroll
            for (int i = 0; i < RT; ++i)
                if (i < tiles) {
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        Weights<T> o;
                        o.get(mine + (16 * i + n) * kRowBytes, 4 * h + g);
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[i][j] = mfma_f32(o, v[h][j], acc[i][j]);
                    }
                }
            return true;
        } else {
            if constexpr (HOW == kAll) {
                float top = 0.0f;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 8; e += 2) top = max3_abs(v[h][j][e >> 2][e & 3], v[h][j][e >> 2][(e & 3) + 1], top);
                if (__any(!(top < kWide))) return false;
            }
            u32x4 hi[H][NT], mid[H][NT], lo[H][NT];
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j) split3(v[h][j][0] * kUp, v[h][j][1] * kUp, hi[h][j], mid[h][j], lo[h][j]);
#pragma unroll
            for (int i = 0; i < RT; ++i)
                if (i < tiles) {
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        Weights<T> r;
                        r.get(mine + (16 * i + n) * kRowBytes, 4 * h + g);
                        const Operands<T> o(r);
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[i][j] = o.times(hi[h][j], mid[h][j], lo[h][j], acc[i][j]);
                    }
                }
            return true;
        }
    };
    Step s;
    int at = from;
    if (at < to) load(s, at);
    if constexpr (T != 2) {
        // (acc is 2^26 z)
        bool fits = true;
#pragma unroll 1
        while (at < to) {
            Step now = s;
            if (at + 1 < to) load(s, at + 1);
            fits = multiply(now, at, std::integral_constant<int, kAll>());
            if (!fits) break;  // uniform
            ++at;
        }
        // from the first step with a large value on: the small ones as before, in the same order, and the large ones after them, so that a row
        // without any has the same sum
        const int first_large = at;
#pragma unroll 1
        for (; at < to; ++at) {
            load(s, at);
            multiply(s, at, std::integral_constant<int, kSmall>());
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] *= kDown;
#pragma unroll 1
        for (at = first_large; at < to; ++at) {
            load(s, at);
            multiply(s, at, std::integral_constant<int, kLarge>());
        }
    } else {
#pragma unroll 1
        for (; at < to; ++at) {
            Step now = s;
            if (at + 1 < to) load(s, at + 1);
            multiply(now, at, std::integral_constant<int, kLarge>());
        }
    }
    __syncthreads();  // (the waves' rows are read)
    f32x4 *s_z = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (i < tiles) s_z[((wave * RT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    // a lane takes ranks 4 (l % 4) .. of row l / 4
    const int of = 16 * (lane & 3) + (lane >> 2);
#pragma unroll
    for (int i = 0; i < RT * NT; i += kWaves) {
        const int tile = i + wave, rt = tile / NT, j = tile % NT;
        if (rt >= tiles) continue;
        f32x4 sum = s_z[tile * 64 + of];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += s_z[(v * RT * NT + tile) * 64 + of];
        const int at = first + 16 * j + (lane >> 2), row = rows(min(at, t.count - 1)), k = group * kRanks + 16 * rt + 4 * (lane & 3);
        if (at < t.count && k < a.max_rank)
            *reinterpret_cast<f32x4 *>(a.z + ((static_cast<size_t>(split) * a.n_mats + mat) * a.rows + row) * a.max_rank + k) = sum;
    }
}

// FEW: tiles of 16 that each wave finds, a workgroup for each that there can be; else those that there are, in turn.
template <int T, bool FEW>
__global__ __launch_bounds__(kThreads, 2) void lora_down_kernel(LoraArgs a) {
    __shared__ __attribute__((aligned(16))) char s_z[kDownBytes];
    const int groups = (a.max_rank + kRanks - 1) / kRanks, units = a.n_mats * groups * a.splits * (FEW ? 1 : kTile / kPart);
    if constexpr (FEW) {
        const int unit = blockIdx.x % units, split = unit % a.splits, rest = unit / a.splits;
        LaneRows rows;
        const Group t = find_tile(a, blockIdx.x / units, rows);
        if (t.adapter >= 0) down<T, 1>(a, t, rows, 0, rest % a.n_mats, rest / a.n_mats, split, s_z);
    } else {
        __shared__ int s_rows[kTile];
        const TileRows rows = {s_rows};
        for (int item = blockIdx.x;; item += gridDim.x) {
            const int unit = item % units;
            __syncthreads();  // (the tile and the sums of before are read)
            const Group of = tile_at(a, item / units, s_rows);
            if (of.count == 0) break;  // uniform
            __syncthreads();
            const int split = unit % a.splits, part = unit / a.splits % (kTile / kPart) * kPart, rest = unit / a.splits / (kTile / kPart);
            if (of.adapter < 0 || part >= of.count) continue;  // uniform
            if (of.count - part <= 16) down<T, 1>(a, of, rows, part, rest % a.n_mats, rest / a.n_mats, split, s_z);
            else down<T, kPart / 16>(a, of, rows, part, rest % a.n_mats, rest / a.n_mats, split, s_z);
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

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// scale z of a tile in LDS: the three bf16 parts of 2^26 of it (Z of bf16 and f16 weights), or f32 values; 0 past the rank.
struct Staged {
    int stride, part;  // bytes from a row to the next one, and from a part
};

// y of 16 NT rows of a tile from its row `from` on, 32 outputs at a time: a line of each row.
// (Rows past the tile's end, ranks past the slot's and outputs past the last one are others again; what comes of them is not
// stored.)
template <int T, int NT>
struct Up {
    static constexpr int K = Weights<T>::kValues, H = K / 32;  // a line of weights
    const qlin_lora &m;
    const float *base[2 * NT];
    float *y[2 * NT];
    bool there[2 * NT];  // rows to be stored
    f32x4 was[2 * NT];
    u32x4 ahead[4];  // the first line of weights of the next outputs
    const char *b;
    char *mine;
    int lane, rank, max_rank;

    template <class R>
    __device__ __forceinline__ Up(const LoraArgs &a, const Group &t, const R &rows, int mat, int from, int rank, char *mine)
        : m(a.mats[mat]), mine(mine), lane(threadIdx.x & 63), rank(rank), max_rank(a.max_rank) {
        b = static_cast<const char *>(m.b) + static_cast<size_t>(max(t.adapter, 0)) * m.out_dim * max_rank * Weights<T>::kBytes;
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
            const int at = from + 8 * j + (lane >> 3), row = rows(min(at, t.count - 1));
            there[j] = at < t.count;
            base[j] = m.base + row * m.base_stride + 4 * (lane & 7);
            y[j] = m.y + row * m.y_stride + 4 * (lane & 7);
        }
    }
    // Only the tile's rows in the mask are stored.
    __device__ __forceinline__ void choose(uint64_t mask, int from, int count) {
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
            const int at = from + 8 * j + (lane >> 3);
            there[j] = at < count && (mask >> at & 1);
        }
    }
    // Weights come before the base: loads arrive in order, and the products can go ahead of it.
    __device__ __forceinline__ void load(int o) {
        if (rank > 0) weights(ahead, o, 0);
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
            if (o + 32 <= m.out_dim) __builtin_memcpy(&was[j], __builtin_assume_aligned(base[j] + o, 4), 16);  // uniform
            else was[j] = values_at(base[j], o, m.out_dim - 4 * (lane & 7));
        }
    }
    __device__ __forceinline__ void weights(u32x4 (&w)[4], int o, int c) const {
        constexpr int each = 16 / Weights<T>::kBytes;
        const int k = min(K * c + each * (lane & 7), max_rank - each);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = *reinterpret_cast<const u32x4 *>(b + (static_cast<size_t>(min(o + 8 * i + (lane >> 3), m.out_dim - 1)) * max_rank + k) * Weights<T>::kBytes);
    }
    template <bool WIDE>
    __device__ __forceinline__ void multiply(f32x4 (&sum)[2][NT], u32x4 (&w)[4], int c, const Staged &z, const char *first) const {
        constexpr int each = 16 / Weights<T>::kBytes;
        if (K * c + K > rank) {  // uniform
#pragma unroll
            for (int i = 0; i < 4; ++i) keep_weights<T>(w[i], rank - K * c - each * (lane & 7));
        }
        wave_sync();
        put_rows(mine, w, lane);
        wave_sync();
        const int n = lane & 15, g = lane >> 4;
        first += n * z.stride;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (K * c + 32 * h >= rank) break;  // uniform
            const int k = K * c + 32 * h + 8 * g;
            Weights<T> r[2];
            r[0].get(mine + n * kRowBytes, 4 * h + g);
            r[1].get(mine + (16 + n) * kRowBytes, 4 * h + g);
            if constexpr (WIDE) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    f32x4 v[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) v[i] = *reinterpret_cast<const f32x4 *>(first + 16 * j * z.stride + 4 * k + 16 * i);
                    sum[0][j] = mfma_f32(r[0], v, sum[0][j]);
                    sum[1][j] = mfma_f32(r[1], v, sum[1][j]);
                }
            } else {
                const Operands<T> b0(r[0]), b1(r[1]);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    u32x4 v[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) v[i] = *reinterpret_cast<const u32x4 *>(first + 16 * j * z.stride + 2 * k + i * z.part);
                    sum[0][j] = b0.times(v[0], v[1], v[2], sum[0][j]);
                    sum[1][j] = b1.times(v[0], v[1], v[2], sum[1][j]);
                }
            }
        }
    }
    // y of outputs o .. o + 31, whose loads are on their way; those of next (if any) follow before anything waits for
    // these.  z: the first row's.
    template <bool WIDE>
    __device__ __forceinline__ void add(int o, int next, const Staged &z, const char *first) {
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        f32x4 sum[2][NT];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NT; ++j) sum[h][j] = zero;
        f32x4 now[2 * NT];
        u32x4 w[4];
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) now[j] = was[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = ahead[i];
        if (next >= 0) load(next);
        if (rank > 0) multiply<WIDE>(sum, w, 0, z, first);
#pragma unroll 1
        for (int c = 1; K * c < rank; ++c) {
            weights(w, o, c);
            multiply<WIDE>(sum, w, c, z, first);
        }
        if (rank > 0) {
            wave_sync();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    *reinterpret_cast<f32x4 *>(mine + (16 * j + (lane & 15)) * kRowBytes + 64 * h + 16 * (lane >> 4)) = sum[h][j];
            wave_sync();
#pragma unroll
            for (int j = 0; j < 2 * NT; ++j) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(mine + (8 * j + (lane >> 3)) * kRowBytes + 16 * (lane & 7));
#pragma unroll
                for (int e = 0; e < 4; ++e) now[j][e] = fmaf(v[e], WIDE ? 1.0f : kDown, now[j][e]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j)
            if (there[j]) {
                if (o + 32 <= m.out_dim) {  // uniform
                    if constexpr (NT > 1) __builtin_nontemporal_store(now[j], reinterpret_cast<f32x4u *>(y[j] + o));
                    else __builtin_memcpy(__builtin_assume_aligned(y[j] + o, 4), &now[j], 16);
                } else {
                    store_values(y[j], o, m.out_dim - 4 * (lane & 7), now[j]);
                }
            }
    }
};
constexpr int kUpBytes = 32 * kRowBytes;  // of a wave

// One run of outputs of one tile, by N threads.  s_z: the waves' own rows, then z of at most M rows.
template <int T, int N, int M, class R>
__device__ __forceinline__ void up(const LoraArgs &a, const Group &t, const R &rows, int run, char *s_z, uint32_t (&s_wide)[2]) {
    int mat = 0;
    while (run >= a.chunks[mat]) ++mat;
    if (mat > 0) run -= a.chunks[mat - 1];
    if (t.adapter < 0 && a.mats[mat].y == a.mats[mat].base) return;  // uniform
    char *const s_parts = s_z + N / 64 * kUpBytes;
    const int width = (a.max_rank + 31) / 32 * 32, wave = threadIdx.x >> 6;
    const int first = run * a.chunk, last = min(first + a.chunk, a.mats[mat].out_dim);
    // a wave takes 32 rows (16 of few): where there are more, waves go two by two
    constexpr int NT = M > 16 ? 2 : 1;
    const bool both = t.count > 16 * NT;
    const int from = both ? 16 * NT * (wave & 1) : 0, step = 32 * (N / 64) / (both ? 2 : 1);
    // Two waves that share outputs go through them half the way apart: the second to ask for a line of weights that is on its way
    // would wait with all that comes after it (2011 rows of 4096 to 14336 at rank 64 82.9 us, so 77.3).
    const int start = first + 32 * (both ? wave >> 1 : wave);
    const int passes = start < last ? (last - start + step - 1) / step : 0, turn = both && (wave & 1) ? passes / 2 : 0;
    auto at = [&](int i) { i += turn; return start + step * (i < passes ? i : i - passes); };
    const int rank = t.rank;
    Up<T, NT> up(a, t, rows, mat, from, rank, s_z + wave * kUpBytes);
    if (passes > 0) up.load(at(0));  // (requested before z is staged)
    const int quads = (rank + 31) / 32 * 8;  // of a row
    const int staged = (t.count + 15) / 16 * 16 * quads;
    const size_t split = static_cast<size_t>(a.n_mats) * a.rows * a.max_rank;
    auto z_of = [&](int row, int k) {  // scale z, 4 values; row < 0: none
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row >= 0 && k < rank) {
            const float *p = a.z + (static_cast<size_t>(mat) * a.rows + row) * a.max_rank + k;
            int s = 0;
#pragma unroll 1
            for (; s + 4 <= a.splits; s += 4) {
                f32x4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const f32x4 *>(p + (s + i) * split);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += v[i];
            }
#pragma unroll 1
            for (; s < a.splits; ++s) sum += *reinterpret_cast<const f32x4 *>(p + s * split);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = k + e < rank ? sum[e] * t.scale : 0.0f;
        }
        return sum;
    };
    auto each = [&](auto put) {  // (whole waves, as rows may stand in their lanes)
#pragma unroll 1
        for (int i0 = wave * 64; i0 < staged; i0 += N) {
            const int i = i0 + (threadIdx.x & 63), r = i / quads;
            const int row = rows(min(r, t.count - 1));
            if (i < staged) put(r, r < t.count ? row : -1, 4 * (i % quads));
        }
    };
    // (rows 16 bytes more than a multiple of 64 apart: 16 lanes meet 16 times 4 banks)
    if constexpr (T != 2) {
        const Staged z = {2 * width + 16, M * (2 * width + 16)};
        each([&](int r, int row, int k) {
            const f32x4 v = z_of(row, k);
            if (!(max3_abs(v[0], v[1], fmaxf(fabsf(v[2]), fabsf(v[3]))) < kWide)) atomicOr(&s_wide[r >> 5], 1u << (r & 31));
            uint2 h, m, l;
            split3(v[0] * kUp, v[1] * kUp, h.x, m.x, l.x);
            split3(v[2] * kUp, v[3] * kUp, h.y, m.y, l.y);
            char *at = s_parts + r * z.stride + 2 * k;
            *reinterpret_cast<uint2 *>(at) = h;
            *reinterpret_cast<uint2 *>(at + z.part) = m;
            *reinterpret_cast<uint2 *>(at + 2 * z.part) = l;
        });
        __syncthreads();
        const uint64_t apart = static_cast<uint64_t>(s_wide[1]) << 32 | s_wide[0];  // rows with a value that the parts cannot hold
        if (apart) up.choose(~apart, from, t.count);  // uniform
        const char *rows_z = s_parts + from * z.stride;
#pragma unroll 1
        for (int i = 0; i < passes; ++i) up.template add<false>(at(i), i + 1 < passes ? at(i + 1) : -1, z, rows_z);
        if (!apart) return;  // uniform
        up.choose(apart, from, t.count);
        if (passes > 0) up.load(at(0));
        __syncthreads();  // (the parts are read)
    }
    const Staged z = {4 * width + 16, 0};
    each([&](int r, int row, int k) { *reinterpret_cast<f32x4 *>(s_parts + r * z.stride + 4 * k) = z_of(row, k); });
    __syncthreads();
    const char *rows_z = s_parts + from * z.stride;
#pragma unroll 1
    for (int i = 0; i < passes; ++i) up.template add<true>(at(i), i + 1 < passes ? at(i + 1) : -1, z, rows_z);
}

template <int T, bool FEW>
__global__ __launch_bounds__(FEW ? kThreads : kUpThreads, 2) void lora_up_kernel(LoraArgs a) {
    extern __shared__ __attribute__((aligned(16))) char s_z[];
    __shared__ uint32_t s_wide[2];  // of a tile's rows
    const int runs = a.chunks[a.n_mats - 1];
    if constexpr (FEW) {
        LaneRows rows;
        const Group t = find_tile(a, blockIdx.x / runs, rows);
        if (t.count == 0) return;  // uniform
        if (threadIdx.x < 2) s_wide[threadIdx.x] = 0;
        __syncthreads();
        up<T, kThreads, 16>(a, t, rows, blockIdx.x % runs, s_z, s_wide);
    } else {
        __shared__ int s_rows[kTile];
        const TileRows rows = {s_rows};
        for (int item = blockIdx.x;; item += gridDim.x) {
            __syncthreads();  // (the tile of before is read)
            const Group of = tile_at(a, item / runs, s_rows);
            if (of.count == 0) break;  // uniform
            if (threadIdx.x < 2) s_wide[threadIdx.x] = 0;
            __syncthreads();
            up<T, kUpThreads, kTile>(a, of, rows, item % runs, s_z, s_wide);
        }
    }
}

bool al(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Whether each wave groups the rows: what that takes grows with the adapters in use, 64 rows at a time, a launch for it takes 4 us.
// (How many are in use stands on the device alone; there are no more than slots.)
bool few_of(int rows, int n_adapters) { return rows <= 64 || (rows <= kFewRows && n_adapters < 32); }

struct Layout {
    int most_tiles, groups, splits;
    size_t tiles, z, bytes;
};
Layout layout_of(int rows, int n_mats, int n_adapters, int max_rank, int in_dim) {
    Layout l;
    const bool few = few_of(rows, n_adapters);
    const int m = few ? 16 : kTile, kinds = rows < n_adapters + 1 ? rows : n_adapters + 1;
    l.most_tiles = rows / m + kinds;
    if (l.most_tiles > rows) l.most_tiles = rows;
    l.groups = (max_rank + kRanks - 1) / kRanks;
    // slices of x: as many as give about 512 workgroups, but each is stored apart and read by every run of outputs, so that a
    // wave has 8 steps of 32 values at least, 2 of few rows, where it is latency that counts (2011 rows of 4096 to 14336 in 8
    // slices of 4 steps 85.0 us, in 4 of 8 82.2); 16 at most (613 rows of 18944 to 3584 in 8 47.5 us, in 16 43.1, in 18 to 32 45.5)
    const int steps = (in_dim + 31) / 32, least = few ? 2 : 8;
    const int64_t tiles = few ? l.most_tiles : (rows + kPart - 1) / kPart;
    l.splits = static_cast<int>(512 / (tiles * n_mats * l.groups));
    if (l.splits > steps / (least * kWaves)) l.splits = steps / (least * kWaves);
    if (l.splits > 16) l.splits = 16;
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
    a.n_mats = kept, a.n_adapters = n_adapters, a.max_rank = max_rank, a.in_dim = in_dim, a.rows = rows, a.splits = l.splits, a.most_tiles = l.most_tiles;
    const bool few = qlin::few_of(rows, n_adapters);
    // outputs of a workgroup: as many as leave 256 workgroups, since each stages z again (128: 2048 rows of 4096 to 4096 at rank 16
    // 40.8 us, 256: 37.0), but a step of its waves at least
    int64_t outputs = 0;
    for (int i = 0; i < kept; ++i) outputs += a.mats[i].out_dim;
    const int64_t tiles = few ? l.most_tiles : (rows + qlin::kTile - 1) / qlin::kTile;
    a.chunk = 4096;
    while (a.chunk > (few ? 128 : 256) && tiles * outputs < static_cast<int64_t>(256) * a.chunk) a.chunk /= 2;
    int runs = 0;
    for (int i = 0; i < kept; ++i) a.chunks[i] = runs += (a.mats[i].out_dim + a.chunk - 1) / a.chunk;
    const int64_t downs = static_cast<int64_t>(l.most_tiles) * kept * l.groups * l.splits * (few ? 1 : qlin::kTile / qlin::kPart), ups = static_cast<int64_t>(l.most_tiles) * runs;
    const hipStream_t s = static_cast<hipStream_t>(qlin_get_stream());
    const size_t width = (max_rank + 31) / 32 * 32, m = few ? 16 : qlin::kTile;
    const size_t lds = (few ? qlin::kThreads : qlin::kUpThreads) / 64 * qlin::kUpBytes + (weight_type == 2 ? m * (4 * width + 16) : 3 * m * (2 * width + 16));
    auto go = [&](auto down, auto up) {
        if (!few) hipLaunchKernelGGL(qlin::lora_group_kernel, dim3(1), dim3(qlin::kGroupThreads), 0, s, a);
        hipLaunchKernelGGL(down, dim3(static_cast<unsigned>(few ? downs : downs < 2048 ? downs : 2048)), dim3(qlin::kThreads), 0, s, a);
        hipLaunchKernelGGL(up, dim3(static_cast<unsigned>(few || ups < 2048 ? ups : 2048)), dim3(few ? qlin::kThreads : qlin::kUpThreads), lds, s, a);
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
