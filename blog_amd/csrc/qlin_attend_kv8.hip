// qlin_attend_kv8.hip -- causal grouped-query attention over the 8-bit cache of blocks (qlin_kv8.hpp), gfx950.
//
// Mathematics: o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = (q . k_j) softmax_scale log2(e), in one pass
// over the positions: m is the largest score so far, and the sums are scaled down when it grows.
//
// The 16 query rows of a tile are (row, head of the key head's group) pairs, so that every code is read once for all
// of a group's heads.  Scores are taken as S^T = K q^T and outputs as O^T = V^T P^T on v_mfma_f32_16x16x32_bf16: lane
// (n, g) then holds, of query row n, the probabilities of positions 4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3 of a block,
// which is what it supplies as the second product's operand (the value codes are stored in that order), so that
// probabilities go from one product to the next without leaving their lane.  Codes are exact in bf16; q (times
// softmax_scale log2(e), one rounding) and p are taken in three exact bf16 parts (qlin_bf16x3.hpp).  A block's own sum
// joins the output by one fma with its scale: a chain through the MFMA's C would be cut off downwards each time.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_bf16x3.hpp"
#include "qlin_internal.hpp"
#include "qlin_kv8.hpp"

namespace qlin {

int check_kv8(const qlin_kv8_cache *c);
Kv8View kv8_view(const qlin_kv8_cache *c);

namespace {

constexpr int kWaves = 4, kTile = 16;
constexpr int kMinItems = 8;  // blocks of a split, at least

// over the four lane groups of a query row
__device__ __forceinline__ float groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(a[0])), __builtin_bit_cast(float, static_cast<uint32_t>(a[1])));
    const auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(b[0])), __builtin_bit_cast(float, static_cast<uint32_t>(b[1])));
}
__device__ __forceinline__ float groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = __builtin_bit_cast(float, static_cast<uint32_t>(a[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(b[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(b[1]));
}
// byte j of a dword of codes
__device__ __forceinline__ float code_at(uint32_t w, int j) { return static_cast<float>(static_cast<int8_t>(w >> (8 * j))); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// What a tile of query rows sees: blocks [0, blocks) and `tails` 16-position tiles of the open block.
struct Span {
    int first, last;  // last position seen by the tile's first and last rows (-1: none)
    int done;         // the cache's complete blocks
    int blocks, tails;
    __device__ __forceinline__ int items() const { return blocks + tails; }
};
__device__ __forceinline__ Span span_of(const Kv8Rows &w, int p0, int group) {
    Span s;
    const int r0 = p0 / group, r1 = min((p0 + kTile - 1) / group, w.rows - 1);
    s.first = min(w.start + r0, w.len - 1);
    s.last = min(w.start + r1, w.len - 1);
    s.done = w.len / kKv8Block;
    s.blocks = s.last < 0 ? 0 : min(s.done, s.last / kKv8Block + 1);
    const int open = s.done * kKv8Block;
    s.tails = s.last >= open ? (s.last - open) / 16 + 1 : 0;
    return s;
}
// items of a split, and how many splits have some
__device__ __forceinline__ int items_per_split(int items, int splits) { return max(kMinItems, (items + splits - 1) / splits); }

// One wave's running sums of a tile.
template <int HD>
struct Sums {
    static constexpr int NT = (HD + 63) / 64;
    f32x4 o[NT][4];    // of query row n: [i][j][r] is dim 64 i + 16 g + 4 r + j (past HD: zeros)
    float m, l;        // l: of this lane's positions
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY;
        l = 0.0f;
    }
    // the maximum becomes that of the tile's scores too; returns what is subtracted
    __device__ __forceinline__ float raise(float mx) {
        mx = fmaxf(m, groups_max(mx));
        if (__any(mx > m)) {  // uniform
            const float al = m == -INFINITY ? 0.0f : exp2_fast(m - mx);
            l *= al;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[i][j][r] *= al;
            m = mx;
        }
        return m == -INFINITY ? 0.0f : m;
    }
};

// A workgroup of 4 waves per (tile, sequence, key head, split of the positions); its waves take the split's blocks
// in turn, each with sums of its own, which meet in LDS.
template <int HD>
__global__ __launch_bounds__(64 * kWaves) void attend_kv8_kernel(Kv8View c, const float *__restrict__ q,
                                                                 float *__restrict__ out, int rows, int n_heads,
                                                                 const int *__restrict__ start_pos,
                                                                 const int *__restrict__ n_rows, float q_scale, int tiles,
                                                                 int splits, float *__restrict__ part) {
    constexpr int NC = HD / 32, NT = Sums<HD>::NT;
    __shared__ float s_o[kWaves][kTile][HD + 4];
    __shared__ float s_m[kWaves][kTile], s_l[kWaves][kTile];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    int id = blockIdx.x;
    const int split = id % splits;
    id /= splits;
    const int kh = id % c.kv;
    id /= c.kv;
    const int tile = id % tiles, seq = id / tiles;
    const int group = n_heads / c.kv, p0 = tile * kTile;
    const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, c.per * kKv8Block);
    const int pairs = w.rows * group;
    if (p0 >= pairs) return;
    const Span sp = span_of(w, p0, group);
    const int per = items_per_split(sp.items(), splits), used = max(1, (sp.items() + per - 1) / per);
    if (split >= used) return;

    const int pair = min(p0 + n, pairs - 1);
    const int seen = min(w.start + pair / group, w.len - 1);  // the last position of this lane's query row
    u32x4 qp[3][NC];
    {
        const float *src = q + ((static_cast<size_t>(seq) * rows + pair / group) * n_heads + kh * group + pair % group) * HD + 8 * g;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            f32x4 a = *reinterpret_cast<const f32x4 *>(src + 32 * i), b = *reinterpret_cast<const f32x4 *>(src + 32 * i + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] *= q_scale;
                b[e] *= q_scale;
            }
            split3(a, b, qp[0][i], qp[1][i], qp[2][i]);
        }
    }
    Sums<HD> t;
    t.clear();
    const int end = min((split + 1) * per, sp.items());
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};

    for (int it = split * per + wave; it < min(end, sp.blocks); it += kWaves) {  // uniform
        const int page = c.page(seq, it);
        if (page < 0) continue;
        const uint8_t *rec = c.record(page, kh, kv8_record_bytes(HD));
        const float2 scale = *reinterpret_cast<const float2 *>(rec + 64 * HD);
        u32x4 kc[NC], vc[NT][2];
#pragma unroll
        for (int i = 0; i < NC; ++i) kc[i] = *reinterpret_cast<const u32x4 *>(rec + 1024 * i + 16 * lane);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int odd = 0; odd < 2; ++odd)  // dims 64 i + 4n .. + 3 of positions 4g + odd, + 2, 16 + 4g + odd, + 2
                vc[i][odd] = 64 * (i + 1) <= HD || 64 * i + 4 * n < HD
                                 ? *reinterpret_cast<const u32x4 *>(rec + kv8_value_byte(4 * g + odd, 64 * i + 4 * n, HD))
                                 : u32x4{0u, 0u, 0u, 0u};
        f32x4 hi[2] = {zero, zero}, lo[2] = {zero, zero};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const u32x4 a = bf16_of_i8(kc[i][2 * u], kc[i][2 * u + 1]);
                hi[u] = mfma(a, qp[0][i], hi[u]);
                lo[u] = mfma(a, qp[1][i], lo[u]);
                lo[u] = mfma(a, qp[2][i], lo[u]);
            }
        }
        f32x4 s[2];
        float mx = -INFINITY;
        const int at = it * kKv8Block + 4 * g;
        const bool edge = it * kKv8Block + kKv8Block - 1 > sp.first;  // uniform
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = (hi[u][r] + lo[u][r]) * scale.x;
                if (edge && at + 16 * u + r > seen) v = -INFINITY;
                s[u][r] = v;
                mx = fmaxf(mx, v);
            }
        const float m = t.raise(mx);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[u][r] = exp2_fast(s[u][r] - m);
                t.l += s[u][r];
            }
        u32x4 ph, pm, pl;
        split3(s[0], s[1], ph, pm, pl);
        // a scale that is not finite meets only the rows that see one of the block's positions
        const float vs = edge && it * kKv8Block > seen ? 0.0f : scale.y;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 a;
#pragma unroll
                for (int h = 0; h < 4; ++h)  // positions 4g, 4g + 1; 4g + 2, + 3; 16 + 4g, + 1; 16 + 4g + 2, + 3
                    a[h] = bf16_tops(code_at(vc[i][0][h], j), code_at(vc[i][1][h], j));
                const f32x4 x = mfma(a, ph, zero);
                f32x4 y = mfma(a, pm, zero);
                y = mfma(a, pl, y);
#pragma unroll
                for (int r = 0; r < 4; ++r) t.o[i][j][r] = fmaf(x[r] + y[r], vs, t.o[i][j][r]);
            }
    }

    // The open block, 16 positions at a time, from the ring: f32 on v_mfma_f32_16x16x4_f32, dims and positions in the
    // same lanes as above.
    for (int it = max(split * per, sp.blocks); it < end; ++it) {
        if ((it - split * per) % kWaves != wave) continue;  // uniform
        if (c.page(seq, sp.done) < 0) continue;
        const int base = sp.done * kKv8Block + 16 * (it - sp.blocks);
        const float *kr = c.ring(seq, kh, 0, HD), *vr = c.ring(seq, kh, 1, HD);
        const int mine = base + n;
        const float *krow = kr + static_cast<size_t>(mine % kKv8Recent) * HD + 8 * g;
        f32x4 acc[4] = {zero, zero, zero, zero};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            f32x4 x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = mine < w.len ? *reinterpret_cast<const f32x4 *>(krow + 32 * i + 4 * h) : zero;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float qv = (bf16_at(qp[0][i], j) + bf16_at(qp[1][i], j)) + bf16_at(qp[2][i], j);  // exact
                acc[j % 4] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j / 4][j % 4], qv, acc[j % 4], 0, 0, 0);
            }
        }
        f32x4 s;
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = (acc[0][r] + acc[1][r]) + (acc[2][r] + acc[3][r]);
            s[r] = base + 4 * g + r > seen ? -INFINITY : v;
            mx = fmaxf(mx, s[r]);
        }
        const float m = t.raise(mx);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = exp2_fast(s[r] - m);
            t.l += s[r];
        }
        bool odd = false;  // a value that is not finite, at a position that some row does not see
        f32x4 v[4][NT];  // dims 64 i + 4n .. + 3 of position 4g + r
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int pos = base + 4 * g + r;
            const float *vrow = vr + static_cast<size_t>(pos % kKv8Recent) * HD + 4 * n;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                v[r][i] = pos < w.len && 64 * i + 4 * n < HD ? *reinterpret_cast<const f32x4 *>(vrow + 64 * i) : zero;
#pragma unroll
                for (int j = 0; j < 4; ++j) odd |= !isfinite(v[r][i][j]);
            }
        }
        if (base + 15 > sp.first && __any(odd)) {  // uniform: 0 times that value would be NaN
            for (int j = 0; j < 16 && base + j < w.len; ++j) {
                const int from = 16 * (j / 4) + n;
                float p = j % 4 == 0 ? s[0] : j % 4 == 1 ? s[1] : j % 4 == 2 ? s[2] : s[3];
                p = __shfl(p, from, 64);
                if (base + j <= seen) {
                    const float *vrow = vr + static_cast<size_t>((base + j) % kKv8Recent) * HD;
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int d = 64 * i + 16 * g + 4 * r;
                            const f32x4 y = d < HD ? *reinterpret_cast<const f32x4 *>(vrow + d) : zero;
#pragma unroll
                            for (int e = 0; e < 4; ++e) t.o[i][e][r] = fmaf(p, y[e], t.o[i][e][r]);
                        }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f32x4 x = zero;
#pragma unroll
                    for (int r = 0; r < 4; ++r) x = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][i][j], s[r], x, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) t.o[i][j][r] += x[r];
                }
        }
    }

    t.l = groups_sum(t.l);
    if (g == 0) {
        s_m[wave][n] = t.m;
        s_l[wave][n] = t.l;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = 64 * i + 16 * g + 4 * r;
            if (d < HD) *reinterpret_cast<f32x4 *>(&s_o[wave][n][d]) = f32x4{t.o[i][0][r], t.o[i][1][r], t.o[i][2][r], t.o[i][3][r]};
        }
    __syncthreads();
    for (int e = threadIdx.x; e < kTile * (HD / 4); e += 64 * kWaves) {
        const int row = e / (HD / 4), d = 4 * (e % (HD / 4));
        if (p0 + row >= pairs) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) mx = fmaxf(mx, s_m[i][row]);
        f32x4 num = zero;
        float den = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float mi = s_m[i][row], li = s_l[i][row];
            if (mi == -INFINITY && li == 0.0f) continue;                    // no position of this row
            const float f = mi == -INFINITY ? 1.0f : exp2_fast(mi - mx);  // (-inf: then li is NaN)
            const f32x4 o = *reinterpret_cast<const f32x4 *>(&s_o[i][row][d]);
#pragma unroll
            for (int r = 0; r < 4; ++r) num[r] = fmaf(o[r], f, num[r]);
            den = fmaf(li, f, den);
        }
        if (used == 1) {
            const int pr = p0 + row;
            f32x4 o = zero;
            if (den != 0.0f)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = num[r] / den;
            *reinterpret_cast<f32x4 *>(out + ((static_cast<size_t>(seq) * rows + pr / group) * n_heads + kh * group + pr % group) * HD + d) = o;
        } else {
            // [tile of this launch][split][row]: HD sums, the maximum, the denominator
            float *dst = part + ((static_cast<size_t>(blockIdx.x / splits) * splits + split) * kTile + row) * (HD + 4);
            *reinterpret_cast<f32x4 *>(dst + d) = num;
            if (d == 0) {
                dst[HD] = mx;
                dst[HD + 1] = den;
            }
        }
    }
}

// A workgroup per query row: the splits' sums joined.
constexpr int kJoinThreads = 256;
template <int HD>
__global__ __launch_bounds__(kJoinThreads) void attend_kv8_join_kernel(Kv8View c, float *__restrict__ out, int rows,
                                                                       int n_heads, const int *__restrict__ start_pos,
                                                                       const int *__restrict__ n_rows, int tiles,
                                                                       int splits, const float *__restrict__ part) {
    constexpr int D4 = HD / 4, C = kJoinThreads / D4;
    __shared__ f32x4 s_num[C][D4];
    __shared__ float s_den[C];
    const int row = blockIdx.x % kTile;
    const unsigned group_id = blockIdx.x / kTile;
    int id = group_id;
    const int kh = id % c.kv;
    id /= c.kv;
    const int tile = id % tiles, seq = id / tiles;
    const int group = n_heads / c.kv, p0 = tile * kTile;
    const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, c.per * kKv8Block);
    const int pr = p0 + row;
    if (pr >= w.rows * group) return;
    const Span sp = span_of(w, p0, group);
    const int per = items_per_split(sp.items(), splits), used = (sp.items() + per - 1) / per;
    if (used <= 1) return;  // written already
    const float *src = part + (static_cast<size_t>(group_id) * splits * kTile + row) * (HD + 4);
    const size_t step = static_cast<size_t>(kTile) * (HD + 4);
    float mx = -INFINITY;
    for (int i = threadIdx.x & 63; i < used; i += 64) mx = fmaxf(mx, src[i * step + HD]);
    mx = wave_max_dpp(mx);
    const int cls = threadIdx.x / D4, d4 = threadIdx.x % D4;
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
    float den = 0.0f;
    if (cls < C) {
        for (int i = cls; i < used; i += C) {
            const float mi = src[i * step + HD], li = src[i * step + HD + 1];
            const f32x4 o = *reinterpret_cast<const f32x4 *>(src + i * step + 4 * d4);
            if (mi == -INFINITY && li == 0.0f) continue;
            const float f = mi == -INFINITY ? 1.0f : exp2_fast(mi - mx);
#pragma unroll
            for (int r = 0; r < 4; ++r) num[r] = fmaf(o[r], f, num[r]);
            den = fmaf(li, f, den);
        }
        s_num[cls][d4] = num;
        if (d4 == 0) s_den[cls] = den;
    }
    __syncthreads();
    if (threadIdx.x < D4) {
        f32x4 o = s_num[0][d4];
        float l = s_den[0];
#pragma unroll
        for (int i = 1; i < C; ++i) {
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] += s_num[i][d4][r];
            l += s_den[i];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = l != 0.0f ? o[r] / l : 0.0f;
        *reinterpret_cast<f32x4 *>(out + ((static_cast<size_t>(seq) * rows + pr / group) * n_heads + kh * group + pr % group) * HD + 4 * d4) = o;
    }
}

struct Plan {
    int64_t tiles, groups;  // tiles of a (sequence, key head), of the launch
    int splits;
};
Plan plan_of(int n_seqs, int rows, int n_heads, int kv, int blocks) {
    Plan p;
    p.tiles = (static_cast<int64_t>(rows) * (n_heads / kv) + kTile - 1) / kTile;
    p.groups = p.tiles * kv * n_seqs;
    // two workgroups for every CU, but no split of less than kMinItems blocks of the longest sequence
    const int64_t want = p.groups > 0 ? (512 + p.groups - 1) / p.groups : 1;
    const int64_t most = (blocks + kMinItems) / kMinItems;
    p.splits = static_cast<int>(want < most ? want : most);
    return p;
}

hipStream_t current_stream() { return static_cast<hipStream_t>(qlin_get_stream()); }
bool aligned_to(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace
}  // namespace qlin

extern "C" {

size_t qlin_attend_kv8_workspace_bytes(int n_seqs, int rows, int n_heads, int kv_heads, int head_dim,
                                       int blocks_per_seq) {
    if (n_seqs <= 0 || rows <= 0 || n_heads <= 0 || kv_heads <= 0 || n_heads % kv_heads || head_dim <= 0 || blocks_per_seq <= 0)
        return 0;
    const qlin::Plan p = qlin::plan_of(n_seqs, rows, n_heads, kv_heads, blocks_per_seq);
    if (p.splits <= 1) return 0;
    return static_cast<size_t>(p.groups) * p.splits * qlin::kTile * (static_cast<size_t>(head_dim) + 4) * sizeof(float);
}

int qlin_launch_attend_kv8(const qlin_kv8_cache *cache, const float *q, float *attn, int rows, int n_heads,
                           const int *start_pos_dev, const int *n_rows_dev, float softmax_scale, void *workspace,
                           size_t workspace_bytes) {
    if (int rc = qlin::check_kv8(cache)) return rc;
    const int kv = cache->kv_heads, hd = cache->head_dim;
    if (rows < 0 || n_heads <= 0 || n_heads % kv || !isfinite(softmax_scale)) return QLIN_ERR_SHAPE;
    if (rows > 1 << 20 || n_heads > 65536) return QLIN_ERR_LIMIT;
    if (rows == 0 || cache->n_seqs == 0) return QLIN_OK;
    if (!q || !attn || !start_pos_dev) return QLIN_ERR_NULL;
    if (!qlin::aligned_to(q, 16) || !qlin::aligned_to(attn, 16) || !qlin::aligned_to(start_pos_dev, 4) ||
        !qlin::aligned_to(n_rows_dev, 4) || !qlin::aligned_to(workspace, 16))
        return QLIN_ERR_ALIGN;
    if (static_cast<int64_t>(rows) * (n_heads / kv) > 1 << 30) return QLIN_ERR_LIMIT;
    const qlin::Plan p = qlin::plan_of(cache->n_seqs, rows, n_heads, kv, cache->blocks_per_seq);
    const int64_t grid = p.groups * p.splits;
    if (grid > (1 << 23) || p.groups * qlin::kTile > (1 << 23)) return QLIN_ERR_LIMIT;
    const size_t need = qlin_attend_kv8_workspace_bytes(cache->n_seqs, rows, n_heads, kv, hd, cache->blocks_per_seq);
    if (need > 0 && !workspace) return QLIN_ERR_NULL;
    if (workspace_bytes < need) return QLIN_ERR_LIMIT;
    const float q_scale = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
    float *part = static_cast<float *>(workspace);
    const qlin::Kv8View view = qlin::kv8_view(cache);
    auto go = [&](auto attend, auto join) {
        hipLaunchKernelGGL(attend, dim3(static_cast<unsigned>(grid)), dim3(64 * qlin::kWaves), 0, qlin::current_stream(),
                           view, q, attn, rows, n_heads, start_pos_dev, n_rows_dev, q_scale, static_cast<int>(p.tiles),
                           p.splits, part);
        if (hipGetLastError() != hipSuccess) return QLIN_ERR_LAUNCH;
        if (p.splits > 1) {
            hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(p.groups * qlin::kTile)), dim3(qlin::kJoinThreads), 0,
                               qlin::current_stream(), view, attn, rows, n_heads, start_pos_dev, n_rows_dev,
                               static_cast<int>(p.tiles), p.splits, part);
            if (hipGetLastError() != hipSuccess) return QLIN_ERR_LAUNCH;
        }
        return QLIN_OK;
    };
    switch (hd) {
        case 64: return go(qlin::attend_kv8_kernel<64>, qlin::attend_kv8_join_kernel<64>);
        case 96: return go(qlin::attend_kv8_kernel<96>, qlin::attend_kv8_join_kernel<96>);
        case 128: return go(qlin::attend_kv8_kernel<128>, qlin::attend_kv8_join_kernel<128>);
        case 192: return go(qlin::attend_kv8_kernel<192>, qlin::attend_kv8_join_kernel<192>);
        default: return go(qlin::attend_kv8_kernel<256>, qlin::attend_kv8_join_kernel<256>);
    }
}

}  // extern "C"
