// qlin_attend_kv8.hip -- causal grouped-query attention over the 8-bit cache of blocks (qlin_kv8.hpp), gfx950.
//
// Mathematics: o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = (q . k_j) softmax_scale log2(e), in one pass
// over the positions: m is the largest score so far, and the sums are scaled down when it grows.
//
// The 16 query rows of a tile are (row, head of the key head's group) pairs, so that every code is read once for all
// of a group's heads.  Scores are taken as S^T = K q^T and outputs as O^T = V^T P^T on v_mfma_f32_16x16x32_f16: lane
// (n, g) then holds, of query row n, the probabilities of positions 4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3 of a block,
// which is what it supplies as the second product's operand, so that probabilities go from one product to the next
// without leaving their lane.
//
// Operands: a code is exact in fp16 (1024 + 128 + code by byte permutes, less 1152).  q (times
// softmax_scale log2(e), one rounding, and a power of two that brings its row's largest value to 2^14 .. 2^15) and p
// (times 2^11) are fp16 pairs hi + lo, 22 bits and a sign, so their products with a code are exact and a score is off by
// 2^-23 of its terms.  What is lost besides lies below 2^-39 of a row's largest q, or 2^-36 of its largest p: a
// position of less weight than that adds nothing.  (Three bf16 parts, which lose nothing, took 3 products instead of 2.)
// A block's own sum joins the output by one fma with the block's scale: a chain of blocks through the MFMA's C would be
// cut off downwards each time.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "qlin.h"
#include "qlin_internal.hpp"
#include "qlin_kv8.hpp"
#include "qlin_mfma.hpp"

namespace qlin {

int check_kv8(const qlin_kv8_cache *c);
Kv8View kv8_view(const qlin_kv8_cache *c);

namespace {

constexpr int kTile = 16;
constexpr int kMinItems = 8;  // blocks of a split, at least
constexpr int kCus = 256;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// No instructions in inline assembly here: the compiler does not see what they do to registers that an MFMA is still
// writing (byte-select conversions, 1 instruction a code, wrote such a register before its MFMA's unused lanes did).
// 1024 + 128 + code, in fp16, less 1152
__device__ __forceinline__ uint32_t less_1152(uint32_t biased) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, biased) + f16x2{-1152.0f16, -1152.0f16});
}
// the 8 codes of two dwords, in order: a byte code ^ 0x80 is code + 128, under the byte 0x64 it is that plus 1024
__device__ __forceinline__ u32x4 f16_of_8(uint32_t a, uint32_t b) {
    const uint32_t u = a ^ 0x80808080u, v = b ^ 0x80808080u, k64 = 0x64646464u;
    return u32x4{less_1152(__builtin_amdgcn_perm(k64, u, 0x04010400u)), less_1152(__builtin_amdgcn_perm(k64, u, 0x04030402u)),
                 less_1152(__builtin_amdgcn_perm(k64, v, 0x04010400u)), less_1152(__builtin_amdgcn_perm(k64, v, 0x04030402u))};
}
// byte J of a and of b
template <int J>
__device__ __forceinline__ uint32_t f16_of_bytes(uint32_t a, uint32_t b) {
    return less_1152(__builtin_amdgcn_perm(b, a, 0x0c000c00u | ((4u + J) << 16) | J) ^ 0x64806480u);
}
// hi + lo of two values, each an fp16 pair
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const f32x2 v = {a, b};
    const f16x2 h = __builtin_convertvector(v, f16x2);
    float minus = -1.0f;
    asm("" : "+s"(minus));  // (unknown to the compiler: one v_fma_mix_f32 a value, where it makes two of a difference)
    const f32x2 r = {__builtin_fmaf(static_cast<float>(h[0]), minus, a), __builtin_fmaf(static_cast<float>(h[1]), minus, b)};  // exact
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, f16x2));
}
__device__ __forceinline__ void split2(const f32x4 &a, const f32x4 &b, u32x4 &hi, u32x4 &lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 &v = i < 2 ? a : b;
        uint32_t h, l;
        split2(v[2 * (i & 1)], v[2 * (i & 1) + 1], h, l);
        hi[i] = h;
        lo[i] = l;
    }
}
// value j of 8 packed fp16 values
__device__ __forceinline__ float f16_at(const u32x4 &v, int j) {
    const uint32_t w = v[j >> 1];
    return f16_bits_to_f32(j & 1 ? w >> 16 : w & 0xffffu);
}

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
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// What `count` query rows from p0 on see: blocks [0, blocks) and `tails` 16-position tiles of the open block.
struct Span {
    int first, last;  // last position seen by the first and the last of the rows (-1: none)
    int done;         // the cache's complete blocks
    int blocks, tails;
    __device__ __forceinline__ int items() const { return blocks + tails; }
};
__device__ __forceinline__ Span span_of(const Kv8Rows &w, int p0, int count, int group) {
    Span s;
    const int r0 = p0 / group, r1 = min((p0 + count - 1) / group, w.rows - 1);
    s.first = min(w.start + r0, w.len - 1);
    s.last = min(w.start + r1, w.len - 1);
    s.done = w.len / kKv8Block;
    s.blocks = s.last < 0 ? 0 : min(s.done, s.last / kKv8Block + 1);
    const int open = s.done * kKv8Block;
    s.tails = s.last >= open ? (s.last - open) / 16 + 1 : 0;
    return s;
}
// items of a split
__device__ __forceinline__ int items_per_split(int items, int splits) { return max(kMinItems, (items + splits - 1) / splits); }

// A tile's queries as operands: value j of slot i is dim 32 i + 8 g + j of query row n, times 1 / inv.
template <int HD>
struct Queries {
    u32x4 hi[HD / 32], lo[HD / 32];
    float inv;
    int seen;  // the last position that query row n sees
    struct Raw {
        f32x4 v[HD / 32][2];
        __device__ __forceinline__ void load(const float *row) {
#pragma unroll
            for (int i = 0; i < HD / 32; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) v[i][h] = *reinterpret_cast<const f32x4 *>(row + 32 * i + 4 * h);
        }
    };
    __device__ __forceinline__ void take(Raw &raw, float q_scale) {
        auto &v = raw.v;
        float most = 0.0f;  // (a NaN is not seen here, and is one in its parts)
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                most = fmaxf(fmaxf(most, fabsf(v[i][h][0])), fabsf(v[i][h][1]));
                most = fmaxf(fmaxf(most, fabsf(v[i][h][2])), fabsf(v[i][h][3]));
            }
        const uint32_t top = __float_as_uint(groups_max(most) * fabsf(q_scale));
        const int up = min(127 + 14 - static_cast<int>(top >> 23), 100);  // at most 2^100
        // (a power of two times q_scale: one rounding a value; NaN for a row whose largest is not finite)
        const float scale = top < 0x7f800000u ? __uint_as_float(static_cast<uint32_t>(127 + up) << 23) * q_scale : NAN;
        inv = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][h][e] *= scale;
            split2(v[i][0], v[i][1], hi[i], lo[i]);
        }
    }
};

// One wave's running sums of a tile.
// Probabilities are 2^(s + a) with a = kUp - m, and a is left as it is until a score would give more than 2^(kUp + kSlack):
// after the first few blocks it rarely changes, where the exact maximum of one row in 16 changes in most of a prompt's blocks
// (47 instructions).  From maxima of 2^20 on (kFar), kUp - m and the unrounded s would be off from each other by more than a
// sixteenth, from 2^24 on by more than fp16 has room for: there s is rounded first and a is -m, so that s + a is exact.
constexpr float kUp = 11.0f, kSlack = 4.0f;  // (2^15 at most, in fp16)
constexpr float kFar = 1048576.0f;
template <int HD>
struct Sums {
    static constexpr int NT = (HD + 63) / 64;
    // Of query row n: [i][j][r] is dim 64 i + 16 g + 4 r + j, from the values' dims 64 i + 4n + j in lane n.  Of a head of 96
    // the last 32 are [i][j < 2][r], 64 i + 16 (g % 2) + 4 r + 2 (g / 2) + j, from 64 i + 4 (n % 8) + 2 (n / 8) + j: half the
    // products (as 64 dims, 32 of them zeros, 1000 rows of 28 heads behind 500 positions took 55 us, so 44.5).
    f32x4 o[NT][4];
    float a, l;  // (a: FLT_MAX without a score, whose sum with -inf is -inf)
    bool far;    // uniform: a maximum has been kFar or beyond
    static constexpr bool half(int i) { return 64 * (i + 1) > HD; }
    static constexpr int js(int i) { return half(i) ? 2 : 4; }
    static __device__ __forceinline__ int dim_of(int i, int g, int r) {
        return half(i) ? 64 * i + 16 * (g & 1) + 4 * r + 2 * (g >> 1) : 64 * i + 16 * g + 4 * r;
    }
    static __device__ __forceinline__ int value_dim(int i, int n) { return half(i) ? 64 * i + 4 * (n & 7) + 2 * (n >> 3) : 64 * i + 4 * n; }
    // 4 dims there, of the last 32 of 96 two
    static __device__ __forceinline__ f32x4 dims_at(int i, const float *p) {
        if (!half(i)) return *reinterpret_cast<const f32x4 *>(p);
        const f32x2 x = *reinterpret_cast<const f32x2 *>(p);
        return f32x4{x[0], x[1], 0.0f, 0.0f};
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        a = FLT_MAX;
        l = 0.0f;
        far = false;
    }
    // a for scores s f, of which mx is this lane's largest; far ones are rounded (and f is 1 then)
    template <int U>
    __device__ __forceinline__ void raise(float mx, f32x4 (&s)[U], float &f) {
        if (__any(mx + a > kUp + kSlack) || far) {  // uniform
            const float top = groups_max(mx);
            far |= __any(fabsf(top) >= kFar && top != -INFINITY);
            const float to = fminf(a, top == -INFINITY ? FLT_MAX : fabsf(top) >= kFar ? -top : kUp - top);
            const float al = exp2_fast(to - a);
            l *= al;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < js(i); ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[i][j][r] *= al;
            a = to;
            if (far) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[u][r] *= f;
                f = 1.0f;
            }
        }
    }
    // a block's sums S (positions block * 32 + 16 u + 4 g + r) to probabilities, as operands
    __device__ __forceinline__ void weigh(f32x4 (&s)[2], float f, bool edge, int block, int g, int seen, u32x4 &hi, u32x4 &lo) {
        float mx = -INFINITY;
        if (edge) {  // uniform
            asm volatile("");  // (a branch: as selects these 30 instructions would go with every block)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float v = s[u][r] * f;
                    s[u][r] = block * kKv8Block + 16 * u + 4 * g + r > seen ? -INFINITY : v;
                    mx = fmaxf(mx, s[u][r]);
                }
            f = 1.0f;
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[u][r]);
            mx *= f;  // (f > 0, 0 with sums of 0, or NaN)
        }
        raise(mx, s, f);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[u][r] = exp2_fast(fmaf(s[u][r], f, a));
            }
        split2(s[0], s[1], hi, lo);
        // the sum of the operands that the values meet, by products with ones (8 additions took as long as 5 MFMAs)
        const uint32_t one = 0x3c003c00u;
        const u32x4 ones = {one, one, one, one};
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        l += mfma16(ones, lo, mfma16(ones, hi, zero))[0];
    }
    __device__ __forceinline__ void join(int i, int j, const f32x4 &t, float vs) {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][j][r] = fmaf(t[r], vs, o[i][j][r]);
    }
    // 16 positions of the open block from base on, from the ring: f32 on v_mfma_f32_16x16x4_f32, dims and positions in
    // the same lanes as above.  kr, vr: the ring's keys and values; first: the last position that every row sees.
    __device__ __forceinline__ void tail(const Queries<HD> &q, const float *kr, const float *vr, int base, int len, int first,
                                         int n, int g) {
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        const int mine = base + n;
        const float *krow = kr + static_cast<size_t>(mine % kKv8Recent) * HD + 8 * g;
        f32x4 acc[4] = {zero, zero, zero, zero};
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            f32x4 x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = mine < len ? *reinterpret_cast<const f32x4 *>(krow + 32 * i + 4 * h) : zero;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                acc[e % 4] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e / 4][e % 4], f16_at(q.hi[i], e) + f16_at(q.lo[i], e), acc[e % 4], 0, 0, 0);
        }
        f32x4 s[1];
        float mx = -INFINITY, f = 1.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = ((acc[0][r] + acc[1][r]) + (acc[2][r] + acc[3][r])) * q.inv;
            s[0][r] = base + 4 * g + r > q.seen ? -INFINITY : v;
            mx = fmaxf(mx, s[0][r]);
        }
        raise(mx, s, f);
        f32x4 p;
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = exp2_fast(s[0][r] + a);
        l += groups_sum((p[0] + p[1]) + (p[2] + p[3]));
        bool odd = false;  // a value that is not finite
        f32x4 v[4][NT];    // dims value_dim .. of position 4g + r
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int pos = base + 4 * g + r;
            const float *vrow = vr + static_cast<size_t>(pos % kKv8Recent) * HD;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                v[r][i] = zero;
                if (pos < len) v[r][i] = dims_at(i, vrow + value_dim(i, n));
#pragma unroll
                for (int j = 0; j < js(i); ++j) odd |= !isfinite(v[r][i][j]);
            }
        }
        if (base + 15 > first && __any(odd)) {  // uniform: 0 times that value, for a row that does not see it, would be NaN
            for (int e = 0; e < 16 && base + e < len; ++e) {
                float pe = e % 4 == 0 ? p[0] : e % 4 == 1 ? p[1] : e % 4 == 2 ? p[2] : p[3];
                pe = __shfl(pe, 16 * (e / 4) + n, 64);
                if (base + e <= q.seen) {
                    const float *vrow = vr + static_cast<size_t>((base + e) % kKv8Recent) * HD;
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const f32x4 y = dims_at(i, vrow + dim_of(i, g, r));
#pragma unroll
                            for (int j = 0; j < js(i); ++j) o[i][j][r] = fmaf(pe, y[j], o[i][j][r]);
                        }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < js(i); ++j) {
                    f32x4 x = zero;
#pragma unroll
                    for (int r = 0; r < 4; ++r) x = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][i][j], p[r], x, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[i][j][r] += x[r];
                }
        }
    }
};

// A workgroup of 4 or 8 waves per (RT tiles of 16 query rows, sequence, key head, split of the positions); its waves take the
// split's blocks in turn, each with sums of its own, which meet in LDS.  A wave knows the pages of its next 64 blocks,
// requests a block's keys while it weighs the values of the one before, and turns codes into operands for its RT tiles
// in registers: there is no barrier before the end.
// Few rows (RT = 1): bound by the latency of a wave's few blocks, and by the codes' bytes.  Many (RT = 2): bound by each
// wave's chain of scores, maximum, exponentials, pairs and values, which its registers let only one other wave of the SIMD
// hide: the vector unit issues in 2/3 of the busy cycles, the matrix unit works in 1/3 (2011 rows of 28 heads 68% and 31%,
// 250 behind 6000 of 32 66% and 37%).  Of a tile's 32 x 16 scores, 8 a lane, each costs an fma, an exp, a sum and 2
// instructions for its operands, then 4 fmas for 64 of its values, and half of the codes' 128.  (A workgroup that turned a block's codes once, into
// LDS, for 64 rows took half of these, but one block after the other: the longest row's time, 86 us for 2011 rows of 28
// heads, was all of it.  Codes turned once for all, by a launch before: 92 us, and 2.5 to 5 more for fewer rows.)
// Heads of 128, 28 over 4: one row over 32002 positions 11.2 us, 2.9 TB/s; 24 rows over up to 8000 27.0, 4.2 TB/s (the
// shortest of 20 in a kernel trace); 2011 rows 85.8, 338 TFLOP/s (of one product each; two are made).  32 over 8: 250 rows
// behind 6000 63.8, 394 TFLOP/s (in a run of passes; in the trace, with clocks and caches colder, 99.9 and 74.6).
template <int HD, int RT, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 2) void attend_kv8_kernel(Kv8View c, const float *__restrict__ q,
                                                                    float *__restrict__ out, int rows, int n_heads,
                                                                    const int *__restrict__ start_pos,
                                                                    const int *__restrict__ n_rows, float q_scale, int macros,
                                                                    int splits, float *__restrict__ part) {
    constexpr int NC = HD / 32, NT = Sums<HD>::NT, kRows = RT * kTile;
    __shared__ float s_o[kWaves][kTile][HD + 4];
    __shared__ float s_m[kWaves][kTile], s_l[kWaves][kTile];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    // (neighbours in the grid: splits, then the key heads, whose codes so stay in their XCD's L2; the longest rows first)
    int id = blockIdx.x;
    const int split = id % splits;
    id /= splits;
    const int kh = id % c.kv;
    id /= c.kv;
    const int macro = macros - 1 - id % macros, seq = id / macros;
    const int group = n_heads / c.kv, p0 = macro * kRows;
    typename Queries<HD>::Raw raw[RT];  // (requested first: nothing that is read has to be known)
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const int pair = min(p0 + k * kTile + n, rows * group - 1);
        raw[k].load(q + ((static_cast<size_t>(seq) * rows + pair / group) * n_heads + kh * group + pair % group) * HD + 8 * g);
    }
    const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, c.per * kKv8Block);
    const int pairs = w.rows * group;
    if (p0 >= pairs) return;
    const Span sp = span_of(w, p0, kRows, group);
    const int per = items_per_split(sp.items(), splits), used = max(1, (sp.items() + per - 1) / per);
    if (split >= used) return;
    const int end = min((split + 1) * per, sp.items());
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr size_t kRec = kv8_record_bytes(HD);

    // this wave's blocks: b0, b0 + kWaves, ...; lane i holds the page of the i-th of the next 64
    const int b0 = split * per + wave, b1 = min(end, sp.blocks);
    const int mine = b0 < b1 ? (b1 - b0 + kWaves - 1) / kWaves : 0;  // uniform
    int pages = lane < mine ? c.page(seq, b0 + kWaves * lane) : -1;

    u32x4 kc[NC], vc[NT][2];
    float2 scale;
    auto load_k = [&](int page) {
        if (page < 0) return;
        const uint8_t *rec = c.record(page, kh, kRec);
        scale = *reinterpret_cast<const float2 *>(rec + 64 * HD);
#pragma unroll
        for (int i = 0; i < NC; ++i) kc[i] = *reinterpret_cast<const u32x4 *>(rec + 1024 * i + 16 * lane);
    };
    auto load_v = [&](int page) {
        if (page < 0) return;
        const uint8_t *rec = c.record(page, kh, kRec);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int odd = 0; odd < 2; ++odd)  // dims 64 i + 4n .. + 3 of positions 4g + odd, + 2, 16 + 4g + odd, + 2
                vc[i][odd] = *reinterpret_cast<const u32x4 *>(rec + kv8_value_byte(4 * g + odd, 64 * i + 4 * (Sums<HD>::half(i) ? n & 7 : n), HD));
    };
    int page = __builtin_amdgcn_readlane(pages, 0);
    load_k(page);
    load_v(page);
    Queries<HD> qs[RT];
    Sums<HD> t[RT];
#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const int pair = min(p0 + k * kTile + n, pairs - 1);
        qs[k].seen = min(w.start + pair / group, w.len - 1);
        qs[k].take(raw[k], q_scale);
        t[k].clear();
    }

    for (int i0 = 0; i0 < mine; ++i0) {  // uniform
        const int block = b0 + kWaves * i0;
        if ((i0 + 1) % 64 == 0) pages = i0 + 1 + lane < mine ? c.page(seq, block + kWaves * (1 + lane)) : -1;
        const int next = i0 + 1 < mine ? __builtin_amdgcn_readlane(pages, (i0 + 1) % 64) : -1;
        if (page >= 0) {
            const float ks = scale.x, vscale = scale.y;
            f32x4 s[RT][2];
#pragma unroll
            for (int k = 0; k < RT; ++k) s[k][0] = s[k][1] = zero;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const u32x4 a0 = f16_of_8(kc[i][0], kc[i][1]), a1 = f16_of_8(kc[i][2], kc[i][3]);
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    s[k][0] = mfma16(a0, qs[k].hi[i], s[k][0]);
                    s[k][1] = mfma16(a1, qs[k].hi[i], s[k][1]);
                }
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    s[k][0] = mfma16(a0, qs[k].lo[i], s[k][0]);
                    s[k][1] = mfma16(a1, qs[k].lo[i], s[k][1]);
                }
            }
            load_k(next);
            const bool edge = block * kKv8Block + kKv8Block - 1 > sp.first;  // uniform
            u32x4 hi[RT], lo[RT];
            float vs[RT];
#pragma unroll
            for (int k = 0; k < RT; ++k) {
                t[k].weigh(s[k], ks * qs[k].inv, edge, block, g, qs[k].seen, hi[k], lo[k]);
                // a scale that is not finite meets only the rows that see one of the block's positions
                vs[k] = edge && block * kKv8Block > qs[k].seen ? 0.0f : vscale;
            }
            auto values = [&](int i, auto jc) {  // two operands, whose chains are independent
                constexpr int J = decltype(jc)::value;
                // positions 4g, 4g + 1; 4g + 2, + 3; 16 + 4g, + 1; 16 + 4g + 2, + 3
                u32x4 a, b;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    a[h] = f16_of_bytes<J>(vc[i][0][h], vc[i][1][h]);
                    b[h] = f16_of_bytes<J + 1>(vc[i][0][h], vc[i][1][h]);
                }
                f32x4 x[RT][2];
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    x[k][0] = mfma16(a, hi[k], zero);
                    x[k][1] = mfma16(b, hi[k], zero);
                }
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    x[k][0] = mfma16(a, lo[k], x[k][0]);
                    x[k][1] = mfma16(b, lo[k], x[k][1]);
                }
#pragma unroll
                for (int k = 0; k < RT; ++k) {
                    t[k].join(i, J, x[k][0], vs[k]);
                    t[k].join(i, J + 1, x[k][1], vs[k]);
                }
            };
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if (Sums<HD>::half(i))
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd) vc[i][odd] >>= 2 * (n & 8);
                values(i, std::integral_constant<int, 0>());
                if (!Sums<HD>::half(i)) values(i, std::integral_constant<int, 2>());
            }
            load_v(next);
        } else {
            load_k(next);
            load_v(next);
        }
        page = next;
    }
    for (int it = max(split * per, sp.blocks); it < end; ++it)
        if ((it - split * per) % kWaves == wave && c.page(seq, sp.done) >= 0)  // uniform
#pragma unroll
            for (int k = 0; k < RT; ++k)
                t[k].tail(qs[k], c.ring(seq, kh, 0, HD), c.ring(seq, kh, 1, HD), sp.done * kKv8Block + 16 * (it - sp.blocks), w.len, sp.first, n, g);

#pragma unroll
    for (int k = 0; k < RT; ++k) {
        const int pk = p0 + k * kTile;
        if (k > 0) __syncthreads();  // (the tile before is read)
        if (g == 0) {
            s_m[wave][n] = -t[k].a;
            s_l[wave][n] = t[k].l;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float *dst = &s_o[wave][n][Sums<HD>::dim_of(i, g, r)];
                if (Sums<HD>::half(i)) *reinterpret_cast<f32x2 *>(dst) = f32x2{t[k].o[i][0][r], t[k].o[i][1][r]};
                else *reinterpret_cast<f32x4 *>(dst) = f32x4{t[k].o[i][0][r], t[k].o[i][1][r], t[k].o[i][2][r], t[k].o[i][3][r]};
            }
        __syncthreads();
        for (int e = threadIdx.x; e < kTile * (HD / 4); e += 64 * kWaves) {
            const int row = e / (HD / 4), d = 4 * (e % (HD / 4));
            if (pk + row >= pairs) continue;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) mx = fmaxf(mx, s_m[i][row]);
            f32x4 num = zero;
            float den = 0.0f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                const float mi = s_m[i][row], li = s_l[i][row];
                const float f = exp2_fast(mi - mx);  // (no position of this row: -FLT_MAX, and sums of 0)
                const f32x4 o = *reinterpret_cast<const f32x4 *>(&s_o[i][row][d]);
#pragma unroll
                for (int r = 0; r < 4; ++r) num[r] = fmaf(o[r], f, num[r]);
                den = fmaf(li, f, den);
            }
            if (used == 1) {
                const int pr = pk + row;
                const float inv = den != 0.0f ? 1.0f / den : 0.0f;  // (no position: num is 0 too)
                f32x4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = num[r] * inv;
                *reinterpret_cast<f32x4 *>(out + ((static_cast<size_t>(seq) * rows + pr / group) * n_heads + kh * group + pr % group) * HD + d) = o;
            } else {
                // [tile of this launch][split][row]: HD sums, the maximum, the denominator
                const size_t tile = (static_cast<size_t>(seq) * (macros * RT) + macro * RT + k) * c.kv + kh;
                float *dst = part + ((tile * splits + split) * kTile + row) * (HD + 4);
                *reinterpret_cast<f32x4 *>(dst + d) = num;
                if (d == 0) *reinterpret_cast<float2 *>(dst + HD) = make_float2(mx, den);
            }
        }
    }
}

// A workgroup per query row: the splits' sums joined (28 rows of 126 splits 4.6 us: the launch and three dependent
// loads).  Each wave finds the splits' weights (a split a lane), and each thread adds four dims of every C-th split, four
// in flight.
constexpr int kJoinThreads = 256;
constexpr int kMaxSplits = 128;
template <int HD>
__global__ __launch_bounds__(kJoinThreads) void attend_kv8_join_kernel(Kv8View c, float *__restrict__ out, int rows,
                                                                       int n_heads, const int *__restrict__ start_pos,
                                                                       const int *__restrict__ n_rows, int tiles,
                                                                       int macro, int splits,
                                                                       const float *__restrict__ part) {
    constexpr int D4 = HD / 4, C = kJoinThreads / D4, kSlots = kMaxSplits / 64;
    __shared__ f32x4 s_num[C][D4];
    __shared__ float s_f[kJoinThreads / 64][kMaxSplits];
    const int row = blockIdx.x % kTile, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned group_id = blockIdx.x / kTile;
    const float *src = part + (static_cast<size_t>(group_id) * splits * kTile + row) * (HD + 4);
    const size_t step = static_cast<size_t>(kTile) * (HD + 4);
    const int cls = threadIdx.x / D4, d4 = threadIdx.x % D4;
    // requested before it is known how many splits there are; what the others hold is not used
    f32x4 first[4];
    float2 ml[kSlots];
#pragma unroll
    for (int k = 0; k < kSlots; ++k)
        ml[k] = lane + 64 * k < splits ? *reinterpret_cast<const float2 *>(src + (lane + 64 * k) * step + HD) : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int u = 0; u < 4; ++u)
        first[u] = cls < C && cls + u * C < splits ? *reinterpret_cast<const f32x4 *>(src + (cls + u * C) * step + 4 * d4) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int id = group_id;
    const int kh = id % c.kv;
    id /= c.kv;
    const int tile = id % tiles, seq = id / tiles;
    const int group = n_heads / c.kv, p0 = tile * kTile;
    const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, c.per * kKv8Block);
    const int pr = p0 + row;
    if (pr >= w.rows * group) return;
    // of the rows that one workgroup took
    const Span sp = span_of(w, p0 / macro * macro, macro, group);
    const int per = items_per_split(sp.items(), splits), used = (sp.items() + per - 1) / per;
    if (used <= 1) return;  // written already
    float mi[kSlots], li[kSlots], mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kSlots; ++k) {
        mi[k] = lane + 64 * k < used ? ml[k].x : -INFINITY;
        li[k] = lane + 64 * k < used ? ml[k].y : 0.0f;
        mx = fmaxf(mx, mi[k]);
    }
    mx = wave_max_dpp(mx);
    float den = 0.0f;
#pragma unroll
    for (int k = 0; k < kSlots; ++k) {
        const float f = exp2_fast(mi[k] - mx);
        s_f[wave][lane + 64 * k] = f;
        den = fmaf(li[k], f, den);
    }
    den = wave_sum(den);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's own row of s_f)
    __builtin_amdgcn_wave_barrier();
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
    if (cls < C) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (cls + u * C < used) {
                const float f = s_f[wave][cls + u * C];
#pragma unroll
                for (int r = 0; r < 4; ++r) num[r] = fmaf(first[u][r], f, num[r]);
            }
        for (int i0 = cls + 4 * C; i0 < used; i0 += 4 * C) {
            f32x4 o[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                o[u] = i0 + u * C < used ? *reinterpret_cast<const f32x4 *>(src + (i0 + u * C) * step + 4 * d4) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float f = i0 + u * C < used ? s_f[wave][i0 + u * C] : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) num[r] = fmaf(o[u][r], f, num[r]);
            }
        }
        s_num[cls][d4] = num;
    }
    __syncthreads();
    if (threadIdx.x < D4) {
        f32x4 o = s_num[0][d4];
#pragma unroll
        for (int i = 1; i < C; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] += s_num[i][d4][r];
        const float inv = den != 0.0f ? 1.0f / den : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] *= inv;
        *reinterpret_cast<f32x4 *>(out + ((static_cast<size_t>(seq) * rows + pr / group) * n_heads + kh * group + pr % group) * HD + 4 * d4) = o;
    }
}

// The same for at most kFewSplits splits, a wave per query row: a workgroup each would find little to do (8000 rows of
// two splits 17 us, so 6; 112 rows of 8 splits with their attention 18.1, so 17.3; but of 16 splits 10.8, so 11.3).
constexpr int kFewSplits = 8;
template <int HD>
__global__ __launch_bounds__(kJoinThreads) void attend_kv8_join_rows_kernel(Kv8View c, float *__restrict__ out, int rows,
                                                                            int n_heads, const int *__restrict__ start_pos,
                                                                            const int *__restrict__ n_rows, int tiles,
                                                                            int macro, int splits,
                                                                            const float *__restrict__ part) {
    constexpr int D4 = HD / 4, C = 64 / D4, kSlots = kFewSplits / C;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (blockIdx.x * 4 + wave) % kTile;
    const unsigned group_id = blockIdx.x / (kTile / 4);
    const float *src = part + (static_cast<size_t>(group_id) * splits * kTile + row) * (HD + 4);
    const size_t step = static_cast<size_t>(kTile) * (HD + 4);
    const int cls = lane / D4, d4 = lane % D4;
    // requested before it is known how many splits there are; what the others hold is not used
    const float2 ml = lane < splits ? *reinterpret_cast<const float2 *>(src + lane * step + HD) : make_float2(-INFINITY, 0.0f);
    f32x4 o[kSlots];
#pragma unroll
    for (int u = 0; u < kSlots; ++u)
        o[u] = cls < C && cls + u * C < splits ? *reinterpret_cast<const f32x4 *>(src + (cls + u * C) * step + 4 * d4) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int id = group_id;
    const int kh = id % c.kv;
    id /= c.kv;
    const int tile = id % tiles, seq = id / tiles;
    const int group = n_heads / c.kv, p0 = tile * kTile;
    const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, c.per * kKv8Block);
    const int pr = p0 + row;
    if (pr >= w.rows * group) return;
    const Span sp = span_of(w, p0 / macro * macro, macro, group);
    const int per = items_per_split(sp.items(), splits), used = (sp.items() + per - 1) / per;
    if (used <= 1) return;  // written already
    const float mi = lane < used ? ml.x : -INFINITY, li = lane < used ? ml.y : 0.0f;
    const float mx = wave_max_dpp(mi);
    const float f = exp2_fast(mi - mx);
    const float den = wave_sum(li * f);
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
        const float fu = __shfl(f, cls + u * C, 64);
        if (cls + u * C < used)
#pragma unroll
            for (int r = 0; r < 4; ++r) num[r] = fmaf(o[u][r], fu, num[r]);
    }
#pragma unroll
    for (int k = 1; k < C; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = __shfl(num[r], (lane + k * D4) & 63, 64);
            if (cls == 0) num[r] += v;
        }
    if (lane < D4) {
        const float inv = den != 0.0f ? 1.0f / den : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) num[r] *= inv;
        *reinterpret_cast<f32x4 *>(out + ((static_cast<size_t>(seq) * rows + pr / group) * n_heads + kh * group + pr % group) * HD + 4 * d4) = num;
    }
}

struct Plan {
    int rt, waves;                     // tiles of a wave, waves of a workgroup
    int64_t macros, tiles, groups;     // workgroups and tiles of a (sequence, key head), tiles of the launch
    int64_t work;                      // workgroups of a split
    int splits;
    size_t bytes;                      // of workspace
};
Plan plan_of(int n_seqs, int rows, int n_heads, int kv, int head_dim, int blocks) {
    Plan p;
    const int64_t pairs = static_cast<int64_t>(rows) * (n_heads / kv);
    p.rt = pairs > kTile && head_dim <= 128 ? 2 : 1;  // (at 192 two tiles' sums and queries do not fit a wave's registers)
    p.macros = (pairs + p.rt * kTile - 1) / (p.rt * kTile);
    p.tiles = p.macros * p.rt;
    p.work = p.macros * kv * n_seqs;
    p.groups = p.work * p.rt;
    // Splits fill CUs that are idle, or that a longer sequence's workgroup keeps waiting for, and cost a join.  They pay where
    // that waiting is long, in caches of more than 64 blocks, unless a single sequence's workgroups, all alike, fill 7/8 of
    // the chip by themselves.  (Where they do not pay: 512 rows of 28 heads of 128 in 448 workgroups behind 2500 positions 62 us,
    // in halves 75; 48 sequences of up to 1000 positions and 8 key heads 20, so 29.  Where they do: these sequences of up to
    // 12000 129, so 157; 320 rows in 280 behind 8000 125, so 145.)
    const bool few = blocks <= 64;
    auto fill = [&](int64_t slots) { return n_seqs == 1 && 8 * p.work >= 7 * slots; };
    // Not split: 8 waves, a workgroup a CU, from a half (three quarters for single tiles) to one workgroup a CU.  384 rows of
    // 14 heads of 64 in 168 workgroups 9.2 us, in splits of 4 waves 13.5; 250 rows behind 6000 positions, 32 heads of 128, in
    // 256 65, so 72; 60 sequences of up to 1000 and 4 key heads 17, so 24.  With fewer workgroups CUs have no work: 56 of 128 rows
    // 10.5, so 9.5; in longer caches 24 sequences of 5 rows and up to 8000 84, so 60.
    p.waves = 4 * p.work > (p.rt == 2 ? 2 : 3) * kCus && p.work <= kCus && (few || fill(kCus)) ? 8 : 4;
    const bool one = p.waves == 8 || p.work > 2 * kCus || (p.work > kCus && (few || fill(2 * kCus)));
    // Otherwise two workgroups for every CU, but no split of less than kMinItems blocks of the longest sequence.
    const int64_t want = p.work > 0 && !one ? (2 * kCus + p.work - 1) / p.work : 1;
    const int64_t most = (blocks + kMinItems) / kMinItems;
    p.splits = static_cast<int>(want < most ? want : most);
    if (p.splits > kMaxSplits) p.splits = kMaxSplits;
    p.bytes = p.splits > 1 ? static_cast<size_t>(p.groups) * p.splits * kTile * (static_cast<size_t>(head_dim) + 4) * sizeof(float) : 0;
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
    const qlin::Plan p = qlin::plan_of(n_seqs, rows, n_heads, kv_heads, head_dim, blocks_per_seq);
    return p.bytes;
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
    const qlin::Plan p = qlin::plan_of(cache->n_seqs, rows, n_heads, kv, hd, cache->blocks_per_seq);
    const int64_t grid = p.work * p.splits;
    if (grid > (1 << 23) || (p.splits > 1 && p.groups * qlin::kTile > (1 << 23))) return QLIN_ERR_LIMIT;
    const size_t need = qlin_attend_kv8_workspace_bytes(cache->n_seqs, rows, n_heads, kv, hd, cache->blocks_per_seq);
    if (need > 0 && !workspace) return QLIN_ERR_NULL;
    if (workspace_bytes < need) return QLIN_ERR_LIMIT;
    const float q_scale = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
    float *part = static_cast<float *>(workspace);
    const qlin::Kv8View view = qlin::kv8_view(cache);
    auto go = [&](auto attend, auto join, auto join_rows) {
        hipLaunchKernelGGL(attend, dim3(static_cast<unsigned>(grid)), dim3(64 * p.waves), 0, qlin::current_stream(), view, q,
                           attn, rows, n_heads, start_pos_dev, n_rows_dev, q_scale, static_cast<int>(p.macros),
                           p.splits, part);
        if (hipGetLastError() != hipSuccess) return QLIN_ERR_LAUNCH;
        if (p.splits > 1) {
            const bool few = p.splits <= qlin::kFewSplits;
            hipLaunchKernelGGL(few ? join_rows : join, dim3(static_cast<unsigned>(p.groups * qlin::kTile / (few ? 4 : 1))),
                               dim3(qlin::kJoinThreads), 0, qlin::current_stream(), view, attn, rows, n_heads, start_pos_dev, n_rows_dev,
                               static_cast<int>(p.tiles), p.rt * qlin::kTile, p.splits, part);
            if (hipGetLastError() != hipSuccess) return QLIN_ERR_LAUNCH;
        }
        return QLIN_OK;
    };
#define QLIN_GO(HD, RT)                                                                                          \
    return go(p.rt == 1 ? p.waves == 4 ? qlin::attend_kv8_kernel<HD, 1, 4> : qlin::attend_kv8_kernel<HD, 1, 8>   \
              : p.waves == 4 ? qlin::attend_kv8_kernel<HD, RT, 4> : qlin::attend_kv8_kernel<HD, RT, 8>,          \
              qlin::attend_kv8_join_kernel<HD>, qlin::attend_kv8_join_rows_kernel<HD>)
    switch (hd) {
        case 64: QLIN_GO(64, 2);
        case 96: QLIN_GO(96, 2);
        case 128: QLIN_GO(128, 2);
        case 192: QLIN_GO(192, 1);
        default: QLIN_GO(256, 1);
    }
#undef QLIN_GO
}

}  // extern "C"
