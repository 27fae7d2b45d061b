// qlin_kv8.hip -- norms of query and key heads with the rotation in the same pass, the store into an f32 cache or
// into the 8-bit cache of blocks (qlin_kv8.hpp), and the read back from the latter, gfx950.
//
// Mathematics (qlin_decoder.h): x' = x (mean x^2 + eps)^(-1/2) w over a head, its first rotary_dim values turned by
// the position's cosines and sines; a complete block of 32 positions as codes rint(x 127 / amax) with one scale.
//
// A head is taken by the lanes t = 0 .. T - 1 of a group (T the power of two from head_dim / 8), 8 values a lane: of
// the turned values 4t .. 4t + 3 and the same of the upper half, so that both pairings turn inside the lane; of the
// rest 8 consecutive ones.  The sum of squares, the root and the turn are in f64: a key next to a border between two
// codes then rounds to the same f32 value, and so gets the same code, whatever the order of the sum (f32 would move
// one code in about 10^5), and on this chip an f64 operation takes an f32 one's time.  Loads are 16 bytes at 4-byte
// alignment, so heads may be any part of a wider row.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_kv8.hpp"

namespace qlin {
namespace {

typedef float f32x4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4v ld4(const float *p) {
    f32x4v v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, 4), 16);
    return v;
}
// Streaming stores: what lies dirty in the L2s at the kernel's end is written back then (a 2011-row prompt's store and
// read back 26.0 us, so 22.2; 1877 rows into the f32 cache 18.3 and 16.5, in graphs).
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void st4(float *p, const f32x4v &v) { __builtin_nontemporal_store(v, reinterpret_cast<f32x4u *>(p)); }

template <int CTRL>
__device__ __forceinline__ double dpp_move64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// The sum over each group of T lanes (T <= 32), in every lane of it.
template <int T>
__device__ __forceinline__ double group_sum(double v) {
    if constexpr (T > 1) v += dpp_move64<0xb1>(v);   // quad_perm [1, 0, 3, 2]
    if constexpr (T > 2) v += dpp_move64<0x4e>(v);   // quad_perm [2, 3, 0, 1]
    if constexpr (T > 4) v += dpp_move64<0x141>(v);  // row_half_mirror
    if constexpr (T > 8) v += dpp_move64<0x140>(v);  // row_mirror
    if constexpr (T > 16) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t l = static_cast<uint32_t>(u), h = static_cast<uint32_t>(u >> 32);
        const auto sl = __builtin_amdgcn_permlane16_swap(l, l, false, false);  // rows 0, 0, 2, 2 and 1, 1, 3, 3
        const auto sh = __builtin_amdgcn_permlane16_swap(h, h, false, false);
        v = __builtin_bit_cast(double, (static_cast<uint64_t>(static_cast<uint32_t>(sh[0])) << 32) | static_cast<uint32_t>(sl[0])) +
            __builtin_bit_cast(double, (static_cast<uint64_t>(static_cast<uint32_t>(sh[1])) << 32) | static_cast<uint32_t>(sl[1]));
    }
    return v;
}

// Where the two runs of 4 values of lane t begin in a head.
struct Runs {
    int a, b;
    bool turned;
    __device__ __forceinline__ Runs(int t, int rd) {
        const int n = rd / 8;
        turned = t < n;
        a = turned ? 4 * t : rd + 8 * (t - n);
        b = turned ? rd / 2 + 4 * t : a + 4;
    }
};

// The 4 weights from w + j (j a multiple of 4) as 16-bit patterns: one load where w is 8-byte aligned (four loads of 2
// bytes for each run of each head kept a prompt's kernel at 28 us where the bytes take 14).
__device__ __forceinline__ uint2 weights_at(const uint16_t *w, int j) {
    if ((reinterpret_cast<uintptr_t>(w) & 7u) == 0) return *reinterpret_cast<const uint2 *>(w + j);  // uniform
    return make_uint2(w[j] | static_cast<uint32_t>(w[j + 1]) << 16, w[j + 2] | static_cast<uint32_t>(w[j + 3]) << 16);
}
__device__ __forceinline__ double weight_of(uint2 w, int e, int type, int one_plus) {
    const uint32_t u = (e < 2 ? w.x : w.y) >> (16 * (e & 1)) & 0xffffu;
    const float v = type == 0 ? __builtin_bit_cast(float, u << 16)
                              : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u)));
    return one_plus ? static_cast<double>(v) + 1.0 : static_cast<double>(v);
}

// One head's norm (w NULL: none) and turn by the table's row of pos (clamped to 0 .. cap - 1), in place; every lane of the
// group calls it, those past the head's end (live false) with zeros.
template <int T>
__device__ __forceinline__ void norm_and_turn(f32x4v &va, f32x4v &vb, const Runs &r, bool live, int hd, const uint16_t *w,
                                              const qlin_qk_rope &how, int pos, int cap) {
    double a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = va[e];
        b[e] = vb[e];
    }
    // (requested before the sum needs them)
    const bool normed = w != nullptr;
    uint2 wa = make_uint2(0u, 0u), wb = make_uint2(0u, 0u);
    if (normed && live) {
        wa = weights_at(w, r.a);
        wb = weights_at(w, r.b);
    }
    const int half = how.rotary_dim / 2, at = min(max(pos, 0), cap - 1);
    f32x4v c0, s0;  // halves: the pairs' cosines and sines; neighbours: (cos, cos, sin, sin) of run a's and b's pairs
    if (r.turned) {
        const float *row = how.table + static_cast<size_t>(min(at, how.table_len - 1)) * how.rotary_dim;
        if (how.pairing == 0) {
            c0 = ld4(row + r.a);
            s0 = ld4(row + half + r.a);
        } else {
            c0 = f32x4v{row[r.a / 2], row[r.a / 2 + 1], row[r.b / 2], row[r.b / 2 + 1]};
            s0 = f32x4v{row[half + r.a / 2], row[half + r.a / 2 + 1], row[half + r.b / 2], row[half + r.b / 2 + 1]};
        }
    }
    if (normed) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) ss += a[e] * a[e] + b[e] * b[e];
        const double inv = 1.0 / sqrt(group_sum<T>(ss) / hd + static_cast<double>(how.eps));
        if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = a[e] * inv * weight_of(wa, e, how.norm_type, how.one_plus);
                b[e] = b[e] * inv * weight_of(wb, e, how.norm_type, how.one_plus);
            }
        }
    }
    if (r.turned) {
        if (at >= how.table_len) c0 = f32x4v{NAN, NAN, NAN, NAN};  // (another position's angles would go unseen)
        if (how.pairing == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double c = c0[e], s = s0[e], x = a[e], y = b[e];
                a[e] = x * c - y * s;
                b[e] = y * c + x * s;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                double c = c0[e / 2], s = s0[e / 2], x = a[e], y = a[e + 1];
                a[e] = x * c - y * s;
                a[e + 1] = y * c + x * s;
                c = c0[2 + e / 2], s = s0[2 + e / 2], x = b[e], y = b[e + 1];
                b[e] = x * c - y * s;
                b[e + 1] = y * c + x * s;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        va[e] = static_cast<float>(a[e]);
        vb[e] = static_cast<float>(b[e]);
    }
}

constexpr int kThreads = 256;
constexpr f32x4v kZero4 = {0.0f, 0.0f, 0.0f, 0.0f};

// A group of lanes for each query, key and value head of each row.  Bound by bytes: 1877 rows of 28 + 4 + 4 heads of 128
// 14.1 to 15.8 us in a kernel trace, 4.4 to 5.0 TB/s; one row 2.6 us, the launch.
template <int T>
__global__ __launch_bounds__(kThreads) void norm_rope_store_kernel(qlin_qk_rope how, const float *q, size_t q_stride,
                                                                   const float *__restrict__ k, size_t k_stride,
                                                                   const float *__restrict__ v, size_t v_stride,
                                                                   float *q_out, float *__restrict__ kc,
                                                                   float *__restrict__ vc, int rows, int n_heads, int kv,
                                                                   int hd, int max_seq, const int *__restrict__ start_pos) {
    const int t = threadIdx.x % T, heads = n_heads + 2 * kv;
    const unsigned unit = blockIdx.x * (kThreads / T) + threadIdx.x / T;  // (the launch has fewer than 2^31)
    const unsigned line = unit / static_cast<unsigned>(heads);
    const bool there = line < static_cast<unsigned>(rows);
    const int row = there ? static_cast<int>(line) : 0, head = there ? static_cast<int>(unit - line * heads) : 0;
    const int64_t at = static_cast<int64_t>(*start_pos) + row;
    const int pos = static_cast<int>(at < 0 ? 0 : at < max_seq ? at : max_seq - 1);
    const Runs r(t, how.rotary_dim);
    const bool live = there && 8 * t < hd;
    const bool is_q = head < n_heads, is_k = !is_q && head < n_heads + kv;
    const float *src = is_q ? q + static_cast<size_t>(row) * q_stride + static_cast<size_t>(head) * hd
                       : is_k ? k + static_cast<size_t>(row) * k_stride + static_cast<size_t>(head - n_heads) * hd
                              : v + static_cast<size_t>(row) * v_stride + static_cast<size_t>(head - n_heads - kv) * hd;
    float *dst = is_q ? q_out + (static_cast<size_t>(row) * n_heads + head) * hd
                 : is_k ? kc + (static_cast<size_t>(pos) * kv + (head - n_heads)) * hd
                        : vc + (static_cast<size_t>(pos) * kv + (head - n_heads - kv)) * hd;
    f32x4v a = live ? ld4(src + r.a) : kZero4, b = live ? ld4(src + r.b) : kZero4;
    f32x4v x = a, y = b;
    Runs rr = r;
    rr.turned = rr.turned && live && (is_q || is_k);
    norm_and_turn<T>(x, y, rr, live, hd, is_q ? how.q_norm : how.k_norm, how, pos, max_seq);
    if (live) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (by value: a choice between vectors goes through memory)
            a[e] = is_q || is_k ? x[e] : a[e];
            b[e] = is_q || is_k ? y[e] : b[e];
        }
        st4(dst + r.a, a);
        st4(dst + r.b, b);
    }
}

template <int HD>
constexpr int lanes_of() {
    return HD <= 64 ? 8 : HD <= 128 ? 16 : 32;
}

// The largest over the workgroup (kThreads), of the bits of two magnitudes: NaN is above infinity, which is above the
// rest.  A barrier lies between two calls' uses of red.
__device__ __forceinline__ uint2 block_max_bits(uint2 v, uint2 *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        v.x = max(v.x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v.x), o, 64)));
        v.y = max(v.y, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v.y), o, 64)));
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) v = make_uint2(max(v.x, red[w].x), max(v.y, red[w].y));
    return v;
}

__device__ __forceinline__ int code_of(float x, float scale) {
    return static_cast<int>(fminf(fmaxf(rintf(x / scale), -127.0f), 127.0f));
}

// Workgroups [0, n_seqs * kv * slots): one per (sequence, key head, block that the rows touch); the rest: the queries'
// heads.  A block's workgroup holds its 32 rows of keys and values in registers, takes the rows that came earlier from
// the ring, writes the new rows of the last two blocks there, and, if the block is complete, its codes (through LDS,
// in the record's order) and scales.
//
// Bound by the queries' bytes (2011 rows of 28 + 4 + 4 heads of 128 14.3 us in a kernel trace, 4.7 TB/s), for few rows by a block's chain: table
// row and norm, largest value, codes through LDS (24 sequences of one row 6.0 us).
//
// The first block's workgroup reads ring rows; the block two (or 2i) further that would overwrite them is its second
// job, after that read, so that no other workgroup writes what it reads.
template <int HD>
__global__ __launch_bounds__(kThreads) void norm_rope_store_kv8_kernel(qlin_qk_rope how, Kv8View c, const float *q,
                                                                       size_t q_stride, const float *__restrict__ k,
                                                                       size_t k_stride, const float *__restrict__ v,
                                                                       size_t v_stride, float *q_out, int rows,
                                                                       int n_heads, int n_seqs, int slots,
                                                                       const int *__restrict__ start_pos,
                                                                       const int *__restrict__ n_rows) {
    constexpr int T = lanes_of<HD>(), kTok = kThreads / T, kPass = kKv8Block / kTok;
    const int t = threadIdx.x % T;
    const unsigned kv_groups = static_cast<unsigned>(n_seqs) * c.kv * slots;
    const int cap = c.per * kKv8Block;
    const Runs r(t, how.rotary_dim);
    const bool in_head = 8 * t < HD;
    if (blockIdx.x >= kv_groups) {
        const unsigned unit = (blockIdx.x - kv_groups) * kTok + threadIdx.x / T;  // (the launch has fewer than 2^31)
        const unsigned at = unit / static_cast<unsigned>(n_heads);
        const bool there = at < static_cast<unsigned>(n_seqs) * static_cast<unsigned>(rows);
        const unsigned line = there ? at : 0;
        const int head = there ? static_cast<int>(unit - at * n_heads) : 0;
        const int seq = static_cast<int>(line / static_cast<unsigned>(rows)), row = static_cast<int>(line - seq * static_cast<unsigned>(rows));
        const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, cap);
        const bool live = there && in_head && row < w.rows;
        const float *src = q + static_cast<size_t>(line) * q_stride + static_cast<size_t>(head) * HD;
        f32x4v a = live ? ld4(src + r.a) : kZero4, b = live ? ld4(src + r.b) : kZero4;
        Runs rr = r;
        rr.turned = rr.turned && live;
        norm_and_turn<T>(a, b, rr, live, HD, how.q_norm, how, w.start + row, cap);
        if (live) {
            float *dst = q_out + (static_cast<size_t>(line) * n_heads + head) * HD;
            st4(dst + r.a, a);
            st4(dst + r.b, b);
        }
        return;
    }
    __shared__ __attribute__((aligned(16))) uint8_t s_rec[64 * HD];
    __shared__ uint2 red[kThreads / 64];
    const int slot = static_cast<int>(blockIdx.x % slots);
    const int head = static_cast<int>(blockIdx.x / slots % c.kv), seq = static_cast<int>(blockIdx.x / slots / c.kv);
    const Kv8Rows w = kv8_rows(start_pos, n_rows, seq, rows, cap);
    const int begin = max(w.start, 0);
    if (w.len <= begin || w.rows == 0) return;  // uniform: nothing is stored
    const int b0 = begin / kKv8Block, lb = (w.len - 1) / kKv8Block;
    // the block whose new ring rows take the place of the first block's old ones
    const int over = begin % kKv8Block != 0 && lb - b0 >= 2 ? lb - ((lb - b0) & 1) : -1;
    float *ring_k = c.ring(seq, head, 0, HD), *ring_v = c.ring(seq, head, 1, HD);

    auto block = [&](int b) {
        const bool complete = (b + 1) * kKv8Block <= w.len;
        const int page = c.page(seq, b);
        f32x4v ka[kPass], kb[kPass], va[kPass], vb[kPass];
#pragma unroll
        for (int p = 0; p < kPass; ++p) {
            const int pos = b * kKv8Block + p * kTok + threadIdx.x / T;
            const bool fresh = in_head && pos >= begin && pos < w.len;
            const bool old = in_head && pos < begin && complete;
            const size_t line = static_cast<size_t>(seq) * rows + (fresh ? pos - w.start : 0);
            const float *ks = fresh ? k + line * k_stride + static_cast<size_t>(head) * HD
                                    : ring_k + static_cast<size_t>(pos % kKv8Recent) * HD;
            const float *vs = fresh ? v + line * v_stride + static_cast<size_t>(head) * HD
                                    : ring_v + static_cast<size_t>(pos % kKv8Recent) * HD;
            const bool any = fresh || old;
            ka[p] = any ? ld4(ks + r.a) : kZero4;
            kb[p] = any ? ld4(ks + r.b) : kZero4;
            va[p] = any ? ld4(vs + r.a) : kZero4;
            vb[p] = any ? ld4(vs + r.b) : kZero4;
        }
        uint32_t k_top = 0, v_top = 0;
#pragma unroll
        for (int p = 0; p < kPass; ++p) {
            const int pos = b * kKv8Block + p * kTok + threadIdx.x / T;
            const bool fresh = in_head && pos >= begin && pos < w.len;
            f32x4v a = ka[p], bb = kb[p];
            Runs rr = r;
            rr.turned = rr.turned && fresh;
            norm_and_turn<T>(a, bb, rr, fresh, HD, how.k_norm, how, pos, cap);
            if (fresh) {
                ka[p] = a;
                kb[p] = bb;
                if (b >= lb - 1) {
                    const size_t at = static_cast<size_t>(pos % kKv8Recent) * HD;
                    st4(ring_k + at + r.a, a);
                    st4(ring_k + at + r.b, bb);
                    st4(ring_v + at + r.a, va[p]);
                    st4(ring_v + at + r.b, vb[p]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (__float_as_uint takes a value: a bit cast of a vector's element reads element 0)
                k_top = max(max(k_top, __float_as_uint(ka[p][e]) & 0x7fffffffu), __float_as_uint(kb[p][e]) & 0x7fffffffu);
                v_top = max(max(v_top, __float_as_uint(va[p][e]) & 0x7fffffffu), __float_as_uint(vb[p][e]) & 0x7fffffffu);
            }
        }
        if (!complete || page < 0) return;  // uniform
        const uint2 top = block_max_bits(make_uint2(k_top, v_top), red);
        k_top = top.x;
        v_top = top.y;
        const bool k_fin = k_top < 0x7f800000u, v_fin = v_top < 0x7f800000u;
        const float k_scale = k_fin ? __builtin_bit_cast(float, k_top) * (1.0f / 127.0f) : NAN;
        const float v_scale = v_fin ? __builtin_bit_cast(float, v_top) * (1.0f / 127.0f) : NAN;
#pragma unroll
        for (int p = 0; p < kPass; ++p) {
            if (!in_head) break;
            const int tok = p * kTok + threadIdx.x / T;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d0 = h == 0 ? r.a : r.b;
                const f32x4v &kx = h == 0 ? ka[p] : kb[p], &vx = h == 0 ? va[p] : vb[p];
                uint32_t kw = 0, vw = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int kq = k_fin && k_scale > 0.0f ? code_of(kx[e], k_scale) : 0;
                    const int vq = v_fin && v_scale > 0.0f ? code_of(vx[e], v_scale) : 0;
                    kw |= (static_cast<uint32_t>(kq) & 0xffu) << (8 * e);
                    vw |= (static_cast<uint32_t>(vq) & 0xffu) << (8 * e);
                }
                *reinterpret_cast<uint32_t *>(s_rec + kv8_key_byte(tok, d0)) = kw;
                *reinterpret_cast<uint32_t *>(s_rec + kv8_value_byte(tok, d0, HD)) = vw;
            }
        }
        __syncthreads();
        uint8_t *rec = c.record(page, head, kv8_record_bytes(HD));
        for (int i = threadIdx.x; i < 4 * HD; i += kThreads)
            reinterpret_cast<uint4 *>(rec)[i] = reinterpret_cast<const uint4 *>(s_rec)[i];
        if (threadIdx.x == 0) *reinterpret_cast<float2 *>(rec + 64 * HD) = make_float2(k_scale, v_scale);
        __syncthreads();  // (s_rec is free again)
    };
    if (b0 + slot > lb || (slot > 0 && b0 + slot == over)) return;  // uniform
    block(b0 + slot);
    if (slot == 0 && over >= 0) {
        __syncthreads();  // the old ring rows are read
        block(over);
    }
}

// A workgroup per (sequence, key head, 32 rows): a thread per 4 dims of a row.  Its rows lie in two blocks at most, whose
// pages are requested first.  Bound by the chain page, code, store: 2011 rows of 4 heads of 128 5.6 us, 24 blocks 3.9.
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(Kv8View c, int hd, const int *__restrict__ first,
                                                            const int *__restrict__ lens, int count, int parts,
                                                            float *__restrict__ k_out, float *__restrict__ v_out) {
    const int part = static_cast<int>(blockIdx.x % parts);
    const int head = static_cast<int>(blockIdx.x / parts % c.kv), seq = static_cast<int>(blockIdx.x / parts / c.kv);
    const int len = min(max(lens[seq], 0), c.per * kKv8Block);
    const int64_t from = static_cast<int64_t>(first[seq]) + part * 32;
    if (from >= len || from + 31 < 0) return;  // uniform
    const int n4 = hd / 4, b0 = from < 0 ? 0 : static_cast<int>(from / kKv8Block);
    const int page0 = c.page(seq, b0), page1 = (b0 + 1) * kKv8Block < len ? c.page(seq, b0 + 1) : -1;
#pragma unroll 4
    for (int i = threadIdx.x; i < 32 * n4; i += kThreads) {
        const int row = part * 32 + i / n4, d = 4 * (i % n4);
        const int64_t at = from + i / n4;
        if (row >= count || at < 0 || at >= len) continue;
        const int pos = static_cast<int>(at), b = pos / kKv8Block, tok = pos % kKv8Block;
        const int page = b == b0 ? page0 : page1;
        if (page < 0) continue;
        f32x4v kx, vx;
        if ((b + 1) * kKv8Block <= len) {
            const uint8_t *rec = c.record(page, head, kv8_record_bytes(hd));
            const float2 s = *reinterpret_cast<const float2 *>(rec + 64 * hd);
            const uint32_t kw = *reinterpret_cast<const uint32_t *>(rec + kv8_key_byte(tok, d));
            const uint32_t vw = *reinterpret_cast<const uint32_t *>(rec + kv8_value_byte(tok, d, hd));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kx[e] = static_cast<float>(static_cast<int8_t>(kw >> (8 * e))) * s.x;
                vx[e] = static_cast<float>(static_cast<int8_t>(vw >> (8 * e))) * s.y;
            }
        } else {
            const size_t o = static_cast<size_t>(pos % kKv8Recent) * hd + d;
            kx = ld4(c.ring(seq, head, 0, hd) + o);
            vx = ld4(c.ring(seq, head, 1, hd) + o);
        }
        const size_t o = ((static_cast<size_t>(seq) * count + row) * c.kv + head) * hd + d;
        st4(k_out + o, kx);
        st4(v_out + o, vx);
    }
}

__global__ __launch_bounds__(kThreads) void rope_table_kernel(float *__restrict__ table, int n_pos, int rd, double log2_theta) {
    const int half = rd / 2;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (at >= static_cast<int64_t>(n_pos) * half) return;
    const int64_t p = at / half;
    const int i = static_cast<int>(at % half);
    double s, c;
    sincos(static_cast<double>(p) * exp2(-log2_theta * (2.0 * i) / rd), &s, &c);
    table[p * rd + i] = static_cast<float>(c);
    table[p * rd + half + i] = static_cast<float>(s);
}

hipStream_t current_stream() { return static_cast<hipStream_t>(qlin_get_stream()); }
int launched(hipError_t e) { return e == hipSuccess ? QLIN_OK : QLIN_ERR_LAUNCH; }
bool aligned_to(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// The checks of a rotation (head_dim already checked).
int check_how(const qlin_qk_rope *how, int head_dim) {
    if (!how) return QLIN_ERR_NULL;
    if (how->norm_type != 0 && how->norm_type != 1) return QLIN_ERR_SHAPE;
    if (how->rotary_dim < 0 || how->rotary_dim > head_dim || how->rotary_dim % 8 || (how->pairing != 0 && how->pairing != 1))
        return QLIN_ERR_SHAPE;
    if (how->rotary_dim > 0 && how->table_len <= 0) return QLIN_ERR_SHAPE;
    if (how->rotary_dim > 0 && !how->table) return QLIN_ERR_NULL;
    if (!aligned_to(how->q_norm, 2) || !aligned_to(how->k_norm, 2) || !aligned_to(how->table, 4)) return QLIN_ERR_ALIGN;
    return QLIN_OK;
}

}  // namespace

int check_kv8(const qlin_kv8_cache *c) {
    if (!c) return QLIN_ERR_NULL;
    if (c->n_seqs < 0 || c->kv_heads <= 0 || c->blocks_per_seq <= 0 || c->n_pages <= 0 || c->head_dim <= 0) return QLIN_ERR_SHAPE;
    const int d = c->head_dim;
    if ((d != 64 && d != 96 && d != 128 && d != 192 && d != 256) || c->blocks_per_seq > 32768 || c->kv_heads > 65536)
        return QLIN_ERR_LIMIT;
    if (!c->block_table && static_cast<int64_t>(c->n_seqs) * c->blocks_per_seq > c->n_pages) return QLIN_ERR_SHAPE;
    if (!c->pages || !c->recent) return QLIN_ERR_NULL;
    if (!aligned_to(c->pages, 16) || !aligned_to(c->recent, 16) || !aligned_to(c->block_table, 4)) return QLIN_ERR_ALIGN;
    return QLIN_OK;
}
Kv8View kv8_view(const qlin_kv8_cache *c) {
    return Kv8View{c->pages, c->recent, c->block_table, c->n_pages, c->blocks_per_seq, c->kv_heads};
}

}  // namespace qlin

extern "C" {

int qlin_launch_rope_table(float *table, int n_pos, int rotary_dim, float theta) {
    if (n_pos < 0 || rotary_dim < 0 || rotary_dim % 2 || !(theta > 0.0f) || isinf(theta)) return QLIN_ERR_SHAPE;
    if (n_pos > 1 << 20 || rotary_dim > 256) return QLIN_ERR_LIMIT;
    if (n_pos == 0 || rotary_dim == 0) return QLIN_OK;
    if (!table) return QLIN_ERR_NULL;
    if (!qlin::aligned_to(table, 4)) return QLIN_ERR_ALIGN;
    const int64_t n = static_cast<int64_t>(n_pos) * (rotary_dim / 2);
    hipLaunchKernelGGL(qlin::rope_table_kernel, dim3(static_cast<unsigned>((n + qlin::kThreads - 1) / qlin::kThreads)),
                       dim3(qlin::kThreads), 0, qlin::current_stream(), table, n_pos, rotary_dim,
                       log2(static_cast<double>(theta)));
    return qlin::launched(hipGetLastError());
}

int qlin_launch_qk_norm_rope_store_kv(const qlin_qk_rope *how, const float *q, size_t q_stride, const float *k,
                                      size_t k_stride, const float *v, size_t v_stride, float *q_out, float *key_cache,
                                      float *value_cache, int rows, int n_heads, int kv_heads, int head_dim,
                                      int max_seq_len, const int *start_pos_dev) {
    if (rows < 0 || n_heads <= 0 || kv_heads <= 0 || n_heads % kv_heads || head_dim <= 0 || head_dim % 8 || max_seq_len <= 0)
        return QLIN_ERR_SHAPE;
    if (head_dim > 256 || max_seq_len > 1 << 20 || rows > 1 << 20 || n_heads > 65536) return QLIN_ERR_LIMIT;
    if (int rc = qlin::check_how(how, head_dim)) return rc;
    const size_t qw = static_cast<size_t>(n_heads) * head_dim, kw = static_cast<size_t>(kv_heads) * head_dim;
    if (q_stride < qw || k_stride < kw || v_stride < kw || (q == q_out && q_stride != qw)) return QLIN_ERR_SHAPE;
    if (rows == 0) return QLIN_OK;
    if (!q || !k || !v || !q_out || !key_cache || !value_cache || !start_pos_dev) return QLIN_ERR_NULL;
    for (const void *p : {static_cast<const void *>(q), static_cast<const void *>(k), static_cast<const void *>(v),
                          static_cast<const void *>(q_out), static_cast<const void *>(key_cache),
                          static_cast<const void *>(value_cache), static_cast<const void *>(start_pos_dev)})
        if (!qlin::aligned_to(p, 4)) return QLIN_ERR_ALIGN;
    int lanes = 1;
    while (8 * lanes < head_dim) lanes *= 2;
    const int64_t groups = qlin::kThreads / lanes;
    const int64_t grid = (static_cast<int64_t>(rows) * (n_heads + 2 * kv_heads) + groups - 1) / groups;
    if (grid > (1 << 23)) return QLIN_ERR_LIMIT;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(qlin::kThreads), 0, qlin::current_stream(), *how,
                           q, q_stride, k, k_stride, v, v_stride, q_out, key_cache, value_cache, rows, n_heads, kv_heads,
                           head_dim, max_seq_len, start_pos_dev);
        return qlin::launched(hipGetLastError());
    };
    switch (lanes) {
        case 1: return go(qlin::norm_rope_store_kernel<1>);
        case 2: return go(qlin::norm_rope_store_kernel<2>);
        case 4: return go(qlin::norm_rope_store_kernel<4>);
        case 8: return go(qlin::norm_rope_store_kernel<8>);
        case 16: return go(qlin::norm_rope_store_kernel<16>);
        default: return go(qlin::norm_rope_store_kernel<32>);
    }
}

int qlin_launch_qk_norm_rope_store_kv8(const qlin_qk_rope *how, const qlin_kv8_cache *cache, const float *q,
                                       size_t q_stride, const float *k, size_t k_stride, const float *v,
                                       size_t v_stride, float *q_out, int rows, int n_heads, const int *start_pos_dev,
                                       const int *n_rows_dev) {
    if (int rc = qlin::check_kv8(cache)) return rc;
    const int kv = cache->kv_heads, hd = cache->head_dim;
    if (rows < 0 || n_heads <= 0 || n_heads % kv) return QLIN_ERR_SHAPE;
    if (rows > 1 << 20 || n_heads > 65536) return QLIN_ERR_LIMIT;
    if (int rc = qlin::check_how(how, hd)) return rc;
    const size_t qw = static_cast<size_t>(n_heads) * hd, kw = static_cast<size_t>(kv) * hd;
    if (q_stride < qw || k_stride < kw || v_stride < kw || (q == q_out && q_stride != qw)) return QLIN_ERR_SHAPE;
    if (rows == 0 || cache->n_seqs == 0) return QLIN_OK;
    if (!q || !k || !v || !q_out || !start_pos_dev) return QLIN_ERR_NULL;
    for (const void *p : {static_cast<const void *>(q), static_cast<const void *>(k), static_cast<const void *>(v),
                          static_cast<const void *>(q_out), static_cast<const void *>(start_pos_dev),
                          static_cast<const void *>(n_rows_dev)})
        if (!qlin::aligned_to(p, 4)) return QLIN_ERR_ALIGN;
    const int lanes = hd <= 64 ? 8 : hd <= 128 ? 16 : 32, tok = qlin::kThreads / lanes;
    const int slots = (rows + qlin::kKv8Block - 2) / qlin::kKv8Block + 1;  // blocks that `rows` positions can touch
    const int64_t kv_groups = static_cast<int64_t>(cache->n_seqs) * kv * slots;
    const int64_t lines = static_cast<int64_t>(cache->n_seqs) * rows;
    if (lines > (int64_t{1} << 31) || kv_groups > (1 << 23)) return QLIN_ERR_LIMIT;
    const int64_t grid = kv_groups + (lines * n_heads + tok - 1) / tok;
    if (grid > (1 << 23)) return QLIN_ERR_LIMIT;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(qlin::kThreads), 0, qlin::current_stream(), *how,
                           qlin::kv8_view(cache), q, q_stride, k, k_stride, v, v_stride, q_out, rows, n_heads,
                           cache->n_seqs, slots, start_pos_dev, n_rows_dev);
        return qlin::launched(hipGetLastError());
    };
    switch (hd) {
        case 64: return go(qlin::norm_rope_store_kv8_kernel<64>);
        case 96: return go(qlin::norm_rope_store_kv8_kernel<96>);
        case 128: return go(qlin::norm_rope_store_kv8_kernel<128>);
        case 192: return go(qlin::norm_rope_store_kv8_kernel<192>);
        default: return go(qlin::norm_rope_store_kv8_kernel<256>);
    }
}

int qlin_launch_kv8_read(const qlin_kv8_cache *cache, const int *first_dev, const int *lens_dev, int count,
                         float *k_out, float *v_out) {
    if (int rc = qlin::check_kv8(cache)) return rc;
    if (count < 0) return QLIN_ERR_SHAPE;
    if (count == 0 || cache->n_seqs == 0) return QLIN_OK;
    if (!first_dev || !lens_dev || !k_out || !v_out) return QLIN_ERR_NULL;
    if (!qlin::aligned_to(first_dev, 4) || !qlin::aligned_to(lens_dev, 4) || !qlin::aligned_to(k_out, 4) ||
        !qlin::aligned_to(v_out, 4))
        return QLIN_ERR_ALIGN;
    const int64_t parts = (static_cast<int64_t>(count) + 31) / 32;
    const int64_t grid = static_cast<int64_t>(cache->n_seqs) * cache->kv_heads * parts;
    if (parts > (1 << 23) || grid > (1 << 23)) return QLIN_ERR_LIMIT;
    hipLaunchKernelGGL(qlin::kv8_read_kernel, dim3(static_cast<unsigned>(grid)), dim3(qlin::kThreads), 0,
                       qlin::current_stream(), qlin::kv8_view(cache), cache->head_dim, first_dev, lens_dev, count,
                       static_cast<int>(parts), k_out, v_out);
    return qlin::launched(hipGetLastError());
}

}  // extern "C"
