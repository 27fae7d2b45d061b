// qlin_f64.hpp -- sums over a wave and the exponential in 64 bits (gfx950 device code).
//
// On this chip an f64 operation takes an f32 one's time, so what must not depend on the order of a sum (codes next to a
// border, random numbers next to the border between two tokens, scores next to one another) is computed in f64.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qlin {

template <int CTRL>
__device__ __forceinline__ double dpp_move_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ double halves(uint32_t hi, uint32_t lo) {
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
// The sum over the wave in every lane, always in the same order (every lane active).
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_move_f64<0xb1>(v);   // quad_perm [1, 0, 3, 2]
    v += dpp_move_f64<0x4e>(v);   // quad_perm [2, 3, 0, 1]
    v += dpp_move_f64<0x141>(v);  // row_half_mirror
    v += dpp_move_f64<0x140>(v);  // row_mirror
    uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t l = static_cast<uint32_t>(u), h = static_cast<uint32_t>(u >> 32);
    const auto l16 = __builtin_amdgcn_permlane16_swap(l, l, false, false);  // rows 0, 0, 2, 2 and 1, 1, 3, 3
    const auto h16 = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    v = halves(h16[0], l16[0]) + halves(h16[1], l16[1]);
    u = __builtin_bit_cast(uint64_t, v);
    l = static_cast<uint32_t>(u), h = static_cast<uint32_t>(u >> 32);
    const auto l32 = __builtin_amdgcn_permlane32_swap(l, l, false, false);
    const auto h32 = __builtin_amdgcn_permlane32_swap(h, h, false, false);
    return halves(h32[0], l32[0]) + halves(h32[1], l32[1]);
}

// The sums over lanes 0 .. l in lane l (every lane active): within rows of 16 lanes by shifts of 1, 2, 4 and 8, then the last
// lane of a row to the row after it, and lane 31 to the upper half.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_from_f64(double x) {  // 0 in lanes that nothing comes to
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
    return halves(hi, lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {
    v += dpp_from_f64<0x111, 0xf>(v);  // row_shr
    v += dpp_from_f64<0x112, 0xf>(v);
    v += dpp_from_f64<0x114, 0xf>(v);
    v += dpp_from_f64<0x118, 0xf>(v);
    v += dpp_from_f64<0x142, 0xa>(v);  // row_bcast15 to rows 1 and 3
    v += dpp_from_f64<0x143, 0xc>(v);  // row_bcast31 to rows 2 and 3
    return v;
}

// e^x: n = rint(x / ln 2), e^x = 2^n e^r with r = x - n ln 2, |r| <= ln 2 / 2, from ln 2 in two parts, and e^r by its
// Taylor polynomial of degree 13 (the first term left out is below 5e-18).  1 to 2 units of the last place; 0 from about
// -745 down, infinite from 710 up, 0 for NaN.
__device__ __forceinline__ double exp_f64(double x) {
    x = fmin(fmax(x, -1100.0), 1100.0);  // (fmax takes the number beside a NaN)
    const double n = __builtin_rint(x * 0x1.71547652b82fep+0);
    double r = __builtin_fma(n, -0x1.62e42fefa39efp-1, x);
    r = __builtin_fma(n, -0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, static_cast<int>(n));
}

}  // namespace qlin
