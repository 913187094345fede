// sin and cos of a rotary angle held in double precision (shared by the rotary kernels).
#pragma once

namespace gkv {

// Cody-Waite reduction by pi/2 in double precision (pi/2 split into two doubles, fused
// multiply-adds), then Taylor polynomials of sin and cos on |x| <= pi/4 in float (Horner with fused
// multiply-adds; truncation error below 2^-28).
__device__ __forceinline__ void rope_sincos_f64(double t, float& s_out, float& c_out) {
    const double k = rint(__dmul_rn(t, 0.63661977236758134308));  // 2/pi
    double r = __fma_rn(-k, 1.5707963267948966192, t);              // pi/2, high part
    r = __fma_rn(-k, 6.1232339957367660359e-17, r);                 // pi/2, low part
    const float x = __double2float_rn(r);
    const float x2 = __fmul_rn(x, x);
    // sin x = x + x^3 (-1/3! + x^2 (1/5! + x^2 (-1/7! + x^2 (1/9! - x^2/11!))))
    float ps = __fmaf_rn(x2, -2.5052108385441720e-8f, 2.7557319223985893e-6f);
    ps = __fmaf_rn(x2, ps, -1.9841269841269841e-4f);
    ps = __fmaf_rn(x2, ps, 8.3333333333333333e-3f);
    ps = __fmaf_rn(x2, ps, -1.6666666666666667e-1f);
    const float sn = __fmaf_rn(__fmul_rn(x, x2), ps, x);
    // cos x = 1 + x^2 (-1/2! + x^2 (1/4! + x^2 (-1/6! + x^2 (1/8! - x^2/10!))))
    float pc = __fmaf_rn(x2, -2.7557319223985891e-7f, 2.4801587301587302e-5f);
    pc = __fmaf_rn(x2, pc, -1.3888888888888889e-3f);
    pc = __fmaf_rn(x2, pc, 4.1666666666666667e-2f);
    pc = __fmaf_rn(x2, pc, -0.5f);
    const float cs = __fmaf_rn(x2, pc, 1.0f);
    switch (static_cast<long long>(k) & 3) {
        case 0: s_out = sn; c_out = cs; break;
        case 1: s_out = cs; c_out = -sn; break;
        case 2: s_out = -sn; c_out = -cs; break;
        default: s_out = -cs; c_out = sn; break;
    }
}

}  // namespace gkv
