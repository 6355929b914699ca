// pgm_exp.h -- the exponential of the N^2 passes and of the draws.
#pragma once
#include <hip/hip_runtime.h>

// exp(x) for x <= 0 in fp64, ~1 ulp: n = rint(x log2 e), r = x - n ln 2 (two-part), degree-13 Taylor
// polynomial on |r| <= ln2/2 (truncation 4e-18), scaled by 2^n with v_ldexp_f64 (underflows to 0
// by itself).  19 instructions against ~35 for the library call; every N^2 pass pays one per
// (pair, mixture, dimension).
// exp_neg_fast: no clamp in front -- for FINITE x far below the underflow threshold n is a large negative number, v_cvt_i32_f64
// saturates and v_ldexp_f64 returns 0, one instruction less per pair and mixture.  Only for arguments that are finite by
// construction: -(a - b)^2 of two staged per-point factors in the 1-D build and its gradient epilogue (|a - b| < 1.3e154, i.e.
// any parameter a constraint admits).  x = -inf would give NaN (inf - inf in the reduction), |x| > 1e45 a garbage reduced
// argument: everything else goes through exp_neg, which clamps first (-800 is far below the underflow of 2^-1074).
__device__ __forceinline__ double exp_neg_fast(double x) {
  const double n = rint(x * 1.4426950408889634074);
  double r = __builtin_fma(-n, 6.93147180369123816490e-01, x);
  r = __builtin_fma(-n, 1.90821492927058770002e-10, r);
  double p = 1.6059043836821613e-10;                      // 1/13!
  p = __builtin_fma(p, r, 2.08767569878681e-09);          // 1/12!
  p = __builtin_fma(p, r, 2.505210838544172e-08);         // 1/11!
  p = __builtin_fma(p, r, 2.755731922398589e-07);         // 1/10!
  p = __builtin_fma(p, r, 2.7557319223985893e-06);        // 1/9!
  p = __builtin_fma(p, r, 2.48015873015873e-05);          // 1/8!
  p = __builtin_fma(p, r, 1.984126984126984e-04);         // 1/7!
  p = __builtin_fma(p, r, 1.388888888888889e-03);         // 1/6!
  p = __builtin_fma(p, r, 8.333333333333333e-03);         // 1/5!
  p = __builtin_fma(p, r, 4.1666666666666664e-02);        // 1/4!
  p = __builtin_fma(p, r, 1.6666666666666666e-01);        // 1/3!
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return ldexp(p, (int)n);                                 // (|n| <= ~1155 after the clamp below; without it the conversion saturates in hardware)
}
// The general form: exp(-inf) = 0, and so is every finite x below the underflow threshold; the integer conversion stays in range.
__device__ __forceinline__ double exp_neg(double x) { return exp_neg_fast(fmax(x, -800.0)); }
