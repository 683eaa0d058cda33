// 64-bit exponentials for decisions that must not hang on a rounding.
#pragma once
#include "common.h"

namespace oco {

constexpr double LOG2E = 1.4426950408889634074;

// 2^x by the Taylor series of e^(f ln 2) about f = 0, f = x - round(x):
// |f ln 2| <= 0.3466, so the first term left out is at most 0.3466^(D+1) /
// (D+1)! relative: 7e-12 for D = 9, 1.7e-16 for D = 12.  0 below 2^-1000
// (and for -Inf), Inf from 2^1000 on, NaN for NaN.
template <int D>
__device__ __forceinline__ double exp2_f64(double x) {
    constexpr double C[13] = {1.0, 0.69314718055994530942, 0.24022650695910071233, 0.055504108664821579953,
                              0.0096181291076284771619, 0.0013333558146428443423, 0.00015403530393381609954,
                              1.5252733804059840280e-5, 1.3215486790144309488e-6, 1.0178086009239699728e-7,
                              7.0549116208011233299e-9, 4.4455382718708114976e-10, 2.5678435993488205142e-11};
    const double n = __builtin_rint(x), f = x - n;
    double r = C[D];
#pragma unroll
    for (int i = D - 1; i >= 0; i--) r = __builtin_fma(r, f, C[i]);
    // |n| <= 1000 keeps ldexp's integer in range
    const double y = __builtin_ldexp(r, (int)fmin(fmax(n, -1000.0), 1000.0));
    return x < -1000.0 ? 0.0 : x >= 1000.0 ? __builtin_inf() : y;
}

__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, o), hi = (uint32_t)__shfl_xor((int)(b >> 32), o);
    return __longlong_as_double(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += shfl_xor_f64(v, o);
    return v;
}

// 64-bit values as integers that order alike (-0 as +0); 0 is below every
// number, -Inf included.
__device__ __forceinline__ uint64_t order_f64(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

}  // namespace oco
