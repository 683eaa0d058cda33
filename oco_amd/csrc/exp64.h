// 64-bit values for decisions that must not hang on a rounding.
#pragma once
#include "common.h"

namespace oco {

constexpr double LOG2E = 1.4426950408889634074;

// 2^x by the Taylor series of e^(f ln 2) about f = 0, f = x - round(x):
// |f ln 2| <= 0.3466, so the first term left out is at most 0.3466^(D+1) /
// (D+1)! relative: 7e-12 for D = 9, 1.7e-16 for D = 12.  N at once, term by
// term: the chains of dependent FMAs run side by side and share their
// constants.  x is taken into -1000 .. 1000 (a NaN too).
template <int D, int N>
__device__ __forceinline__ void exp2_clamped(const double *x, double *y) {
    constexpr double C[13] = {1.0, 0.69314718055994530942, 0.24022650695910071233, 0.055504108664821579953,
                              0.0096181291076284771619, 0.0013333558146428443423, 0.00015403530393381609954,
                              1.5252733804059840280e-5, 1.3215486790144309488e-6, 1.0178086009239699728e-7,
                              7.0549116208011233299e-9, 4.4455382718708114976e-10, 2.5678435993488205142e-11};
    double n[N], f[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const double t = fmin(fmax(x[i], -1000.0), 1000.0);
        n[i] = __builtin_rint(t);
        f[i] = t - n[i];
        y[i] = C[D];
    }
#pragma unroll
    for (int d = D - 1; d >= 0; d--)
#pragma unroll
        for (int i = 0; i < N; i++) y[i] = __builtin_fma(y[i], f[i], C[d]);
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = __builtin_ldexp(y[i], (int)n[i]);
}
// The same of one x, with 0 below 2^-1000 (and for -Inf), Inf from 2^1000 on and NaN for NaN.
template <int D>
__device__ __forceinline__ double exp2_f64(double x) {
    double y;
    exp2_clamped<D, 1>(&x, &y);
    return x < -1000.0 ? 0.0 : x < 1000.0 ? y : x + __builtin_inf();
}

// 1 / d for a normal d whose reciprocal is normal: the hardware's estimate and two Newton steps.
__device__ __forceinline__ double recip_f64(double d) {
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}
// 1 / sqrt(d) likewise; 0 and Inf give Inf and 0.
__device__ __forceinline__ double rsqrt_f64(double d) {
    const double e = __builtin_amdgcn_rsq(d);
    double r = e;
#pragma unroll
    for (int i = 0; i < 2; i++) r = __builtin_fma(0.5 * r, __builtin_fma(-d * r, r, 1.0), r);
    return d > 0.0 && d < __builtin_inf() ? r : e;
}

// 64-bit values across a wavefront by DPP and permlane swaps: a step is a few
// clocks where a shuffle through LDS is over a hundred.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double v) {  // 0 where the source is outside, or the row is masked
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double words_f64(uint32_t lo, uint32_t hi) {
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
// The inclusive sums over the lanes: within rows of 16, then the rows before.
__device__ __forceinline__ double wave_scan_f64(double v) {
    v += dpp_f64<0x111>(v);  // row_shr 1, 2, 4, 8
    v += dpp_f64<0x112>(v);
    v += dpp_f64<0x114>(v);
    v += dpp_f64<0x118>(v);
    v += dpp_f64<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
    v += dpp_f64<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
    return v;
}
// The value of a lane that is the same for all.
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return words_f64((uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane));
}

// The sum in every lane: lane 0's (the rotations add in another order in other lanes).
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x124>(v);
    v += dpp_f64<0x128>(v);
    uint64_t b = (uint64_t)__double_as_longlong(v);
    auto l = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
    auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    v = words_f64(l[0], h[0]) + words_f64(l[1], h[1]);
    b = (uint64_t)__double_as_longlong(v);
    l = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
    h = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    return lane_f64(words_f64(l[0], h[0]) + words_f64(l[1], h[1]), 0);
}

// Maximum and minimum of 32-bit words over a wavefront, uniform: within rows of
// 16 by rotations, then each row takes the last lane of the rows before it
// (f of a value with itself is that value, so lanes without a source keep
// theirs); lane 63 has it all.
template <class F>
__device__ __forceinline__ uint32_t wave_reduce_u32(uint32_t v, F f) {
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xf, 0xf, true));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xf, 0xf, true));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x124, 0xf, 0xf, true));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x128, 0xf, 0xf, true));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x142, 0xf, 0xf, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x143, 0xf, 0xf, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    return wave_reduce_u32(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {
    return wave_reduce_u32(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ float wave_max_f32(float v) {
    return __uint_as_float(wave_reduce_u32(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}

// 64-bit values as integers that order alike (-0 as +0); 0 is below every
// number, -Inf included.
__device__ __forceinline__ uint64_t order_f64(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

}  // namespace oco
