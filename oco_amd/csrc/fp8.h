// Rows in 8-bit floating point (OCP e4m3: four exponent bits, three mantissa
// bits, largest value 448) with one f32 scale per 128 columns, and their
// products.
#pragma once
#include "exp64.h"

namespace oco {

constexpr uint32_t FP8_BLOCK = 128;
constexpr float FP8_FLOOR = 0x1.cp-118f;  // 448 * 2^-126: the least block maximum, so that scales are normal

// Maximum over the 16 lanes of a DPP row, in every lane.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp16(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, dpp16<0xB1>(v));
    v = max(v, dpp16<0x4E>(v));
    v = max(v, dpp16<0x124>(v));
    return max(v, dpp16<0x128>(v));
}

// The codes and the scale of a block of 128 columns, eight in each of 16
// consecutive lanes (all of them active): scale = max|v| / 448, code =
// e4m3(448 v / max|v|), nearest even.  The quotient is formed as
// (0.875 v) / (max|v| / 512), whose operands are exact for 16-bit v, and is
// rounded to f32 once: reciprocal, product, and one residual step, which
// returns the rounded quotient where the reciprocal is itself rounded
// correctly (Markstein).  A quotient on the border between two codes thus
// stays on it.  Blocks under 2^-64 enter 2^64 times larger, as the residual of
// those near the least normal number would be subnormal.  A block that holds a
// NaN or an infinity has a NaN scale (its row's products are NaN) and NaN codes.
// |v| orders by its bits: finite values, then infinity, then NaN.
__device__ __forceinline__ uint2 fp8_block(const float *v, float &scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    m = row16_max(m);
    float top = fmaxf(__uint_as_float(m), FP8_FLOOR);
    if (m >= 0x7f800000u) {
        scale = __uint_as_float(0x7fc00000u);
        return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    }
    scale = top / 448.0f;
    float rate = 0.875f;
    if (__ballot(top < 0x1p-64f)) {  // a branch, which the asm keeps: 4096 x 4096 bf16 in 10.7 us, 11.1 as selects
        asm volatile("" ::: "memory");
        const bool tiny = top < 0x1p-64f;
        top = tiny ? top * 0x1p64f : top;
        rate = tiny ? 0.875f * 0x1p64f : 0.875f;
    }
    const float den = top * 0x1p-9f, inv = 1.0f / den;
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float num = v[j] * rate, first = num * inv;
        q[j] = copysignf(fmaf(fmaf(-first, den, num), inv, first), first);  // -0 stays -0
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// The same for f32 rows that were computed in 64 bits, v[j] times `factor`:
// the codes are those of the 64-bit quotients, so that a value next to a
// border between two codes does not hang on the roundings of a norm.  Whether
// all are finite is seen on the f32 values o.
__device__ __forceinline__ uint2 fp8_block(const double *v, double factor, const float *o, float &scale) {
    uint32_t m = 0;
    double top = 0.0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        m = max(m, __float_as_uint(o[j]) & 0x7fffffffu);
        top = fmax(top, fabs(v[j]));
    }
    m = row16_max(m);
    top = fmax(top, dpp_f64<0xB1>(top));
    top = fmax(top, dpp_f64<0x4E>(top));
    top = fmax(top, dpp_f64<0x124>(top));
    top = fmax(top, dpp_f64<0x128>(top)) * factor;
    if (m >= 0x7f800000u) {
        scale = __uint_as_float(0x7fc00000u);
        return make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    }
    top = fmax(top, (double)FP8_FLOOR);
    scale = (float)(top * (1.0 / 448.0));
    const double rate = 448.0 * factor * recip_f64(top);
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // to f32 by chopping, with the last bit set where that is inexact: the code is then rounded once
        const uint64_t b = (uint64_t)__double_as_longlong(v[j] * rate);
        const uint32_t lo = (uint32_t)b;
        q[j] = (float)words_f64((lo & 0xe0000000u) | (lo & 0x1fffffffu ? 0x20000000u : 0u), (uint32_t)(b >> 32));
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

}  // namespace oco
