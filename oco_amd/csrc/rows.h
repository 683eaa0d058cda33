// Rows of f32, bf16 or f16 values, eight per thread, at any alignment of the
// type: gfx950's global accesses take any byte address, so a row of odd
// length or stride keeps its 16-byte accesses.
#pragma once
#include "common.h"

namespace oco {

struct f16_t {
    uint16_t bits;
};

template <class T>
struct RowIO;

template <>
struct RowIO<float> {
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static __device__ __forceinline__ float round(float v) { return v; }
    static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
    static __device__ __forceinline__ void load8(const float *p, float *v) {
        const u32x4_u *q = reinterpret_cast<const u32x4_u *>(p);
        const u32x4_u a = q[0], b = q[1];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = __uint_as_float(a[j]);
            v[4 + j] = __uint_as_float(b[j]);
        }
    }
    static __device__ __forceinline__ void store8(float *p, const float *v) {
        u32x4_u a, b;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            a[j] = __float_as_uint(v[j]);
            b[j] = __float_as_uint(v[4 + j]);
        }
        u32x4_u *q = reinterpret_cast<u32x4_u *>(p);
        q[0] = a;
        q[1] = b;
    }
};

template <>
struct RowIO<bf16_t> {
    static __device__ __forceinline__ float one(const bf16_t *p) { return bf16_bits_to_f32(p->bits); }
    static __device__ __forceinline__ float round(float v) { return round_bf16(v); }
    static __device__ __forceinline__ void put(bf16_t *p, float v) { p->bits = f32_to_bf16_bits(v); }
    static __device__ __forceinline__ void load8(const bf16_t *p, float *v) {
        const u32x4_u a = *reinterpret_cast<const u32x4_u *>(p);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[2 * j] = __uint_as_float(a[j] << 16);
            v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store8(bf16_t *p, const float *v) {
        u32x4_u a;
#pragma unroll
        for (int j = 0; j < 4; j++)
            a[j] = (uint32_t)f32_to_bf16_bits(v[2 * j]) | ((uint32_t)f32_to_bf16_bits(v[2 * j + 1]) << 16);
        *reinterpret_cast<u32x4_u *>(p) = a;
    }
};

template <>
struct RowIO<f16_t> {
    static __device__ __forceinline__ uint32_t bits(float v) {
        const _Float16 h = (_Float16)v;
        uint16_t b;
        __builtin_memcpy(&b, &h, 2);
        return b;
    }
    static __device__ __forceinline__ float one(const f16_t *p) { return half_bits_to_f32(p->bits); }
    static __device__ __forceinline__ float round(float v) { return half_bits_to_f32(bits(v)); }
    static __device__ __forceinline__ void put(f16_t *p, float v) { p->bits = (uint16_t)bits(v); }
    static __device__ __forceinline__ void load8(const f16_t *p, float *v) {
        const u32x4_u a = *reinterpret_cast<const u32x4_u *>(p);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[2 * j] = half_bits_to_f32(a[j] & 0xffffu);
            v[2 * j + 1] = half_bits_to_f32(a[j] >> 16);
        }
    }
    static __device__ __forceinline__ void store8(f16_t *p, const float *v) {
        u32x4_u a;
#pragma unroll
        for (int j = 0; j < 4; j++) a[j] = bits(v[2 * j]) | (bits(v[2 * j + 1]) << 16);
        *reinterpret_cast<u32x4_u *>(p) = a;
    }
};

// Columns c0 .. c0 + 7 of a row of n; those past its end read as `fill` and
// are not written.
template <class T>
__device__ __forceinline__ void load_run(const T *row, uint32_t c0, uint32_t n, float *v, float fill = 0.f) {
    if (c0 + 8 <= n) {
        RowIO<T>::load8(row + c0, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = c0 + j < n ? RowIO<T>::one(row + c0 + j) : fill;
    }
}
template <class T>
__device__ __forceinline__ void store_run(T *row, uint32_t c0, uint32_t n, const float *v) {
    if (c0 + 8 <= n) {
        RowIO<T>::store8(row + c0, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c0 + j < n) RowIO<T>::put(row + c0 + j, v[j]);
    }
}

// Columns c0 .. c0 + 3 of a row of n.
template <class T>
__device__ __forceinline__ void load_four(const T *row, uint32_t c0, uint32_t n, float *v, float fill = 0.f) {
    if (c0 + 4 <= n) {
        if constexpr (sizeof(T) == 4) {
            const u32x4_u a = *reinterpret_cast<const u32x4_u *>(row + c0);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __uint_as_float(a[j]);
        } else {
            const u32x2_u a = *reinterpret_cast<const u32x2_u *>(row + c0);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const T h = {(uint16_t)(a[j / 2] >> (16 * (j % 2)))};
                v[j] = RowIO<T>::one(&h);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = c0 + j < n ? RowIO<T>::one(row + c0 + j) : fill;
    }
}

}  // namespace oco
