// Eight values of a row as they lie in memory, rounded by the hardware's
// conversions.
#pragma once
#include <type_traits>

#include "rows.h"

namespace oco {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <class T>
struct Eight {
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = ((const GLOBAL u32x4_u *)gp((const u32x4_u *)p))[i];
    }
    __device__ __forceinline__ void values(float *v) const {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t u = sizeof(T) == 4 ? w[j / 4 % (sizeof(T) / 2)][j % 4] : w[0][j / 2];
            if constexpr (sizeof(T) == 4)
                v[j] = __uint_as_float(u);
            else if constexpr (std::is_same_v<T, bf16_t>)
                v[j] = __uint_as_float(j % 2 ? u & 0xffff0000u : u << 16);
            else
                v[j] = half_bits_to_f32(j % 2 ? u >> 16 : u & 0xffff);
        }
    }
    // rounded by the hardware's conversions
    __device__ __forceinline__ void round(const float *v) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (sizeof(T) == 4) {
                w[j / 4][j % 4] = __float_as_uint(v[j]);
            } else if (j % 2 == 0) {
                if constexpr (std::is_same_v<T, bf16_t>)
                    w[0][j / 2] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[j], (__bf16)v[j + 1]});
                else
                    w[0][j / 2] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[j], (_Float16)v[j + 1]});
            }
        }
    }
    // past the caches
    __device__ __forceinline__ void stream(T *p) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) __builtin_nontemporal_store(w[i], (GLOBAL u32x4_u *)gp((u32x4_u *)p) + i);
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) ((GLOBAL u32x4_u *)gp((u32x4_u *)p))[i] = w[i];
    }
    // the first n of them (LDS or memory)
    __device__ __forceinline__ void store_some(T *p, uint32_t n) const {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            if (j >= n) break;
            if constexpr (sizeof(T) == 4)
                p[j] = __uint_as_float(w[j / 4][j % 4]);
            else
                p[j].bits = (uint16_t)(w[0][j / 2] >> (16 * (j % 2)));
        }
    }
};

}  // namespace oco
