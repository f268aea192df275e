// 16-bit element types of the decoding kernels (w4.hip, rope.hip, tree_attention.hip): vectors, conversions, matrix instructions; loops over constants.
#ifndef R355_HALF_TYPES_HPP
#define R355_HALF_TYPES_HPP

#include <cstdint>
#include <type_traits>

#include <hip/hip_runtime.h>

namespace r355
{
    using f32x4 = float __attribute__((ext_vector_type(4)));
    using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
    using u32x2 = uint32_t __attribute__((ext_vector_type(2)));

    template <typename T, int N>
    using vec = T __attribute__((ext_vector_type(N)));

    // D = A B + C on one 16 x 16 block.  Lane l holds row (A) or column (B) l % 16, k = 8 (l / 16) + 0..7 of 32, and of C and D
    // column l % 16, rows 4 (l / 16) + 0..3.
    template <typename T>
    __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c)
    {
        if constexpr(__is_same(T, __bf16))
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec<__bf16, 8>, a), __builtin_bit_cast(vec<__bf16, 8>, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec<_Float16, 8>, a), __builtin_bit_cast(vec<_Float16, 8>, b), c, 0, 0, 0);
    }

    // the same with k = 4 (l / 16) + 0..3 of 16
    template <typename T>
    __device__ __forceinline__ f32x4 mfma16(u32x2 a, u32x2 b, f32x4 c)
    {
        if constexpr(__is_same(T, __bf16))
            return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(vec<short, 4>, a), __builtin_bit_cast(vec<short, 4>, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(vec<_Float16, 4>, a), __builtin_bit_cast(vec<_Float16, 4>, b), c, 0, 0, 0);
    }

    // two floats rounded to nearest even, the first in the low half
    template <typename T>
    __device__ __forceinline__ uint32_t pack2(float lo, float hi)
    {
        return __builtin_bit_cast(uint32_t, vec<T, 2>{static_cast<T>(lo), static_cast<T>(hi)});
    }

    // calls f with the integral constants 0 .. N - 1
    template <uint32_t N, typename F>
    __device__ __forceinline__ void each(F&& f)
    {
        if constexpr(N > 0u)
        {
            each<N - 1u>(f);
            f(std::integral_constant<uint32_t, N - 1u>{});
        }
    }
} // namespace r355

#endif // R355_HALF_TYPES_HPP
