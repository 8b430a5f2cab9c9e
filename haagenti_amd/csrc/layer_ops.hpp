// What the decoder-layer operators (linear.hip, kv_cache.hip,
// kv_attention.hip) share on the device.
#pragma once

#include "hh_internal.hpp"

namespace hh {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16-bit element DT (HH_F16 or HH_BF16) -> f32 (exact) and back (nearest even).
template <int DT>
__device__ __forceinline__ float half_to_f32(uint32_t bits) {
    if constexpr (DT == HH_BF16)
        return __uint_as_float(bits << 16);
    else
        return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
template <int DT>
__device__ __forceinline__ uint32_t f32_to_half(float f) {
    if constexpr (DT == HH_BF16)
        return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f);
    else
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f);
}

// The checks of a cache that its entry points share (kv_cache.hip).
int32_t check_kv_cache(const hh_kv_cache *c);

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

}  // namespace hh
