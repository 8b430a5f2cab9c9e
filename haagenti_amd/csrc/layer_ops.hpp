// What the decoder-layer operators (linear.hip, gated.hip, gated_backward.hip,
// norm.hip, rotary.hip, kv_cache.hip, kv_attention.hip, diff_attention.hip)
// share.
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
// The checks that the gated products' two passes share (gated.hip).
int32_t check_gated(const hh_gated_args *a);
// Whether two rows of `dim` elements, `tokens` of them `ts` apart for each of
// `heads` heads `hs` apart, share an element (kv_cache.hip).
bool rows_meet(uint64_t tokens, uint64_t heads, uint64_t ts, uint64_t hs, uint64_t dim);

// A wave's sum, in every lane and the same in all of them: neighbours, pairs
// and halves of a row of 16 lanes by DPP, rows by swaps (no LDS).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0xb1>(v);   // lane ^ 1
    v += dpp<0x4e>(v);   // lane ^ 2
    v += dpp<0x141>(v);  // 7 - lane of 8
    v += dpp<0x140>(v);  // 15 - lane of 16
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

}  // namespace hh
