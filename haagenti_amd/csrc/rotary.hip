// Rotary positions (hh_rotary; rules: haagenti_hip.h): pair j of every head
// of a token turns by the angle (token's position on j's axis) x freq[j],
//   (a, b) -> (a cos - b sin, b cos + a sin),
// the inverse by the negative angle, which is also the gradient's way back.
//
// Bound by memory.  A workgroup takes a few tokens: it first computes their
// cosines and sines into LDS, once for all heads, then turns 8 pairs a thread
// at a time (16 bytes of each half, or 32 bytes of neighbours).  Angles are
// counted in turns in 64 bits, reduced there and rounded to f32: a position of
// a million times a frequency of 1 is off by 2^-26 of a turn like any other,
// where f32 throughout would be off by 2^-7.
// 16200 tokens of 20 heads of 128 bf16, three axes: 28 us, 166 MB at 5.9 TB/s;
// 16 tokens of 40 heads 3.7 us.
#include "layer_ops.hpp"

namespace hh {
namespace {

struct RotaryArgs {
    hh_rotary_args a;
    uint32_t pairs, tokens_each, heads_each;  // a workgroup's tokens and heads
    uint32_t chunks, rest;                    // 8 pairs each; pieces of 16 values past the pairs that are copied
};

template <int XT>
struct Of {
    typedef uint16_t type;
    static __device__ __forceinline__ float get(type v) { return half_to_f32<XT>(v); }
    static __device__ __forceinline__ type put(float v) { return (type)f32_to_half<XT>(v); }
};
template <>
struct Of<HH_F32> {
    typedef float type;
    static __device__ __forceinline__ float get(type v) { return v; }
    static __device__ __forceinline__ type put(float v) { return v; }
};
template <typename E>
struct Eight {
    E v[8];
};
// 8 values at an address aligned to its elements only.
template <typename E>
__device__ __forceinline__ Eight<E> load8(const E *p) {
    typedef u32x4 any __attribute__((aligned(2)));
    Eight<E> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; i++) {
        const u32x4 x = reinterpret_cast<const any *>(p)[i];
        __builtin_memcpy(reinterpret_cast<char *>(&r) + 16 * i, &x, 16);
    }
    return r;
}
template <typename E>
__device__ __forceinline__ void store8(E *p, const Eight<E> &r) {
    typedef u32x4 any __attribute__((aligned(2)));
#pragma unroll
    for (int i = 0; i < (int)sizeof(E) / 2; i++) {
        u32x4 x;
        __builtin_memcpy(&x, reinterpret_cast<const char *>(&r) + 16 * i, 16);
        reinterpret_cast<any *>(p)[i] = x;
    }
}

template <int XT, bool NEXT>  // NEXT: pairs are neighbours (2 j, 2 j + 1), else j and j + pairs
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs p) {
    typedef typename Of<XT>::type E;
    extern __shared__ __align__(16) float table[];  // cosines [token][pairs], sines
    const hh_rotary_args &a = p.a;
    const uint32_t t0 = blockIdx.x * p.tokens_each, tokens = min(p.tokens_each, a.tokens - t0);
    const uint32_t h0 = blockIdx.y * p.heads_each, heads = min(p.heads_each, a.heads - h0);
    float *cosine = table, *sine = table + p.tokens_each * p.pairs;
    for (uint32_t i = threadIdx.x; i < tokens * p.pairs; i += 256) {
        const uint32_t t = i / p.pairs, j = i % p.pairs;
        uint32_t axis = 0, end = a.sections[0];
        while (axis + 1 < a.axes && j >= end) end += a.sections[++axis];
        const double turns = (double)a.d_positions[axis * a.position_stride + t0 + t] * (double)a.d_freq[j] *
                             0.15915494309189533576888;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        cosine[i] = c, sine[i] = a.inverse ? -s : s;
    }
    __syncthreads();
    const E *x = reinterpret_cast<const E *>(a.d_x);
    E *y = reinterpret_cast<E *>(a.d_y);
    const uint32_t each = p.chunks + p.rest, items = tokens * heads * each;
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < items; i += 256) {
        const uint32_t piece = i % each, th = i / each, h = th % heads, t = th / heads;
        const E *from = x + (uint64_t)(t0 + t) * a.x_token_stride + (uint64_t)(h0 + h) * a.x_head_stride;
        E *to = y + (uint64_t)(t0 + t) * a.y_token_stride + (uint64_t)(h0 + h) * a.y_head_stride;
        if (piece >= p.chunks) {
            const uint32_t at = 2 * p.pairs + (piece - p.chunks) * 8;
            if (at + 8 <= a.dim)
                store8(to + at, load8(from + at));
            else
                for (uint32_t e = at; e < a.dim; e++) to[e] = from[e];
            continue;
        }
        const uint32_t j = piece * 8;
        const float *c = cosine + t * p.pairs + j, *s = sine + t * p.pairs + j;
        if (j + 8 <= p.pairs) {
            Eight<E> u = load8(from + (NEXT ? 2 * j : j)), v = load8(from + (NEXT ? 2 * j + 8 : j + p.pairs));
            Eight<E> lo, hi;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                E &first = NEXT ? (e < 4 ? u.v[2 * e & 7] : v.v[2 * e & 7]) : u.v[e];
                E &second = NEXT ? (e < 4 ? u.v[(2 * e & 7) + 1] : v.v[(2 * e & 7) + 1]) : v.v[e];
                const float p0 = Of<XT>::get(first), p1 = Of<XT>::get(second);
                const E q0 = Of<XT>::put(fmaf(-p1, s[e], p0 * c[e])), q1 = Of<XT>::put(fmaf(p0, s[e], p1 * c[e]));
                if (NEXT) {
                    (e < 4 ? lo : hi).v[2 * e & 7] = q0;
                    (e < 4 ? lo : hi).v[(2 * e & 7) + 1] = q1;
                } else {
                    lo.v[e] = q0, hi.v[e] = q1;
                }
            }
            store8(to + (NEXT ? 2 * j : j), lo);
            store8(to + (NEXT ? 2 * j + 8 : j + p.pairs), hi);
        } else {
            for (uint32_t e = 0; j + e < p.pairs; e++) {
                const uint32_t i0 = NEXT ? 2 * (j + e) : j + e, i1 = NEXT ? i0 + 1 : i0 + p.pairs;
                const float p0 = Of<XT>::get(from[i0]), p1 = Of<XT>::get(from[i1]);
                to[i0] = Of<XT>::put(fmaf(-p1, s[e], p0 * c[e]));
                to[i1] = Of<XT>::put(fmaf(p0, s[e], p1 * c[e]));
            }
        }
    }
}

template <int XT>
void launch_rotary(const RotaryArgs &p, dim3 grid, size_t lds, hipStream_t s) {
    if (p.a.interleaved)
        hipLaunchKernelGGL((rotary_kernel<XT, true>), grid, dim3(256), lds, s, p);
    else
        hipLaunchKernelGGL((rotary_kernel<XT, false>), grid, dim3(256), lds, s, p);
}

}  // namespace
}  // namespace hh

extern "C" int32_t hh_rotary(hh_context *ctx, const hh_rotary_args *a, void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    if (a->dtype != HH_F32 && a->dtype != HH_F16 && a->dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (a->axes < 1 || a->axes > 4) return HH_ERR_UNSUPPORTED;
    uint64_t pairs = 0;
    for (uint32_t i = 0; i < a->axes; i++) pairs += a->sections[i];
    if (pairs > 512 || a->dim > 65536) return HH_ERR_UNSUPPORTED;
    if (2 * pairs > a->dim) return HH_ERR_INVALID_ARGUMENT;
    if (a->tokens >= 1u << 31 || a->heads > 65535) return HH_ERR_INVALID_ARGUMENT;
    if (!a->tokens || !a->heads || !a->dim) return HH_OK;
    if (!a->d_x || !a->d_y || (pairs && (!a->d_positions || !a->d_freq))) return HH_ERR_INVALID_ARGUMENT;
    const uintptr_t size = a->dtype == HH_F32 ? 4 : 2;
    if ((((uintptr_t)a->d_x | (uintptr_t)a->d_y) & (size - 1)) || (((uintptr_t)a->d_positions | (uintptr_t)a->d_freq) & 3u))
        return HH_ERR_INVALID_ARGUMENT;
    if (hh::rows_meet(a->tokens, a->heads, a->y_token_stride, a->y_head_stride, a->dim)) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hh::RotaryArgs p = {};
    p.a = *a;
    p.pairs = (uint32_t)pairs;
    p.chunks = (p.pairs + 7) / 8;
    // what lies past the pairs stays as it is: nothing to do in place
    const bool in_place = a->d_x == a->d_y && (a->tokens == 1 || a->x_token_stride == a->y_token_stride) &&
                          (a->heads == 1 || a->x_head_stride == a->y_head_stride);
    if (a->d_x == a->d_y && !in_place) return HH_ERR_INVALID_ARGUMENT;
    p.rest = in_place ? 0 : (a->dim - 2 * p.pairs + 7) / 8;
    const uint32_t each = p.chunks + p.rest;
    if (!each) return HH_OK;
    // A workgroup's threads have about 4 pieces each where there are enough
    // tokens for 8 workgroups to a CU, else one token and a piece or two.
    const uint64_t cus = ctx->num_cus > 0 ? ctx->num_cus : 256, all = (uint64_t)each * a->heads;
    uint64_t want = (1024 + all - 1) / all, most = a->tokens / (8 * cus);
    if (want > most) want = most;
    if (want > 16) want = 16;
    const uint64_t room = p.pairs ? 4096 / p.pairs : 16;  // 32 KiB of cosines and sines
    if (want > room) want = room;
    p.tokens_each = want < 1 ? 1 : (uint32_t)want;
    p.heads_each = a->heads;
    if (p.tokens_each == 1 && a->tokens < 2 * cus) {
        p.heads_each = 512 / each < 1 ? 1 : 512 / each;
        if (p.heads_each > a->heads) p.heads_each = a->heads;
    }
    const dim3 grid((a->tokens + p.tokens_each - 1) / p.tokens_each, (a->heads + p.heads_each - 1) / p.heads_each);
    if ((uint64_t)grid.x * 256 >= 1ull << 32) return HH_ERR_UNSUPPORTED;
    const size_t lds = (size_t)p.tokens_each * p.pairs * 2 * sizeof(float);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (a->dtype) {
        case HH_F32: hh::launch_rotary<HH_F32>(p, grid, lds, s); break;
        case HH_F16: hh::launch_rotary<HH_F16>(p, grid, lds, s); break;
        default: hh::launch_rotary<HH_BF16>(p, grid, lds, s); break;
    }
    return hh::from_hip(hipGetLastError());
}
