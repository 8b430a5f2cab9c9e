// y = act(x W^T + bias) * mul + residual (hh_linear, include/haagenti_hip.h).
//
// Both routes put W's rows on the first operand of the matrix instructions
// and x's on the second, so a lane ends with 4 consecutive outputs n of one
// row m: bias, mul, residual and y move 4 values at a time.
//
// INT4 weights stay integers: nibbles become the 16-bit numbers 16..31 by
// shifts and ors (exact in f16 and bf16), and the offset of 24 goes into the
// accumulator's start, -24 sum(x) over the group, from one more product with
// a constant operand.  A group's 32 values are one product of 32 deep; its
// sum is multiplied by the group's scale in f32.  So an INT4 weight is exact
// whatever x's type.
#include "layer_ops.hpp"

namespace hh {
namespace {

struct LinearArgs {
    hh_linear_args a;
    const uint16_t *scales;   // INT4: f16 bits, one per 32 values
    const uint8_t *nibbles;
    int vec;                  // bias, mul, residual and y allow 4 values at a time
};

enum WeightMode { kHalf, kInt4, kInt4Any };  // kInt4: k a multiple of 32 (a group lies in one row)

typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <int DT>
__device__ __forceinline__ f32x4 mma16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    if constexpr (DT == HH_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Values at .. at + 7 of a row of k, zeros past its end.
__device__ __forceinline__ u32x4 row8(const uint16_t *row, uint32_t at, uint32_t k) {
    if (at + 8 <= k) return *reinterpret_cast<const u32x4_any *>(row + at);
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t e = 0; e < 8; e++)
        if (at + e < k) v[e >> 1] |= (uint32_t)row[at + e] << (16 * (e & 1));
    return v;
}

// The 8 nibbles of w as 16 + nibble, in order.
template <int DT>
__device__ __forceinline__ u32x4 nibbles_to_half(uint32_t w) {
    // f16: 16 is 0x4c00 with 6 bits below the units, bf16: 0x4180 with 3
    constexpr uint32_t magic = DT == HH_BF16 ? 0x41804180u : 0x4c004c00u;
    constexpr int up = DT == HH_BF16 ? 3 : 6;
    constexpr uint32_t mask = 0x000f000fu << up;
    // a value pair 2 i, 2 i + 1 is a byte: spread it to the halves first
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t b = (w >> (8 * i)) & 255u;
        v[i] = (((b | b << 12) << up) & mask) | magic;
    }
    return v;
}

__device__ __forceinline__ float act_of(float z, int act) {
    switch (act) {
        case HH_ACT_RELU: return fmaxf(z, 0.0f) + (z != z ? z : 0.0f);
        case HH_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752440f));
        case HH_ACT_GELU_TANH: {
            // 0.5 z (1 + tanh u) = z / (1 + exp(-2 u))
            const float u = 0.79788456080286535588f * (z + 0.044715f * z * z * z);
            return z / (1.0f + __expf(-2.0f * u));
        }
        case HH_ACT_SILU: return z / (1.0f + __expf(-z));
        default: return z;
    }
}

// Writes outputs n .. n + 3 of row m from their sums.
template <int DT, int YT>
__device__ __forceinline__ void finish4(const LinearArgs &p, uint32_t m, uint32_t n, const f32x4 &sum) {
    const hh_linear_args &a = p.a;
    const uint16_t *bias = reinterpret_cast<const uint16_t *>(a.d_bias);
    const uint16_t *mul = reinterpret_cast<const uint16_t *>(a.d_mul) + m * a.mul_stride + n;
    const uint16_t *res = reinterpret_cast<const uint16_t *>(a.d_residual) + m * a.residual_stride + n;
    float v[4];
    if (p.vec && n + 4 <= a.n) {
        u32x2 b = {0, 0}, c = {0, 0}, d = {0, 0};
        if (a.d_bias) b = *reinterpret_cast<const u32x2 *>(bias + n);
        if (a.d_mul) c = *reinterpret_cast<const u32x2 *>(mul);
        if (a.d_residual) d = *reinterpret_cast<const u32x2 *>(res);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int sh = 16 * (i & 1);
            v[i] = sum[i];
            if (a.d_bias) v[i] += half_to_f32<DT>((b[i >> 1] >> sh) & 0xffffu);
            v[i] = act_of(v[i], a.activation);
            if (a.d_mul) v[i] *= half_to_f32<DT>((c[i >> 1] >> sh) & 0xffffu);
            if (a.d_residual) v[i] += half_to_f32<DT>((d[i >> 1] >> sh) & 0xffffu);
        }
        if constexpr (YT == HH_F32) {
            *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(a.d_y) + m * a.y_stride + n) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
            *reinterpret_cast<u32x2 *>(reinterpret_cast<uint16_t *>(a.d_y) + m * a.y_stride + n) =
                u32x2{f32_to_half<YT>(v[0]) | f32_to_half<YT>(v[1]) << 16, f32_to_half<YT>(v[2]) | f32_to_half<YT>(v[3]) << 16};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (n + i >= a.n) break;
        float z = sum[i];
        if (a.d_bias) z += half_to_f32<DT>(bias[n + i]);
        z = act_of(z, a.activation);
        if (a.d_mul) z *= half_to_f32<DT>(mul[i]);
        if (a.d_residual) z += half_to_f32<DT>(res[i]);
        if constexpr (YT == HH_F32)
            reinterpret_cast<float *>(a.d_y)[m * a.y_stride + n + i] = z;
        else
            reinterpret_cast<uint16_t *>(a.d_y)[m * a.y_stride + n + i] = (uint16_t)f32_to_half<YT>(z);
    }
}

// ---------------------------------------------------------------- few rows
//
// Bound by reading W once.  A workgroup takes 16 NT rows of W; its 8 waves
// take every eighth 128 columns of them, straight to registers (the next 128
// on their way while these are used), and join their sums in LDS.  x (at most
// 16 MT rows) comes from L1 / L2; its row is the products' first operand, so
// a lane's sums belong to one row of W and have one scale.
//
// A lane loads 16 bytes of nibbles, one group of its row; four lanes hold the
// row's 4 groups.  Two swaps between lanes (32 and 16 apart) turn these into
// a quarter of each group per lane, what the products take.  The nibbles of a
// word leave it in the order 0 4 1 5 2 6 3 7 (one shift and one and-or per
// pair); x's values are put in that order too.

// The 8 nibbles of w as 16 + nibble, in the order 0 4 1 5 2 6 3 7.
template <int DT>
__device__ __forceinline__ u32x4 nibbles_0415(uint32_t w) {
    constexpr uint32_t magic = DT == HH_BF16 ? 0x41804180u : 0x4c004c00u;
    constexpr int up = DT == HH_BF16 ? 3 : 6;
    constexpr uint32_t mask = 0x000f000fu << up;
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = ((4 * i > up ? w >> (4 * i - up) : w << (up - 4 * i)) & mask) | magic;
    return v;
}
__device__ __forceinline__ u32x4 order_0415(const u32x4 &x) {
    return u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                 __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}
// Lane (r, g) holds words 0..3 of group g; afterwards word g of groups 0..3.
__device__ __forceinline__ u32x4 groups_across(u32x4 w) {
    auto s = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto t = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    auto u = __builtin_amdgcn_permlane16_swap(s[0], t[0], false, false);
    auto v = __builtin_amdgcn_permlane16_swap(s[1], t[1], false, false);
    return u32x4{u[0], u[1], v[0], v[1]};
}
template <int DT>
__device__ __forceinline__ u32x4 minus24() {
    constexpr uint32_t v = DT == HH_BF16 ? 0xc1c0c1c0u : 0xce00ce00u;
    return u32x4{v, v, v, v};
}

template <int DT, int YT, int MT, int NT, bool INT4>
__global__ __launch_bounds__(512) void linear_rows_kernel(const LinearArgs p) {
    constexpr int W = INT4 ? 1 : 4;  // loads of 16 bytes per lane and 128 columns
    __shared__ __align__(16) float part[8][16 * MT][20];
    const hh_linear_args &a = p.a;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, r = lane & 15u, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * (16 * NT);
    uint64_t row[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) row[j] = min(n0 + 16 * j + r, a.n - 1);
    const uint16_t *x[MT];
#pragma unroll
    for (int t = 0; t < MT; t++)
        x[t] = reinterpret_cast<const uint16_t *>(a.d_x) + (uint64_t)min(16 * t + r, a.m - 1) * a.x_stride;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[t][j] = f32x4{0, 0, 0, 0};

    struct Cols {
        u32x4 w[NT][W];
        u32x2 s[NT];
    };
    auto fetch = [&](uint32_t k, Cols &c) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            if constexpr (INT4) {
                const uint64_t at = (row[j] * a.k + k) / 32;  // in groups
                c.w[j][0] = u32x4{0, 0, 0, 0}, c.s[j] = u32x2{0, 0};
                if (k + 32 * g < a.k) c.w[j][0] = *reinterpret_cast<const u32x4_any *>(p.nibbles + (at + g) * 16);
                if (k + 128 <= a.k) {
                    typedef u32x2 u32x2_any __attribute__((aligned(2)));
                    c.s[j] = *reinterpret_cast<const u32x2_any *>(p.scales + at);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++)
                        if (k + 32 * e < a.k) c.s[j][e >> 1] |= (uint32_t)p.scales[at + e] << (16 * (e & 1));
                }
            } else {
                const uint16_t *w = reinterpret_cast<const uint16_t *>(a.d_w) + row[j] * a.w_stride;
#pragma unroll
                for (uint32_t f = 0; f < 4; f++) c.w[j][f % W] = row8(w, k + 32 * f + 8 * g, a.k);
            }
        }
    };
    Cols cur, next;
    if (wave * 128 < a.k) fetch(wave * 128, cur);
    for (uint32_t k = wave * 128; k < a.k; k += 1024) {
        if (k + 1024 < a.k) fetch(k + 1024, next);
        if constexpr (INT4) {
#pragma unroll
            for (int j = 0; j < NT; j++) cur.w[j][0] = groups_across(cur.w[j][0]);
        }
#pragma unroll
        for (uint32_t f = 0; f < 4; f++) {
            u32x4 xf[MT];
#pragma unroll
            for (int t = 0; t < MT; t++) xf[t] = row8(x[t], k + 32 * f + 8 * g, a.k);
            if constexpr (INT4) {
                f32x4 corr[MT];
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    xf[t] = order_0415(xf[t]);
                    corr[t] = mma16<DT>(xf[t], minus24<DT>(), f32x4{0, 0, 0, 0});
                }
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const u32x4 w = nibbles_0415<DT>(cur.w[j][0][f]);
                    const float s = half_to_f32<HH_F16>((cur.s[j][f >> 1] >> (16 * (f & 1))) & 0xffffu);
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        const f32x4 q = mma16<DT>(xf[t], w, corr[t]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[t][j][e] = fmaf(s, q[e], acc[t][j][e]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int t = 0; t < MT; t++) acc[t][j] = mma16<DT>(xf[t], cur.w[j][f % W], acc[t][j]);
            }
        }
        cur = next;
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        if (j) __syncthreads();
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[wave][16 * t + 4 * g + e][r] = acc[t][j][e];
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 64 * MT; i += 512) {
            const uint32_t m = i >> 2, n = (i & 3u) * 4, at = n0 + 16 * j + n;
            if (m >= a.m || at >= a.n) continue;
            f32x4 s = *reinterpret_cast<const f32x4 *>(&part[0][m][n]);
#pragma unroll
            for (int v = 1; v < 8; v++) s += *reinterpret_cast<const f32x4 *>(&part[v][m][n]);
            finish4<DT, YT>(p, m, at, s);
        }
    }
}

// ---------------------------------------------------------------- many rows
//
// Tiles of 128 n x 128 m, 32 deep, through LDS; 4 waves of 64 x 64.  INT4
// buffers whose groups cross rows (k not a multiple of 32) give W as the sum
// of two bf16 numbers (4 + 11 bits of a value fit 8 + 8) and x, if f16, too
// (11 bits); the products of the parts are exact up to the f32 sums.

template <int DT, int YT, int MODE>
__global__ __launch_bounds__(256) void linear_tile_kernel(const LinearArgs p) {
    constexpr int PITCH = 40;  // halves: rows an odd number of 16-byte units apart
    constexpr int WP = MODE == kInt4Any ? 2 : 1, XP = MODE == kInt4Any && DT == HH_F16 ? 2 : 1;
    constexpr int MT = MODE == kInt4Any ? (int)HH_BF16 : DT;
    __shared__ __align__(16) uint16_t lw[WP][128 * PITCH], lx[XP][128 * PITCH];
    __shared__ float ls[128];
    const hh_linear_args &a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, r = lane & 15u, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * 128, m0 = blockIdx.y * 128, wn = (wave & 1u) * 64, wm = (wave >> 1) * 64;
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0, 0, 0, 0};

    u32x4 wv[2][WP], xv[2][XP];
    float sv = 0.0f;
    auto fetch = [&](uint32_t k0) {
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
            const uint32_t row = (j * 256 + tid) >> 2, k = k0 + (tid & 3u) * 8;
            const uint32_t n = n0 + row, m = m0 + row;
#pragma unroll
            for (int q = 0; q < WP; q++) wv[j][q] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < XP; q++) xv[j][q] = u32x4{0, 0, 0, 0};
            if (m < a.m) {
                const u32x4 x = row8(reinterpret_cast<const uint16_t *>(a.d_x) + (uint64_t)m * a.x_stride, k, a.k);
                if constexpr (XP == 1) {
                    xv[j][0] = x;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float f = half_to_f32<DT>((x[e >> 1] >> (16 * (e & 1))) & 0xffffu);
                        const uint32_t hi = f32_to_half<HH_BF16>(f);
                        const float rest = f - half_to_f32<HH_BF16>(hi);
                        xv[j][0][e >> 1] |= hi << (16 * (e & 1));
                        // infinities and NaN are in the first part
                        xv[j][1][e >> 1] |= (rest == rest ? f32_to_half<HH_BF16>(rest) : 0u) << (16 * (e & 1));
                    }
                }
            }
            if (n < a.n) {
                if constexpr (MODE == kHalf) {
                    wv[j][0] = row8(reinterpret_cast<const uint16_t *>(a.d_w) + (uint64_t)n * a.w_stride, k, a.k);
                } else if constexpr (MODE == kInt4) {
                    typedef uint32_t u32_any __attribute__((aligned(1)));
                    if (k < a.k)
                        wv[j][0] = nibbles_to_half<DT>(
                            *reinterpret_cast<const u32_any *>(p.nibbles + ((uint64_t)n * a.k + k) / 2));
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) {
                        if (k + e >= a.k) break;
                        const uint64_t i = (uint64_t)n * a.k + k + e;
                        const int q = (int)((p.nibbles[i / 2] >> (4 * (i & 1))) & 15u) - 8;
                        const float f = (float)q * f16_bits_to_f32(p.scales[i / 32]);
                        const uint32_t hi = f32_to_half<HH_BF16>(f);
                        const float rest = f - half_to_f32<HH_BF16>(hi);
                        wv[j][0][e >> 1] |= hi << (16 * (e & 1));
                        wv[j][WP - 1][e >> 1] |= (rest == rest ? f32_to_half<HH_BF16>(rest) : 0u) << (16 * (e & 1));
                    }
                }
            }
        }
        if constexpr (MODE == kInt4) {
            if (tid < 128)
                sv = n0 + tid < a.n && k0 < a.k
                         ? f16_bits_to_f32(p.scales[((uint64_t)(n0 + tid) * a.k + k0) / 32])
                         : 0.0f;
        }
    };

    if (a.k) fetch(0);
    for (uint32_t k0 = 0; k0 < a.k; k0 += 32) {
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < 2; j++) {
            const uint32_t at = ((j * 256 + tid) >> 2) * PITCH + (tid & 3u) * 8;
#pragma unroll
            for (int q = 0; q < WP; q++) *reinterpret_cast<u32x4 *>(&lw[q][at]) = wv[j][q];
#pragma unroll
            for (int q = 0; q < XP; q++) *reinterpret_cast<u32x4 *>(&lx[q][at]) = xv[j][q];
        }
        if (MODE == kInt4 && tid < 128) ls[tid] = sv;
        __syncthreads();
        if (k0 + 32 < a.k) fetch(k0 + 32);
#pragma unroll
        for (int qx = 0; qx < XP; qx++) {
            u32x4 x[4];
            f32x4 corr[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[j] = *reinterpret_cast<const u32x4 *>(&lx[qx][(wm + 16 * j + r) * PITCH + 8 * g]);
                if constexpr (MODE == kInt4) {
                    constexpr uint32_t m24 = DT == HH_BF16 ? 0xc1c0c1c0u : 0xce00ce00u;  // -24
                    corr[j] = mma16<DT>(u32x4{m24, m24, m24, m24}, x[j], f32x4{0, 0, 0, 0});
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f32x4 s;
                if constexpr (MODE == kInt4) s = *reinterpret_cast<const f32x4 *>(&ls[wn + 16 * i + 4 * g]);
#pragma unroll
                for (int qw = 0; qw < WP; qw++) {
                    const u32x4 w = *reinterpret_cast<const u32x4 *>(&lw[qw][(wn + 16 * i + r) * PITCH + 8 * g]);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if constexpr (MODE == kInt4) {
                            const f32x4 part = mma16<DT>(w, x[j], corr[j]);
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(s[e], part[e], acc[i][j][e]);
                        } else {
                            acc[i][j] = mma16<MT>(w, x[j], acc[i][j]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t m = m0 + wm + 16 * j + r;
        if (m >= a.m) continue;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t n = n0 + wn + 16 * i + 4 * g;
            if (n < a.n) finish4<DT, YT>(p, m, n, acc[i][j]);
        }
    }
}

template <int DT, int YT, int MT, bool INT4>
hipError_t launch_rows(const LinearArgs &p, hipStream_t s) {
    const uint32_t tiles = (p.a.n + 15) / 16;
    if (tiles >= 512)
        hipLaunchKernelGGL((linear_rows_kernel<DT, YT, MT, 2, INT4>), dim3((tiles + 1) / 2), dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((linear_rows_kernel<DT, YT, MT, 1, INT4>), dim3(tiles), dim3(512), 0, s, p);
    return hipGetLastError();
}

template <int DT, int YT>
hipError_t launch_linear(const LinearArgs &p, hipStream_t s) {
    const hh_linear_args &a = p.a;
    if (a.m <= 64 && (a.w_dtype != HH_INT4 || a.k % 32 == 0)) {
        const int rows = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
        return a.w_dtype == HH_INT4 ? (rows == 1   ? launch_rows<DT, YT, 1, true>(p, s)
                                       : rows == 2 ? launch_rows<DT, YT, 2, true>(p, s)
                                                   : launch_rows<DT, YT, 4, true>(p, s))
                                    : (rows == 1   ? launch_rows<DT, YT, 1, false>(p, s)
                                       : rows == 2 ? launch_rows<DT, YT, 2, false>(p, s)
                                                   : launch_rows<DT, YT, 4, false>(p, s));
    }
    auto kernel = a.w_dtype != HH_INT4 ? linear_tile_kernel<DT, YT, kHalf>
                  : a.k % 32 == 0      ? linear_tile_kernel<DT, YT, kInt4>
                                       : linear_tile_kernel<DT, YT, kInt4Any>;
    hipLaunchKernelGGL(kernel, dim3((a.n + 127) / 128, (a.m + 127) / 128), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace
}  // namespace hh

extern "C" int32_t hh_linear(hh_context *ctx, const hh_linear_args *a, void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    if (a->dtype != HH_F16 && a->dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (a->w_dtype != a->dtype && a->w_dtype != HH_INT4) return HH_ERR_UNSUPPORTED;
    if (a->y_dtype != a->dtype && a->y_dtype != HH_F32) return HH_ERR_UNSUPPORTED;
    if (a->activation < HH_ACT_NONE || a->activation > HH_ACT_SILU) return HH_ERR_UNSUPPORTED;
    if (a->m >= 1u << 23 || a->n >= 1u << 31 || a->k >= 1u << 31) return HH_ERR_INVALID_ARGUMENT;
    if (a->m == 0 || a->n == 0) return HH_OK;
    const bool int4 = a->w_dtype == HH_INT4;
    if (!a->d_y || (a->k && (!a->d_x || !a->d_w))) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)a->d_x | (uintptr_t)a->d_w | (uintptr_t)a->d_bias | (uintptr_t)a->d_mul | (uintptr_t)a->d_residual) & 1u)
        return HH_ERR_INVALID_ARGUMENT;
    if ((uintptr_t)a->d_y & (a->y_dtype == HH_F32 ? 3u : 1u)) return HH_ERR_INVALID_ARGUMENT;
    if (a->x_stride < a->k || a->y_stride < a->n || (!int4 && a->w_stride < a->k) ||
        (a->d_mul && a->mul_stride < a->n) || (a->d_residual && a->residual_stride < a->n))
        return HH_ERR_INVALID_ARGUMENT;
    hh::LinearArgs p = {};
    p.a = *a;
    if (int4) {
        const uint64_t count = (uint64_t)a->n * a->k;
        if (a->w_bytes < (count + 31) / 32 * 2 + (count + 1) / 2) return HH_ERR_UNEXPECTED_EOF;
        p.scales = reinterpret_cast<const uint16_t *>(a->d_w);
        p.nibbles = reinterpret_cast<const uint8_t *>(a->d_w) + (count + 31) / 32 * 2;
    }
    const uintptr_t side = (uintptr_t)a->d_bias | (uintptr_t)a->d_mul | (uintptr_t)a->d_residual;
    p.vec = !(side & 7u) && !((uintptr_t)a->d_y & (a->y_dtype == HH_F32 ? 15u : 7u)) && !(a->y_stride & 3u) &&
            !(a->d_mul && (a->mul_stride & 3u)) && !(a->d_residual && (a->residual_stride & 3u));
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hipError_t e;
    if (a->dtype == HH_BF16)
        e = a->y_dtype == HH_F32 ? hh::launch_linear<HH_BF16, HH_F32>(p, s) : hh::launch_linear<HH_BF16, HH_BF16>(p, s);
    else
        e = a->y_dtype == HH_F32 ? hh::launch_linear<HH_F16, HH_F32>(p, s) : hh::launch_linear<HH_F16, HH_F16>(p, s);
    return hh::from_hip(e);
}
