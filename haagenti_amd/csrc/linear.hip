// y = act(x W^T + bias) * mul + residual (hh_linear, include/haagenti_hip.h).
//
// Three routes: few rows of x (W straight to registers), many rows in tiles
// copied straight to LDS where the layout is aligned, and tiles through
// registers for any other layout and for INT4.  The tiles put W's rows on the
// first operand of the matrix instructions and x's on the second, so a lane
// ends with 4 consecutive outputs n of one row m; bias, mul, residual and y
// move 4 values at a time on every route.
//
// INT4 weights stay integers: nibbles become the 16-bit numbers 16..31 by
// shifts and ors (exact in f16 and bf16), and the offset of 24 goes into the
// accumulator's start, -24 sum(x) over the group, from one more product with
// a constant operand.  A group's 32 values are one product of 32 deep; its
// sum is multiplied by the group's scale in f32.  So an INT4 weight is exact
// whatever x's type; what f32 rounds are sums of up to 31 |x| and 24 |x| where
// the weight's own integer is at most 8.
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

// __expf is the hardware's power of two of x log2(e): off by 2^-23 of itself
// and by 2^-24 |x|, so by less than 2^-20 |z| in what SiLU and GELU make of it.
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

// What the epilogue of outputs n .. n + 3 of row m reads, where 4 values move
// at a time.
struct Side {
    u32x2 bias, mul, res;
};
__device__ __forceinline__ bool whole4(const LinearArgs &p, uint32_t n) { return p.vec && n + 4 <= p.a.n; }
__device__ __forceinline__ Side load_side(const LinearArgs &p, uint32_t m, uint32_t n) {
    const hh_linear_args &a = p.a;
    Side s = {{0, 0}, {0, 0}, {0, 0}};
    if (a.d_bias) s.bias = *reinterpret_cast<const u32x2 *>(reinterpret_cast<const uint16_t *>(a.d_bias) + n);
    if (a.d_mul) s.mul = *reinterpret_cast<const u32x2 *>(reinterpret_cast<const uint16_t *>(a.d_mul) + m * a.mul_stride + n);
    if (a.d_residual)
        s.res = *reinterpret_cast<const u32x2 *>(reinterpret_cast<const uint16_t *>(a.d_residual) + m * a.residual_stride + n);
    return s;
}
template <int DT, int YT>
__device__ __forceinline__ void finish_whole4(const LinearArgs &p, uint32_t m, uint32_t n, const f32x4 &sum, const Side &s) {
    const hh_linear_args &a = p.a;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int sh = 16 * (i & 1);
        v[i] = sum[i];
        if (a.d_bias) v[i] += half_to_f32<DT>((s.bias[i >> 1] >> sh) & 0xffffu);
        v[i] = act_of(v[i], a.activation);
        if (a.d_mul) v[i] *= half_to_f32<DT>((s.mul[i >> 1] >> sh) & 0xffffu);
        if (a.d_residual) v[i] += half_to_f32<DT>((s.res[i >> 1] >> sh) & 0xffffu);
    }
    if constexpr (YT == HH_F32) {
        *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(a.d_y) + m * a.y_stride + n) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
        *reinterpret_cast<u32x2 *>(reinterpret_cast<uint16_t *>(a.d_y) + m * a.y_stride + n) =
            u32x2{f32_to_half<YT>(v[0]) | f32_to_half<YT>(v[1]) << 16, f32_to_half<YT>(v[2]) | f32_to_half<YT>(v[3]) << 16};
    }
}

// Writes outputs n .. n + 3 of row m from their sums.
template <int DT, int YT>
__device__ __forceinline__ void finish4(const LinearArgs &p, uint32_t m, uint32_t n, const f32x4 &sum) {
    const hh_linear_args &a = p.a;
    if (whole4(p, n)) {
        finish_whole4<DT, YT>(p, m, n, sum, load_side(p, m, n));
        return;
    }
#pragma unroll 1
    for (uint32_t i = 0; i < 4 && n + i < a.n; i++) {
        float z = i == 0 ? sum[0] : i == 1 ? sum[1] : i == 2 ? sum[2] : sum[3];
        if (a.d_bias) z += half_to_f32<DT>(reinterpret_cast<const uint16_t *>(a.d_bias)[n + i]);
        z = act_of(z, a.activation);
        if (a.d_mul) z *= half_to_f32<DT>(reinterpret_cast<const uint16_t *>(a.d_mul)[m * a.mul_stride + n + i]);
        if (a.d_residual) z += half_to_f32<DT>(reinterpret_cast<const uint16_t *>(a.d_residual)[m * a.residual_stride + n + i]);
        if constexpr (YT == HH_F32)
            reinterpret_cast<float *>(a.d_y)[m * a.y_stride + n + i] = z;
        else
            reinterpret_cast<uint16_t *>(a.d_y)[m * a.y_stride + n + i] = (uint16_t)f32_to_half<YT>(z);
    }
}

// ---------------------------------------------------------------- few rows
//
// Bound by reading W once: a row of 4096 x 4096 in bf16 7.8 us (4.3 TB/s of W,
// 5.4 at the copy's 6.2), of 14336 x 4096 26 us, of 8192 x 8192 28 us; INT4 of
// 14336 x 4096 16 us for 1 row, 17.5 for 8 (5.4 at the copy's rate: without
// the loads of x and of the scales it takes 12, without the products as long
// as with them).  A workgroup takes 16 NT rows of W; its KW
// waves take every KW-th 128 columns of them, straight to registers (the next
// ones on their way while these are used), and join their sums in LDS.  x (at most
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

template <int DT, int YT, int MT, int NT, int KW, bool INT4>
__global__ __launch_bounds__(64 * KW) void linear_rows_kernel(const LinearArgs p) {
    constexpr uint32_t STEP = 128 * KW;                       // columns between a wave's 128s
    constexpr int W = INT4 ? 1 : 4;                           // loads of 16 bytes per lane and 128 columns
    constexpr int AHEAD = 2;       // 128s of W in registers, one in use
    constexpr bool XA = MT <= 2;                              // x's values one 128 ahead, where registers allow
    __shared__ __align__(16) float part[KW][16 * MT][20];
    const hh_linear_args &a = p.a;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = lane & 15u, g = lane >> 4, n0 = blockIdx.x * (16 * NT);
    uint64_t row[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) row[j] = min(n0 + 16 * j + r, a.n - 1);
    // INT4: the lane's group of a row's first four, the row's scales; else
    // its first 8 columns
    const uint8_t *nib[NT];
    const uint16_t *scl[NT], *w[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        nib[j] = p.nibbles + row[j] * (a.k / 2) + g * 16, scl[j] = p.scales + row[j] * (a.k / 32);
        w[j] = reinterpret_cast<const uint16_t *>(a.d_w) + row[j] * a.w_stride + 8 * g;
    }
    const uint16_t *x[MT];
#pragma unroll
    for (int t = 0; t < MT; t++)
        x[t] = reinterpret_cast<const uint16_t *>(a.d_x) + (uint64_t)min(16 * t + r, a.m - 1) * a.x_stride;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[t][j] = f32x4{0, 0, 0, 0};

    // W's 128s go around AHEAD sets of registers, x's around two; x's are
    // loaded first, as loads come back in order.
    struct Cols {
        u32x4 w[NT][W];
        u32x2 s[NT];
    };
    auto fetch = [&](uint32_t k, Cols &c) {
        typedef u32x2 u32x2_any __attribute__((aligned(2)));
#pragma unroll
        for (int j = 0; j < NT; j++) {
            if constexpr (INT4) {
                c.w[j][0] = *reinterpret_cast<const u32x4_any *>(nib[j] + k / 2);
                c.s[j] = *reinterpret_cast<const u32x2_any *>(scl[j] + k / 32);
            } else {
#pragma unroll
                for (uint32_t f = 0; f < 4; f++) c.w[j][f % W] = *reinterpret_cast<const u32x4_any *>(w[j] + k + 32 * f);
            }
        }
    };
    auto fetch_x = [&](uint32_t k, u32x4 (&v)[MT][4]) {
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (uint32_t f = 0; f < 4; f++) v[t][f] = *reinterpret_cast<const u32x4_any *>(x[t] + k + 32 * f + 8 * g);
    };
    // one group of 32 columns: word(j) and scale(j) of W's rows in INT4
    auto group = [&](const u32x4 (&xu)[MT], auto word, auto scale) {
        u32x4 xf[MT];
        f32x4 corr[MT];
#pragma unroll
        for (int t = 0; t < MT; t++) {
            xf[t] = order_0415(xu[t]);
            corr[t] = mma16<DT>(xf[t], minus24<DT>(), f32x4{0, 0, 0, 0});
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const u32x4 v = nibbles_0415<DT>(word(j));
            const float s = half_to_f32<HH_F16>(scale(j));
#pragma unroll
            for (int t = 0; t < MT; t++) {
                const f32x4 q = mma16<DT>(xf[t], v, corr[t]);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[t][j][e] = fmaf(s, q[e], acc[t][j][e]);
            }
        }
    };
    auto multiply = [&](Cols &c, const u32x4 (&xu)[MT][4]) {
        if constexpr (INT4) {
#pragma unroll
            for (int j = 0; j < NT; j++) c.w[j][0] = groups_across(c.w[j][0]);
        }
#pragma unroll
        for (uint32_t f = 0; f < 4; f++) {
            u32x4 xf[MT];
#pragma unroll
            for (int t = 0; t < MT; t++) xf[t] = xu[t][f];
            if constexpr (INT4) {
                group(xf, [&](int j) { return c.w[j][0][f]; },
                      [&](int j) { return (c.s[j][f >> 1] >> (16 * (f & 1))) & 0xffffu; });
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int t = 0; t < MT; t++) acc[t][j] = mma16<DT>(xf[t], c.w[j][f % W], acc[t][j]);
            }
        }
    };
    const uint32_t whole = a.k / 128 * 128;
    if (wave * 128 < whole) {
        Cols cols[AHEAD];
        u32x4 xv[2][MT][4];
        if (XA) fetch_x(wave * 128, xv[0]);
#pragma unroll
        for (int u = 0; u < AHEAD; u++) if (wave * 128 + u * STEP < whole) fetch(wave * 128 + u * STEP, cols[u]);
#pragma unroll 1
        for (uint32_t k0 = wave * 128; k0 < whole; k0 += AHEAD * STEP) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const uint32_t k = k0 + u * STEP;
                if (k >= whole) break;
                if (!XA)
                    fetch_x(k, xv[0]);
                else if (k + STEP < whole)
                    fetch_x(k + STEP, xv[(u + 1) & 1]);
                multiply(cols[u], xv[XA ? u & 1 : 0]);
                if (k + AHEAD * STEP < whole) fetch(k + AHEAD * STEP, cols[u]);
            }
        }
    }
    // what is left of the columns, 32 at a time, the next wave's turn
    if (whole < a.k && wave == whole / 128 % KW) {
#pragma unroll 1
        for (uint32_t k = whole; k < a.k; k += 32) {
            u32x4 xf[MT];
#pragma unroll
            for (int t = 0; t < MT; t++) xf[t] = row8(x[t], k + 8 * g, a.k);
            if constexpr (INT4) {
                typedef uint32_t u32_any __attribute__((aligned(2)));
                group(xf, [&](int j) { return *reinterpret_cast<const u32_any *>(nib[j] + k / 2 + g * 4 - g * 16); },
                      [&](int j) { return (uint32_t)scl[j][k / 32]; });
            } else {
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const u32x4 wf = row8(w[j] - 8 * g, k + 8 * g, a.k);
#pragma unroll
                    for (int t = 0; t < MT; t++) acc[t][j] = mma16<DT>(xf[t], wf, acc[t][j]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        if (j) __syncthreads();
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[wave][16 * t + 4 * g + e][r] = acc[t][j][e];
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 64 * MT; i += 64 * KW) {
            const uint32_t m = i >> 2, n = (i & 3u) * 4, at = n0 + 16 * j + n;
            if (m >= a.m || at >= a.n) continue;
            f32x4 s = *reinterpret_cast<const f32x4 *>(&part[0][m][n]);
#pragma unroll
            for (int v = 1; v < KW; v++) s += *reinterpret_cast<const f32x4 *>(&part[v][m][n]);
            finish4<DT, YT>(p, m, at, s);
        }
    }
}

// ---------------------------------------------------------------- many rows, any layout
//
// Tiles of S n x S m, 64 deep, through registers and LDS; 4 waves.  The next
// 64 columns are loaded while these are multiplied.  INT4 buffers whose groups
// cross rows (k not a multiple of 32) give W as the sum of two bf16 numbers
// (4 + 11 bits of a value fit 8 + 8) and x, if f16, too (11 bits); the
// products of the parts are exact up to the f32 sums.

// Splits of k: steps of 64 each takes, sums to `partial`.
struct Split {
    uint32_t steps;
    float *partial;  // [split][m][n rounded up to 4], or null: one split, y itself
};

// A split's sums of outputs n .. n + 3 of row m.  Rows of the sums are whole
// groups of 4, so that all are written and read 16 bytes at a time.
__device__ __forceinline__ uint32_t partial_row(const LinearArgs &p) { return (p.a.n + 3) / 4 * 4; }
__device__ __forceinline__ void store_partial(const LinearArgs &p, const Split &split, uint32_t index, uint32_t m, uint32_t n,
                                              const f32x4 &v) {
    *reinterpret_cast<f32x4 *>(split.partial + ((uint64_t)index * p.a.m + m) * partial_row(p) + n) = v;
}

// f as the sum of two bf16 numbers, e-th of 8 each; what is not finite is in
// the first.
__device__ __forceinline__ void split_bf16(float f, int e, u32x4 &hi, u32x4 &lo) {
    const uint32_t h = f32_to_half<HH_BF16>(f);
    const float rest = f - half_to_f32<HH_BF16>(h);
    hi[e >> 1] |= h << (16 * (e & 1));
    lo[e >> 1] |= (fabsf(rest) < __builtin_inff() ? f32_to_half<HH_BF16>(rest) : 0u) << (16 * (e & 1));
}

template <int DT, int YT, int MODE, int S>
__global__ __launch_bounds__(256) void linear_tile_kernel(const LinearArgs p, const Split split) {
    constexpr int H = S / 2, F = H / 16, P = S / 32;  // a wave's side, its tiles, pieces of 8 values per thread
    constexpr int PITCH = 72;                         // halves: rows an odd number of 16-byte units apart
    constexpr int WP = MODE == kInt4Any ? 2 : 1, XP = MODE == kInt4Any && DT == HH_F16 ? 2 : 1;
    constexpr int MT = MODE == kInt4Any ? (int)HH_BF16 : DT;
    __shared__ __align__(16) uint16_t lw[WP][S * PITCH], lx[XP][S * PITCH];
    __shared__ __align__(16) float ls[2][S];
    const hh_linear_args &a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, r = lane & 15u, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * S, m0 = blockIdx.y * S, wn = (wave & 1u) * H, wm = (wave >> 1) * H;
    const uint32_t k1 = (uint32_t)min((uint64_t)a.k, (uint64_t)(blockIdx.z + 1) * split.steps * 64), kb = blockIdx.z * split.steps * 64;
    f32x4 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < F; j++) acc[i][j] = f32x4{0, 0, 0, 0};

    u32x4 wv[P][WP], xv[P][XP];
    uint32_t sv = 0;
    auto fetch = [&](uint32_t k0) {
#pragma unroll
        for (uint32_t j = 0; j < P; j++) {
            const uint32_t row = (j * 256 + tid) >> 3, k = k0 + (tid & 7u) * 8;
            const uint32_t n = n0 + row, m = m0 + row;
#pragma unroll
            for (int q = 0; q < WP; q++) wv[j][q] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < XP; q++) xv[j][q] = u32x4{0, 0, 0, 0};
            if (m < a.m) xv[j][0] = row8(reinterpret_cast<const uint16_t *>(a.d_x) + (uint64_t)m * a.x_stride, k, k1);
            if (n < a.n) {
                if constexpr (MODE == kHalf) {
                    wv[j][0] = row8(reinterpret_cast<const uint16_t *>(a.d_w) + (uint64_t)n * a.w_stride, k, k1);
                } else if constexpr (MODE == kInt4) {
                    typedef uint32_t u32_any __attribute__((aligned(1)));
                    if (k < k1) wv[j][0][0] = *reinterpret_cast<const u32_any *>(p.nibbles + ((uint64_t)n * a.k + k) / 2);
                } else {
                    // 8 nibbles: 4 bytes, or 5 from the middle of one; at most two groups
                    const uint64_t i = (uint64_t)n * a.k + k;
                    const uint32_t count = k < k1 ? min(k1 - k, 8u) : 0u, odd = (uint32_t)(i & 1);
                    if (count) {
                        uint64_t bytes = 0;
#pragma unroll
                        for (uint32_t e = 0; e < 5; e++)
                            if (2 * e < count + odd) bytes |= (uint64_t)p.nibbles[i / 2 + e] << (8 * e);
                        bytes >>= 4 * odd;
                        const float s0 = f16_bits_to_f32(p.scales[i / 32]), s1 = f16_bits_to_f32(p.scales[(i + count - 1) / 32]);
#pragma unroll
                        for (uint32_t e = 0; e < 8; e++) {
                            if (e >= count) break;
                            const int q = (int)((uint32_t)(bytes >> (4 * e)) & 15u) - 8;
                            split_bf16((float)q * ((i + e) / 32 == i / 32 ? s0 : s1), e, wv[j][0], wv[j][WP - 1]);
                        }
                    }
                }
            }
        }
        if constexpr (MODE == kInt4) {
            const uint32_t row = tid % S, k = k0 + tid / S * 32;  // 2 S scales
            if (tid < 2 * S) sv = n0 + row < a.n && k < k1 ? p.scales[((uint64_t)(n0 + row) * a.k + k) / 32] : 0u;
        }
    };
    // what is done to the values on their way to LDS waits until they are here
    auto stage = [&]() {
#pragma unroll
        for (uint32_t j = 0; j < P; j++) {
            const uint32_t at = ((j * 256 + tid) >> 3) * PITCH + (tid & 7u) * 8;
            if constexpr (MODE == kInt4) {
                *reinterpret_cast<u32x4 *>(&lw[0][at]) = nibbles_0415<DT>(wv[j][0][0]);
                *reinterpret_cast<u32x4 *>(&lx[0][at]) = order_0415(xv[j][0]);
            } else {
                if constexpr (XP == 2) {
                    const u32x4 x = xv[j][0];
                    xv[j][0] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        split_bf16(half_to_f32<DT>((x[e >> 1] >> (16 * (e & 1))) & 0xffffu), e, xv[j][0], xv[j][XP - 1]);
                }
#pragma unroll
                for (int q = 0; q < WP; q++) *reinterpret_cast<u32x4 *>(&lw[q][at]) = wv[j][q];
#pragma unroll
                for (int q = 0; q < XP; q++) *reinterpret_cast<u32x4 *>(&lx[q][at]) = xv[j][q];
            }
        }
        if (MODE == kInt4 && tid < 2 * S) ls[tid / S][tid % S] = f16_bits_to_f32(sv);
    };

    if (kb < k1) fetch(kb);
    for (uint32_t k0 = kb; k0 < k1; k0 += 64) {
        __syncthreads();
        stage();
        __syncthreads();
        if (k0 + 64 < k1) fetch(k0 + 64);
#pragma unroll
        for (int f = 0; f < 2; f++)
#pragma unroll
            for (int qx = 0; qx < XP; qx++) {
                u32x4 x[F];
                f32x4 corr[F];
#pragma unroll
                for (int j = 0; j < F; j++) {
                    x[j] = *reinterpret_cast<const u32x4 *>(&lx[qx][(wm + 16 * j + r) * PITCH + 32 * f + 8 * g]);
                    if constexpr (MODE == kInt4) corr[j] = mma16<DT>(minus24<DT>(), x[j], f32x4{0, 0, 0, 0});
                }
#pragma unroll
                for (int i = 0; i < F; i++) {
                    f32x4 s;
                    if constexpr (MODE == kInt4) s = *reinterpret_cast<const f32x4 *>(&ls[f][wn + 16 * i + 4 * g]);
#pragma unroll
                    for (int qw = 0; qw < WP; qw++) {
                        const u32x4 w = *reinterpret_cast<const u32x4 *>(&lw[qw][(wn + 16 * i + r) * PITCH + 32 * f + 8 * g]);
#pragma unroll
                        for (int j = 0; j < F; j++) {
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
    for (int j = 0; j < F; j++) {
        const uint32_t m = m0 + wm + 16 * j + r;
        if (m >= a.m) continue;
#pragma unroll
        for (int i = 0; i < F; i++) {
            const uint32_t n = n0 + wn + 16 * i + 4 * g;
            if (n >= a.n) continue;
            if (split.partial)
                store_partial(p, split, blockIdx.z, m, n, acc[i][j]);
            else
                finish4<DT, YT>(p, m, n, acc[i][j]);
        }
    }
}

// ---------------------------------------------------------------- many rows, aligned
//
// Tiles of TN n x TM m, 64 deep, copied straight to LDS, two of them in turn:
// the next tile's copies are under way while this one is multiplied, one
// barrier per tile.  The buffers are four arrays of their own, so that the
// compiler sees which of them a copy writes and waits for it at the barrier
// only.  A row of 64 values is 8 pieces of 16 bytes; row r's piece c lies at
// place c ^ (r & 7), so that rows read together lie in different banks (the
// copy's lanes choose their source piece accordingly: LDS is written in lane
// order).  Rows past the matrices repeat the last one.  Bound by LDS and the
// matrix pipes alike: at 256 x 256 a tile's reads (192 KiB by 8 waves of
// 128 x 64) and copies (64 KiB) take as long as its products.  bf16 4096 x
// 8192 x 8192 takes 413 us (1330 TFLOP/s; 0.82 of the library's product),
// 2048 x 14336 x 4096 221 (1090; 0.78), with SiLU and a product 239 to 280 by
// what the caches and clocks hold, 512 x 4096 x 14336 70 (860; the library's 78).
//
// Tiles are numbered down the rows of x, and consecutive ones go to one XCD,
// whose L2 then serves W's panel to all of them.

template <int ROWS, int T>
__device__ __forceinline__ void tile_offsets(uint32_t stride, uint32_t rows, uint32_t (&off)[ROWS * 8 / T]) {
#pragma unroll
    for (int j = 0; j < ROWS * 8 / T; j++) {
        const uint32_t slot = j * T + threadIdx.x, row = slot >> 3, piece = (slot & 7u) ^ (row & 7u);
        off[j] = (min(row, rows - 1) * stride + piece * 8) * 2;
    }
}
template <int ROWS, int T, typename Source>
__device__ __forceinline__ void tile_copy(const Source &from, uint32_t at, const uint32_t (&off)[ROWS * 8 / T], uint16_t *lds,
                                          uint32_t wave) {
#if defined(__HIP_DEVICE_COMPILE__)  // 16-byte copies exist in the device's pass only
#pragma unroll
    for (int j = 0; j < ROWS * 8 / T; j++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            from, (__attribute__((address_space(3))) void *)(lds + (j * T + wave * 64) * 8), 16, off[j], at, 0, 0);
#endif
}

template <int DT, int YT, int TN, int TM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM) void linear_large_kernel(const LinearArgs p, const Split split) {
    constexpr int T = 64 * WN * WM, NI = TN / WN / 16, MI = TM / WM / 16;
    __shared__ __align__(16) uint16_t lw0[TN * 64], lw1[TN * 64], lx0[TM * 64], lx1[TM * 64];
    const hh_linear_args &a = p.a;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = lane & 15u, g = lane >> 4;
    const uint32_t mt = (a.m + TM - 1) / TM, share = gridDim.x / 8, rest = gridDim.x % 8, xcd = blockIdx.x % 8;
    const uint32_t id = xcd * share + min(xcd, rest) + blockIdx.x / 8;
    const uint32_t n0 = id / mt * TN, m0 = id % mt * TM, wn = wave % WN * (TN / WN), wm = wave / WN * (TM / WM);
    const uint32_t k0 = blockIdx.y * split.steps * 64, k1 = min(a.k, k0 + split.steps * 64);
    f32x4 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < MI; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    uint32_t ow[TN * 8 / T], ox[TM * 8 / T];
    tile_offsets<TN, T>((uint32_t)a.w_stride, a.n - n0, ow);
    tile_offsets<TM, T>((uint32_t)a.x_stride, a.m - m0, ox);
    // offsets stay inside the matrices (rows are clamped): no size limit here
    const auto w = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t *>(reinterpret_cast<const uint16_t *>(a.d_w) + n0 * a.w_stride), 0, 0xffffffffu, 0x00027000);
    const auto x = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t *>(reinterpret_cast<const uint16_t *>(a.d_x) + m0 * a.x_stride), 0, 0xffffffffu, 0x00027000);
    auto copy = [&](uint16_t *lw, uint16_t *lx, uint32_t k) {
        tile_copy<TN, T>(w, 2 * k, ow, lw, wave);
        tile_copy<TM, T>(x, 2 * k, ox, lx, wave);
    };
    auto multiply = [&](const uint16_t *lw, const uint16_t *lx) {
#pragma unroll
        for (uint32_t f = 0; f < 2; f++) {
            const uint32_t piece = ((g + 4 * f) ^ (r & 7u)) * 8;
            u32x4 wf[NI], xf[MI];
#pragma unroll
            for (int j = 0; j < MI; j++) xf[j] = *reinterpret_cast<const u32x4 *>(&lx[(wm + 16 * j + r) * 64 + piece]);
#pragma unroll
            for (int i = 0; i < NI; i++) wf[i] = *reinterpret_cast<const u32x4 *>(&lw[(wn + 16 * i + r) * 64 + piece]);
#pragma unroll
            for (int i = 0; i < NI; i++)
#pragma unroll
                for (int j = 0; j < MI; j++) acc[i][j] = mma16<DT>(wf[i], xf[j], acc[i][j]);
        }
        // the first reads, then one between every two products, then the
        // products that are left
        constexpr int reads = 2 * (NI + MI), lead = MI + 2;
        __builtin_amdgcn_sched_group_barrier(0x100, lead, 0);
#pragma unroll
        for (int i = 0; i < reads - lead; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 2 * NI * MI - 2 * (reads - lead), 0);
    };
    // a barrier waits for the copies into the buffers that are read after it,
    // and for the reads of the ones that are copied to after it
    copy(lw0, lx0, k0);
    for (uint32_t k = k0; k < k1; k += 128) {
        __syncthreads();
        if (k + 64 < k1) {
            copy(lw1, lx1, k + 64);
        } else {
            // an odd number of steps ends with one of zeros
            for (uint32_t i = threadIdx.x; i < TN * 8; i += T) reinterpret_cast<u32x4 *>(lw1)[i] = u32x4{0, 0, 0, 0};
            for (uint32_t i = threadIdx.x; i < TM * 8; i += T) reinterpret_cast<u32x4 *>(lx1)[i] = u32x4{0, 0, 0, 0};
        }
        multiply(lw0, lx0);
        __syncthreads();
        if (k + 128 < k1) copy(lw0, lx0, k + 128);
        multiply(lw1, lx1);
    }
    // Sums go out by way of LDS, 16 rows x 64 columns of each wave at a time,
    // so that a wave writes pieces of rows; a row's groups of 4 lie at q ^ row.
    constexpr int Q = 16;
    f32x4 *own = reinterpret_cast<f32x4 *>(TN >= TM ? lw0 : lx0) + wave * 16 * Q;
    static_assert(WN * WM * 16 * Q * 16 <= (TN >= TM ? TN : TM) * 128, "every wave's piece fits one buffer");
#pragma unroll
    for (int j = 0; j < MI; j++)
#pragma unroll
        for (int h = 0; h < NI / 4; h++) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) own[r * Q + ((4 * i + g) ^ r)] = acc[4 * h + i][j];
            __syncthreads();
            // what the epilogue reads first, all at once
            Side side[4];
            uint32_t n = n0 + wn + 64 * h + r * 4, m = m0 + wm + 16 * j + g;
            asm volatile("" : "+v"(n), "+v"(m));  // no addresses of later pieces in registers meanwhile
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (!split.partial && m + 4 * c < a.m && whole4(p, n)) side[c] = load_side(p, m + 4 * c, n);
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
                const uint32_t row = 4 * c + g, at = m + 4 * c;
                const f32x4 v = own[row * Q + (r ^ row)];
                auto pick = [&](u32x2 Side::*f) {
                    const u32x2 lo = c & 1 ? side[1].*f : side[0].*f, hi = c & 1 ? side[3].*f : side[2].*f;
                    return c & 2 ? hi : lo;
                };
                const Side sd = {pick(&Side::bias), pick(&Side::mul), pick(&Side::res)};
                if (at >= a.m || n >= a.n) continue;
                if (split.partial) {
                    store_partial(p, split, blockIdx.y, at, n, v);
                } else if (whole4(p, n)) {
                    finish_whole4<DT, YT>(p, at, n, v, sd);
                } else {
                    finish4<DT, YT>(p, at, n, v);
                }
            }
        }
}

// The splits' sums, in order, and the epilogue.
template <int DT, int YT>
__global__ __launch_bounds__(256) void linear_join_kernel(const LinearArgs p, const float *partial, uint32_t splits) {
    const hh_linear_args &a = p.a;
    const uint32_t quads = (a.n + 3) / 4;
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (uint64_t)a.m * quads) return;
    const uint32_t m = (uint32_t)(i / quads), n = (uint32_t)(i % quads) * 4;
    const uint64_t step = (uint64_t)a.m * quads * 4;
    const float *at = partial + (uint64_t)m * quads * 4 + n;
    f32x4 s = {0, 0, 0, 0};
#pragma unroll 8
    for (uint32_t j = 0; j < splits; j++) s += *reinterpret_cast<const f32x4 *>(at + j * step);
    finish4<DT, YT>(p, m, n, s);
}

// 8 waves to a workgroup's rows while there are at most two workgroups to a
// CU, else 4 (all workgroups resident at once: a row of 8192 x 8192 28 us
// against 35); two tiles of W's rows where x's values are what a wave loads
// most.
template <int DT, int YT, int MT, bool INT4>
hipError_t launch_rows(const LinearArgs &p, int cus, hipStream_t s) {
    const uint32_t tiles = (p.a.n + 15) / 16;
    constexpr int NT = INT4 || MT > 1 ? 2 : 1;
    if (tiles <= 2 * (uint32_t)cus)
        hipLaunchKernelGGL((linear_rows_kernel<DT, YT, MT, 1, 8, INT4>), dim3(tiles), dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((linear_rows_kernel<DT, YT, MT, NT, 4, INT4>), dim3((tiles + NT - 1) / NT), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <int DT, int YT, int TN, int TM, int WN, int WM>
void launch_tiles(const LinearArgs &p, const Split &split, uint32_t splits, hipStream_t s) {
    const uint32_t tiles = ((p.a.n + TN - 1) / TN) * ((p.a.m + TM - 1) / TM);
    hipLaunchKernelGGL((linear_large_kernel<DT, YT, TN, TM, WN, WM>), dim3(tiles, splits), dim3(64 * WN * WM), 0, s, p, split);
}

// A tile shape: workgroups to a CU, microseconds per 64 columns of k with all
// of them and with one alone.
struct Shape {
    uint32_t n, m, per_cu;
    double us, alone;
};
struct TilePlan {
    int shape;
    uint32_t splits, steps;
};
// Tile and splits of k: the least of an estimate in microseconds.  4 for a
// tile's start and end; the splits' sums are written and read at 4 TB/s and
// joined by one more launch.
template <int N>
inline TilePlan plan_tiles(const hh_linear_args &a, int cus, const Shape (&shapes)[N]) {
    TilePlan best = {0, 1, 1};
    double least = 1e30;
    const uint32_t steps = (a.k + 63) / 64;
    for (int i = 0; i < N; i++)
        for (uint32_t want = 1; want <= 16 && (want == 1 || want <= steps); want *= 2) {
            const uint32_t each = steps ? (steps + want - 1) / want : 1, splits = steps ? (steps + each - 1) / each : 1;
            const uint64_t tiles = (uint64_t)((a.n + shapes[i].n - 1) / shapes[i].n) * ((a.m + shapes[i].m - 1) / shapes[i].m);
            const uint64_t slots = (uint64_t)cus * shapes[i].per_cu, work = tiles * splits;
            if (splits > 1 && (uint64_t)a.m * a.n > 1ull << 30) continue;  // their sums: at most 64 GiB, one launch to join
            const double step = work <= (uint64_t)cus ? shapes[i].alone : shapes[i].us;
            double us = (double)((work + slots - 1) / slots) * (step * each + 4.0);
            if (splits > 1) us += 4.0 + (double)a.m * a.n * 8.0 * splits / 4e6;
            if (us < least) least = us, best = {i, splits, each};
        }
    return best;
}
// Of tiles copied straight to LDS, and through registers (16-bit W).  For
// products of 33 to 4096 rows by 4096 to 14336 columns the estimates are
// within 30 % of the times, half of them within 10 %; INT4 through registers
// takes up to 1.2 of them, with groups across rows 2.6 to 4.
constexpr Shape kLargeShapes[] = {{256, 256, 1, 1.65, 1.65}, {256, 128, 1, 1.0, 1.0}, {128, 256, 1, 1.0, 1.0},
                                  {128, 128, 2, 1.13, 0.67}, {128, 64, 3, 1.0, 0.45}};
constexpr Shape kAnyShapes[] = {{128, 128, 2, 2.0, 1.3}, {64, 64, 4, 1.6, 0.9}};

// Room for the splits' sums.
int32_t split_room(hh_context *ctx, const LinearArgs &p, const TilePlan &plan, hipStream_t s, Split *split) {
    *split = {plan.steps, nullptr};
    if (plan.splits == 1) return HH_OK;
    return op_room(ctx, s, (size_t)plan.splits * p.a.m * ((p.a.n + 3) / 4 * 4) * sizeof(float), &split->partial);
}
template <int DT, int YT>
int32_t join_splits(const LinearArgs &p, const TilePlan &plan, const Split &split, hipStream_t s) {
    if (split.partial)
        hipLaunchKernelGGL((linear_join_kernel<DT, YT>), dim3((uint32_t)(((uint64_t)p.a.m * ((p.a.n + 3) / 4) + 255) / 256)),
                           dim3(256), 0, s, p,
                           split.partial, plan.splits);
    return from_hip(hipGetLastError());
}

template <int DT, int YT, int MODE>
int32_t launch_any(hh_context *ctx, const LinearArgs &p, int cus, hipStream_t s) {
    const uint32_t n = p.a.n, m = p.a.m;
    const TilePlan plan = plan_tiles(p.a, cus, kAnyShapes);
    Split split;
    const int32_t rc = split_room(ctx, p, plan, s, &split);
    if (rc != HH_OK) return rc;
    const uint32_t S = kAnyShapes[plan.shape].n;
    const dim3 grid((n + S - 1) / S, (m + S - 1) / S, plan.splits);
    if (S == 128)
        hipLaunchKernelGGL((linear_tile_kernel<DT, YT, MODE, 128>), grid, dim3(256), 0, s, p, split);
    else
        hipLaunchKernelGGL((linear_tile_kernel<DT, YT, MODE, 64>), grid, dim3(256), 0, s, p, split);
    return join_splits<DT, YT>(p, plan, split, s);
}

template <int DT, int YT>
int32_t launch_linear(hh_context *ctx, const LinearArgs &p, hipStream_t s) {
    const hh_linear_args &a = p.a;
    const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
    const bool int4 = a.w_dtype == HH_INT4;
    if (int4 && a.k % 32) return launch_any<DT, YT, kInt4Any>(ctx, p, cus, s);
    const bool aligned = !int4 && !(((uintptr_t)a.d_x | (uintptr_t)a.d_w) & 15u) && !((a.x_stride | a.w_stride) & 7u) &&
                         a.k % 64 == 0 && a.k && a.x_stride < 1u << 22 && a.w_stride < 1u << 22;  // offsets in a tile: 32 bits
    // up to 64 rows straight from memory; above 32 aligned tiles are faster
    // (64 rows of 4096 x 4096 18 us against 22, of 8192 x 8192 43 against 77).
    // Large products of 33 to 64 rows an odd number of values apart would be
    // too: 56 and 213 us, in tiles through registers 19 and 47.
    if (a.m <= (aligned ? 32u : 64u)) {
        const int rows = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
        return from_hip(int4 ? (rows == 1   ? launch_rows<DT, YT, 1, true>(p, cus, s)
                                : rows == 2 ? launch_rows<DT, YT, 2, true>(p, cus, s)
                                            : launch_rows<DT, YT, 4, true>(p, cus, s))
                             : (rows == 1   ? launch_rows<DT, YT, 1, false>(p, cus, s)
                                : rows == 2 ? launch_rows<DT, YT, 2, false>(p, cus, s)
                                            : launch_rows<DT, YT, 4, false>(p, cus, s)));
    }
    if (int4) return launch_any<DT, YT, kInt4>(ctx, p, cus, s);
    if (!aligned) return launch_any<DT, YT, kHalf>(ctx, p, cus, s);
    const TilePlan plan = plan_tiles(a, cus, kLargeShapes);
    Split split;
    const int32_t rc = split_room(ctx, p, plan, s, &split);
    if (rc != HH_OK) return rc;
    switch (plan.shape) {
        case 0: launch_tiles<DT, YT, 256, 256, 2, 4>(p, split, plan.splits, s); break;
        case 1: launch_tiles<DT, YT, 256, 128, 4, 2>(p, split, plan.splits, s); break;
        case 2: launch_tiles<DT, YT, 128, 256, 2, 4>(p, split, plan.splits, s); break;
        case 3: launch_tiles<DT, YT, 128, 128, 2, 2>(p, split, plan.splits, s); break;
        default: launch_tiles<DT, YT, 128, 64, 2, 2>(p, split, plan.splits, s); break;
    }
    return join_splits<DT, YT>(p, plan, split, s);
}

}  // namespace
}  // namespace hh

extern "C" int32_t hh_linear(hh_context *ctx, const hh_linear_args *a, void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    if (a->dtype != HH_F16 && a->dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (a->w_dtype != a->dtype && a->w_dtype != HH_INT4) return HH_ERR_UNSUPPORTED;
    if (a->y_dtype != a->dtype && a->y_dtype != HH_F32) return HH_ERR_UNSUPPORTED;
    if (a->activation < HH_ACT_NONE || a->activation > HH_ACT_SILU) return HH_ERR_UNSUPPORTED;
    if (a->m >= 1u << 21 || a->n >= 1u << 26 || a->k >= 1u << 31) return HH_ERR_INVALID_ARGUMENT;
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
    if (a->dtype == HH_BF16)
        return a->y_dtype == HH_F32 ? hh::launch_linear<HH_BF16, HH_F32>(ctx, p, s)
                                    : hh::launch_linear<HH_BF16, HH_BF16>(ctx, p, s);
    return a->y_dtype == HH_F32 ? hh::launch_linear<HH_F16, HH_F32>(ctx, p, s) : hh::launch_linear<HH_F16, HH_F16>(ctx, p, s);
}
