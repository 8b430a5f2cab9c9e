// The gradients of y = act(x G^T + gate bias) * (x U^T + up bias)
// (hh_gated_linear_backward, include/haagenti_hip.h).
//
// 1. slope: dg = dy up act'(gate), du = dy act(gate), in f32 from the sums
//    that the forward pass kept, rounded to x's type (half a step, what the
//    matrix instructions take) into D = [dg | du]: m rows of 2 N columns, N =
//    n rounded up to 64, zeros past both.  The biases' sums are taken here,
//    before the rounding.  Bound by memory (14 bytes an element).  f16 has too
//    short a range for this (dg above 65504 though dx isn't, or below 2^-24):
//    there a first pass finds the largest |dg|, |du| of each row and of each
//    column, and D is written twice, for dx with its rows scaled by powers of
//    two to a largest of 2^14 to 2^15, for the weights with its columns; the
//    products' results are scaled back in f32.  So a value is off by half a step
//    of its own, or by 2^-39 of the largest of its row (column) if that is more.  2048
//    x 14336 x 4096 1037 us a call (917 without), 77 x 1003 x 1001 28 (20).
// 2. dx = D [G; U]: a product over D's columns, the weights' rows.
// 3. [dG; dU] = D^T x: a product over the rows of both.
//
// The products' sums run over the slow index of their operands (both in 3).
// Tiles come to LDS as they lie in memory, 32 of that index deep (64 through
// registers), and are transposed on their way to registers:
// ds_read_b64_tr_b16 gives lane i of 16 column i of 4 rows that the 16 lanes
// read.  Nothing is transposed through memory (the weights alone would cost 85
// us at 2 x 14336 x 4096).
//
// 2048 x 14336 x 4096 bf16, calls of one run: all 908 us; the slope alone 82,
// with dx 490, so that dx and the join of its two splits take 408 (1180 TFLOP/s;
// the library's product 395), with the weights' 481, so 399 (1200; 444).  By a
// profiler, where all are slower: 85, 447 + 15 and 473.  Bound by LDS reads
// beside the matrix pipes.
#include <type_traits>

#include "layer_ops.hpp"

namespace hh {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

template <int DT>
__device__ __forceinline__ f32x4 mma16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    if constexpr (DT == HH_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------- slope

struct SlopeArgs {
    const uint16_t *dy;
    const float *saved;   // [m][gate's n, up's n]
    uint16_t *d;          // [rows][2 N]; f16: for dx, or null
    uint16_t *d_cols;     // f16: for the weights, or null
    // f16: bits of the largest magnitudes
    uint32_t *row_top;    // of D's rows, m rounded up to 64, and then
    uint32_t *col_top;    // of its 2 N columns
    uint32_t *row_part;   // [n / 256][m rounded up to 64], of 256 columns of a row, or null
    uint32_t *col_part;   // [row block][2 N], or null
    float *part;          // [row block][2 n]: the biases' sums, or null
    float *gate_bias, *up_bias;
    uint64_t dy_stride;
    uint32_t m, n, wide;  // wide: N
    uint32_t rows;        // m, or m rounded up to 64 where the rows past it are read
    uint32_t block_rows;  // of a workgroup
    int act;
};

// act(z) and act'(z).
__device__ __forceinline__ void act_and_slope(float z, int act, float &a, float &s) {
    switch (act) {
        case HH_ACT_RELU: a = fmaxf(z, 0.0f) + (z != z ? z : 0.0f), s = z > 0.0f ? 1.0f : z != z ? z : 0.0f; break;
        case HH_ACT_GELU: {
            const float p = 0.5f * (1.0f + erff(z * 0.70710678118654752440f));
            a = z * p, s = fmaf(z * 0.39894228040143267794f, __expf(-0.5f * z * z), p);
            break;
        }
        case HH_ACT_GELU_TANH: {
            // 0.5 (1 + tanh u) = p = 1 / (1 + exp(-2 u)); its slope 2 p (1 - p) u'
            const float u = 0.79788456080286535588f * (z + 0.044715f * z * z * z);
            const float p = 1.0f / (1.0f + __expf(-2.0f * u));
            a = z * p;
            const float du = 0.79788456080286535588f * (1.0f + 0.134145f * z * z);
            const float q = p * (1.0f - p);
            s = q == 0.0f ? p : fmaf(2.0f * z * q, du, p);  // far out du may be infinite
            break;
        }
        case HH_ACT_SILU: {
            const float p = 1.0f / (1.0f + __expf(-z));
            a = z * p;
            const float q = p * (1.0f - p);
            s = q == 0.0f ? p : fmaf(z, q, p);
            break;
        }
        default: a = z, s = 1.0f;
    }
}

// The power of two that brings a largest magnitude (its bits) to 2^14 .. 2^15,
// and what undoes it.  Infinities and NaN stay what they are, beside them what
// is finite stays finite.
__device__ __forceinline__ int power_of(uint32_t top) { return min(141 - (int)(top >> 23), 126); }
__device__ __forceinline__ float scale_to(uint32_t top) { return __uint_as_float((uint32_t)(127 + power_of(top)) << 23); }
__device__ __forceinline__ float scale_back(uint32_t top) { return __uint_as_float((uint32_t)(127 - power_of(top)) << 23); }

__device__ __forceinline__ f32x4 scaled(const f32x4 &v, const f32x4 &by) {
    return f32x4{v[0] * by[0], v[1] * by[1], v[2] * by[2], v[3] * by[3]};
}
template <int DT>
__device__ __forceinline__ u32x2 packed(const f32x4 &v) {
    return u32x2{f32_to_half<DT>(v[0]) | f32_to_half<DT>(v[1]) << 16, f32_to_half<DT>(v[2]) | f32_to_half<DT>(v[3]) << 16};
}
// Bits of the larger magnitude (NaN above all).
__device__ __forceinline__ uint32_t larger(uint32_t top, float v) { return max(top, __float_as_uint(fabsf(v))); }

// A wave's largest, in every lane.
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
    auto with = [&](float other) { v = max(v, __float_as_uint(other)); };
    with(dpp<0xb1>(__uint_as_float(v)));
    with(dpp<0x4e>(__uint_as_float(v)));
    with(dpp<0x141>(__uint_as_float(v)));
    with(dpp<0x140>(__uint_as_float(v)));
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)s[0], (uint32_t)s[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t)t[0], (uint32_t)t[1]);
}

// 4 columns a lane, 256 a wave, every 4th row of the block a wave, R of them at
// a time: all their loads are done, at places that are there (behind
// conditions they wait for one another: 77 x 1003 14 us, so 4).  2048 x 14336:
// 84 us, 411 MB at 4.9 TB/s.  TOPS: the pass that finds the largest magnitudes.
template <int DT, int R, bool TOPS>
__global__ __launch_bounds__(256) void gated_slope_kernel(const SlopeArgs p) {
    __shared__ __align__(16) float sums[2][4][256];
    const uint32_t across = (p.wide + 255) / 256, block = blockIdx.x / across, c0 = blockIdx.x % across * 256;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = c0 + lane * 4, r0 = block * p.block_rows;
    const uint32_t end = min(r0 + p.block_rows, p.rows);
    f32x4 sg = {0, 0, 0, 0}, su = {0, 0, 0, 0};
    u32x4 top_g = {0, 0, 0, 0}, top_u = {0, 0, 0, 0};
    f32x4 by_g = {1, 1, 1, 1}, by_u = {1, 1, 1, 1};  // f16: the columns' powers of two
    if (TOPS || c < p.wide) {
        if (!TOPS && DT == HH_F16 && p.d_cols) {
            const u32x4 g = *reinterpret_cast<const u32x4 *>(p.col_top + c), u = *reinterpret_cast<const u32x4 *>(p.col_top + p.wide + c);
#pragma unroll
            for (int e = 0; e < 4; e++) by_g[e] = scale_to(g[e]), by_u[e] = scale_to(u[e]);
        }
        for (uint32_t first = r0 + wave; first < end; first += 4 * R) {
            f32x4 d[R], g[R], u[R];
            if (c0 + 256 <= p.n) {
#pragma unroll
                for (int k = 0; k < R; k++) {
                    const uint32_t r = min(first + 4 * k, p.m - 1);
                    const float *s = p.saved + (uint64_t)r * 2 * p.n + c;
                    const u32x2 v = *reinterpret_cast<const u32x2_any *>(p.dy + r * p.dy_stride + c);
                    g[k] = *reinterpret_cast<const f32x4_any *>(s), u[k] = *reinterpret_cast<const f32x4_any *>(s + p.n);
#pragma unroll
                    for (int e = 0; e < 4; e++) d[k][e] = half_to_f32<DT>((v[e >> 1] >> (16 * (e & 1))) & 0xffffu);
                }
            } else {
#pragma unroll
                for (int k = 0; k < R; k++) {
                    const uint32_t r = min(first + 4 * k, p.m - 1);
                    const float *s = p.saved + (uint64_t)r * 2 * p.n;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t col = min(c + e, p.n - 1);
                        d[k][e] = half_to_f32<DT>(p.dy[r * p.dy_stride + col]), g[k][e] = s[col], u[k][e] = s[p.n + col];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < R; k++) {
                const uint32_t r = first + 4 * k;
                if (r >= end) break;
                f32x4 dg = {0, 0, 0, 0}, du = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float a, slope;
                    act_and_slope(g[k][e], p.act, a, slope);
                    if (r < p.m && c + e < p.n) dg[e] = d[k][e] * u[k][e] * slope, du[e] = d[k][e] * a;
                }
                const uint64_t at = (uint64_t)r * 2 * p.wide + c;
                if constexpr (TOPS) {
                    uint32_t top = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        top_g[e] = larger(top_g[e], dg[e]), top_u[e] = larger(top_u[e], du[e]);
                        top = larger(larger(top, dg[e]), du[e]);
                    }
                    top = wave_top(top);
                    if (p.row_part && lane == 0) p.row_part[(uint64_t)(c0 / 256) * ((p.m + 63) / 64 * 64) + r] = top;
                    continue;
                }
                sg += dg, su += du;
                if constexpr (DT == HH_F16) {
                    if (p.d) {
                        const float by = r < p.m ? scale_to(p.row_top[r]) : 1.0f;
                        *reinterpret_cast<u32x2 *>(p.d + at) = packed<DT>(dg * by);
                        *reinterpret_cast<u32x2 *>(p.d + at + p.wide) = packed<DT>(du * by);
                    }
                    if (p.d_cols) {
                        *reinterpret_cast<u32x2 *>(p.d_cols + at) = packed<DT>(scaled(dg, by_g));
                        *reinterpret_cast<u32x2 *>(p.d_cols + at + p.wide) = packed<DT>(scaled(du, by_u));
                    }
                } else {
                    *reinterpret_cast<u32x2 *>(p.d + at) = packed<DT>(dg);
                    *reinterpret_cast<u32x2 *>(p.d + at + p.wide) = packed<DT>(du);
                }
            }
        }
    }
    if constexpr (TOPS) {
        if (!p.col_part) return;
        uint32_t (*tops)[4][256] = reinterpret_cast<uint32_t (*)[4][256]>(sums);
        *reinterpret_cast<u32x4 *>(&tops[0][wave][lane * 4]) = top_g;
        *reinterpret_cast<u32x4 *>(&tops[1][wave][lane * 4]) = top_u;
        __syncthreads();
        if (c0 + threadIdx.x >= p.wide) return;
#pragma unroll
        for (uint32_t k = 0; k < 2; k++)
            p.col_part[((uint64_t)block * 2 + k) * p.wide + c0 + threadIdx.x] =
                max(max(tops[k][0][threadIdx.x], tops[k][1][threadIdx.x]), max(tops[k][2][threadIdx.x], tops[k][3][threadIdx.x]));
        return;
    }
    if (!p.part) return;
    *reinterpret_cast<f32x4 *>(&sums[0][wave][lane * 4]) = sg;
    *reinterpret_cast<f32x4 *>(&sums[1][wave][lane * 4]) = su;
    __syncthreads();
    const uint32_t col = c0 + threadIdx.x;
    if (col >= p.n) return;
#pragma unroll
    for (int k = 0; k < 2; k++)
        p.part[((uint64_t)block * 2 + k) * p.n + col] = (sums[k][0][threadIdx.x] + sums[k][1][threadIdx.x]) +
                                                             (sums[k][2][threadIdx.x] + sums[k][3][threadIdx.x]);
}
// The row blocks' sums, in order: 32 columns to a workgroup, its 32 rows of
// threads over every 32nd block.
__global__ __launch_bounds__(1024) void gated_bias_kernel(const SlopeArgs p, uint32_t blocks) {
    __shared__ float sum[32][33];
    const uint32_t col = blockIdx.x * 32 + (threadIdx.x & 31u), q = threadIdx.x >> 5, k = blockIdx.y;
    float *out = k ? p.up_bias : p.gate_bias;
    if (!out) return;
    float s = 0.0f;
    if (col < p.n)
        for (uint32_t i = q; i < blocks; i += 32) s += p.part[((uint64_t)i * 2 + k) * p.n + col];
    sum[q][threadIdx.x & 31u] = s;
    __syncthreads();
    if (q || col >= p.n) return;
    for (int i = 1; i < 32; i++) s += sum[i][threadIdx.x & 31u];
    out[col] = s;
}

// The largest of the parts of 32 rows (columns) to a workgroup, its 32 rows of
// threads over every 32nd part.
__global__ __launch_bounds__(1024) void gated_tops_kernel(const SlopeArgs p, uint32_t rows, uint32_t across, uint32_t blocks) {
    __shared__ uint32_t tops[32][33];
    const uint32_t at = blockIdx.x * 32 + (threadIdx.x & 31u), q = threadIdx.x >> 5;
    const bool row = blockIdx.x * 32 < rows;  // (rows are whole 64s)
    const uint32_t *part = row ? p.row_part : p.col_part;
    if (!part) return;
    const uint32_t parts = row ? across : blocks, step = row ? rows : 2 * p.wide, col = row ? at : at - rows;
    uint32_t top = 0;
    if (!row || at < p.m)
        for (uint32_t i = q; i < parts; i += 32) top = max(top, part[(uint64_t)i * step + col]);
    tops[q][threadIdx.x & 31u] = top;
    __syncthreads();
    if (q) return;
    for (int i = 1; i < 32; i++) top = max(top, tops[i][threadIdx.x & 31u]);
    p.row_top[at] = top;
}

// ---------------------------------------------------------------- products
//
// C[r][c] = sum over t of R[r][t] L[t][c].  For dx: r the rows of x, c its
// columns, t the weights' rows (G's, zeros up to N, U's), R = D.  For the
// weights (TURN: both operands are transposed): r D's columns, c x's columns,
// t the rows, R[r][t] = D[t][r].

struct BackArgs {
    const uint16_t *l[2];    // the left matrix's parts: G and U, or x
    uint64_t l_stride[2];
    const uint16_t *d;
    const uint32_t *top;     // f16: of each row of C, what D's was scaled by
    uint16_t *out[2];        // dx, or dG and dU
    uint64_t out_stride[2];
    float *partial;          // [split][rows][cols rounded up to 4], or null
    uint32_t rows, cols;     // of C; TURN: rows counts 2 N
    uint32_t depth;          // t of one part
    uint32_t n, wide;
    uint32_t steps;          // of a split: of 32 t, through registers of 64
};

// Where 16 columns' unit of 32 bytes of row t of a transposed tile lies: rows
// that are read together (t = 8 g + 0..3) in different banks.
__device__ __forceinline__ uint32_t twist(uint32_t t, uint32_t units) { return ((t & 3u) | (t >> 1 & 4u)) & (units - 1); }

// Steps of 32 t of a part (D has zeros where its last one ends later).
__device__ __forceinline__ uint32_t steps_of(uint32_t depth) { return (depth + 31) / 32; }

template <int W>
struct Turned {
    // LDS offsets (elements) of this lane's reads: fragment i's rows t = 8 g + (lane / 4 % 4)
    template <int N>
    static __device__ __forceinline__ void places(uint32_t lane, uint32_t first, uint32_t (&at)[N]) {
        const uint32_t t = (lane >> 4) * 8 + (lane >> 2 & 3u);
#pragma unroll
        for (int i = 0; i < N; i++) at[i] = t * W + ((first / 16 + i) ^ twist(t, W / 16)) * 16 + (lane & 3u) * 4;
    }
    // 8 t of a column: t = 32 f + 8 g + 0..7
    static __device__ __forceinline__ u32x4 read(const uint16_t *lds, uint32_t at, uint32_t f) {
#if defined(__HIP_DEVICE_COMPILE__)
        typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds + at + f * 32 * W));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(lds + at + f * 32 * W + 4 * W));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return u32x4{a[0], a[1], b[0], b[1]};
#else
        return u32x4{};
#endif
    }
};

// The tile of a workgroup: bands of 8 tiles of r, in them down the band and
// then along c, consecutive ones on one XCD (32 of them at a time read 8 + 4
// tiles' operands).
struct Place {
    uint32_t r, c;
};
__device__ __forceinline__ Place place_of(uint32_t rt, uint32_t ct) {
    const uint32_t share = gridDim.x / 8, rest = gridDim.x % 8, xcd = blockIdx.x % 8;
    const uint32_t id = xcd * share + min(xcd, rest) + blockIdx.x / 8;
    const uint32_t band = id / (8 * ct), in = id % (8 * ct), high = min(8u, rt - 8 * band);
    return {8 * band + in % high, in / high};
}

// Outputs c .. c + 3 of row r.
template <int DT, bool TURN>
__device__ __forceinline__ void store_back(const BackArgs &p, uint32_t split, uint32_t r, uint32_t c, f32x4 v) {
    if (p.partial) {
        *reinterpret_cast<f32x4 *>(p.partial + ((uint64_t)split * p.rows + r) * ((p.cols + 3) / 4 * 4) + c) = v;
        return;
    }
    const uint32_t side = TURN && r >= p.wide, row = TURN && side ? r - p.wide : r;
    if (TURN && row >= p.n) return;
    if constexpr (DT == HH_F16) v *= scale_back(p.top[r]);
    uint16_t *to = p.out[side] + row * p.out_stride[side] + c;
    if (c + 4 <= p.cols) {
        *reinterpret_cast<u32x2_any *>(to) =
            u32x2{f32_to_half<DT>(v[0]) | f32_to_half<DT>(v[1]) << 16, f32_to_half<DT>(v[2]) | f32_to_half<DT>(v[3]) << 16};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (c + i < p.cols) to[i] = (uint16_t)f32_to_half<DT>(v[i]);
}

// Aligned operands, copied straight to LDS in tiles 32 deep, four of them in
// turn: three are on their way while one is multiplied (64 deep and two in
// turn, a copy has one tile's products to arrive in: 483 and 479 us where
// these took 440 and 457, by a profiler), 16-byte pieces at places that depend on their row.  One
// barrier a tile: before it a wave waits for its own part of the next tile's
// copies, the oldest under way, and for its reads of the last one.
__device__ __forceinline__ uint32_t shift_of(uint32_t row) { return (0u - (row >> 2)) & 3u; }
template <int ROWS, int T>
__device__ __forceinline__ void plain_offsets(uint32_t stride, uint32_t rows, uint32_t (&off)[ROWS * 4 / T]) {
#pragma unroll
    for (int j = 0; j < ROWS * 4 / T; j++) {
        const uint32_t slot = j * T + threadIdx.x, row = slot >> 2, piece = (slot & 3u) ^ shift_of(row);
        off[j] = (min(row, rows - 1) * stride + piece * 8) * 2;
    }
}
// A transposed tile of 32 rows t by W columns: chunks of 1 KiB, what a wave
// copies at once, hold 512 / W rows; which ones, the unit of 16 columns that a
// row's own is swapped with and the gap after a chunk are chosen so that the 8
// rows of 32 bytes that half a wave reads together lie in different banks, and
// so that few registers hold a lane's places: fragment i's is the (i mod 512 /
// W)-th and a constant.
template <int W>
struct Chunks {
    static constexpr int ROWS = 512 / W, GAP = W == 64 ? 0 : 16 * ROWS, SIZE = 512 + GAP, ALL = 32 / ROWS * SIZE;  // elements
    static constexpr int NEXT = W == 256 ? 4 * SIZE : W == 128 ? 2 * SIZE : SIZE;  // from t to t + 4
    static constexpr int PLACES = W == 64 ? 4 : ROWS;
    static __device__ __forceinline__ uint32_t sub(uint32_t t) {
        return W == 256 ? t >> 3 & 1u : W == 128 ? (t >> 2 & 2u) | (t & 1u) : (t >> 1 & 4u) | (t & 3u);
    }
    static __device__ __forceinline__ uint32_t chunk(uint32_t t) {
        return W == 256 ? (t & 7u) | (t >> 1 & 8u) : W == 128 ? (t >> 1 & 3u) | (t >> 2 & 4u) : (t >> 2 & 1u) | (t >> 3 & 2u);
    }
    static __device__ __forceinline__ uint32_t row(uint32_t chunk, uint32_t sub) {
        return W == 256   ? (chunk & 7u) | sub << 3 | (chunk & 8u) << 1
               : W == 128 ? (sub & 1u) | (chunk & 3u) << 1 | (sub & 2u) << 2 | (chunk & 4u) << 2
                          : (sub & 3u) | (chunk & 1u) << 2 | (sub & 4u) << 1 | (chunk & 2u) << 3;
    }
    // the row and the column of what piece `place` of a chunk holds
    static __device__ __forceinline__ void held(uint32_t chunk, uint32_t place, uint32_t &t, uint32_t &c) {
        const uint32_t s = place / (64 / ROWS), piece = place % (64 / ROWS);
        t = row(chunk, s), c = ((piece >> 1 ^ (s & (PLACES - 1))) * 2 + (piece & 1u)) * 8;
    }
    // this lane's reads: rows t = 8 g + (lane / 4 % 4), columns from `first` on
    static __device__ __forceinline__ void places(uint32_t lane, uint32_t first, uint32_t (&at)[PLACES]) {
        const uint32_t t = (lane >> 4) * 8 + (lane >> 2 & 3u), s = sub(t);
#pragma unroll
        for (int i = 0; i < PLACES; i++)
            at[i] = chunk(t) * SIZE + s * W + ((first / 16 + i) ^ (s & (PLACES - 1))) * 16 + (lane & 3u) * 4;
    }
    // 8 t of fragment i's column
    static __device__ __forceinline__ u32x4 read(const uint16_t *lds, const uint32_t (&at)[PLACES], int i) {
#if defined(__HIP_DEVICE_COMPILE__)
        typedef __attribute__((address_space(3))) s16x4 *lds_s16x4;
        const uint16_t *from = lds + at[i % PLACES] + i / PLACES * PLACES * 16;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)from);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(from + NEXT));
        const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
        return u32x4{a[0], a[1], b[0], b[1]};
#else
        return u32x4{};
#endif
    }
    // Offsets of a lane's pieces in the matrix (bytes): `rows` rows of it are
    // there, others repeat the last; columns past it (`cols` of it, a multiple
    // of 8) its last piece.
    template <int T>
    static __device__ __forceinline__ void offsets(uint32_t thread, uint32_t stride, uint32_t rows, uint32_t cols,
                                                   uint32_t (&off)[W * 4 / T]) {
#pragma unroll
        for (int j = 0; j < W * 4 / T; j++) {
            uint32_t t, c;
            held(j * (T / 64) + thread / 64, thread & 63u, t, c);
            off[j] = (min(t, rows - 1) * stride + min(c, cols - 8)) * 2;
        }
    }
    // Zeros to rows from `rows` on.
    template <int T>
    static __device__ __forceinline__ void clear(uint32_t thread, uint16_t *lds, uint32_t rows) {
#pragma unroll
        for (int j = 0; j < W * 4 / T; j++) {
            uint32_t t, c;
            const uint32_t chunk = j * (T / 64) + thread / 64;
            held(chunk, thread & 63u, t, c);
            if (t >= rows) *reinterpret_cast<u32x4 *>(lds + chunk * SIZE + (thread & 63u) * 8) = u32x4{0, 0, 0, 0};
        }
    }
};
template <int N, int T, int SIZE, typename Source>
__device__ __forceinline__ void copy_pieces(const Source &from, uint32_t at, const uint32_t (&off)[N], uint16_t *lds, uint32_t wave) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int j = 0; j < N; j++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            from, (__attribute__((address_space(3))) void *)(lds + (j * (T / 64) + wave) * SIZE), 16, off[j], at, 0, 0);
#endif
}
__device__ __forceinline__ auto source(const uint16_t *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(p), 0, 0xffffffffu, 0x00027000);
}
// Waits until at most N of the wave's loads are under way and all its LDS
// reads are done.
template <int N>
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);
}

template <int DT, bool TURN, int TC, int TR, int WC, int WR>
__global__ __launch_bounds__(64 * WC * WR) void gated_back_kernel(const BackArgs p) {
    constexpr int T = 64 * WC * WR, NI = TC / WC / 16, MI = TR / WR / 16, LP = TC * 4 / T, RP = TR * 4 / T;
    // a tile of the left matrix, then one of the right; arrays of their own, so
    // that the compiler sees which of them a copy writes
    typedef Chunks<TC> Left;
    typedef Chunks<TR> Right;
    constexpr int L = Left::ALL, ALL = L + (TURN ? Right::ALL : TR * 32);
    __shared__ __align__(16) uint16_t t0[ALL], t1[ALL], t2[ALL], t3[ALL];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t r = lane & 15u, g = lane >> 4;
    const Place at = place_of((p.rows + TR - 1) / TR, (p.cols + TC - 1) / TC);
    const uint32_t c0 = at.c * TC, r0 = at.r * TR, wc = wave % WC * (TC / WC), wr = wave / WC * (TR / WR);
    const uint32_t each = steps_of(p.depth), all = TURN ? each : 2 * each;
    const uint32_t s0 = blockIdx.y * p.steps, s1 = min(all, s0 + p.steps);
    f32x4 acc[NI][MI];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < MI; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    uint32_t lo[LP], ro[RP], la[Left::PLACES], ra[Right::PLACES];
    if constexpr (TURN)
        Right::template offsets<T>(threadIdx.x, 2 * p.wide, 32, p.rows - r0, ro);
    else
        plain_offsets<TR, T>(2 * p.wide, p.rows - r0, ro);
    Left::places(lane, wc, la);
    if constexpr (TURN)
        Right::places(lane, wr, ra);
    else
        ra[0] = (wr + r) * 32 + (g ^ shift_of(r)) * 8;
    // (what is computed from this is computed where it is needed, and not kept
    // in registers through all steps)
    auto thread = []() {
        uint32_t t = threadIdx.x;
        asm volatile("" : "+v"(t));
        return t;
    };
    // Step s: rows of a part from t on; those past the part repeat its last
    // one and are cleared where they have come (D's are zeros).
    auto copy = [&](uint16_t *to, uint32_t s) {
        const uint32_t part = !TURN && s >= each, t = (s - (part ? each : 0)) * 32, left = p.depth - t;
        if (s == s0 || (!TURN && s == each) || left < 32)
            Left::template offsets<T>(thread(), (uint32_t)p.l_stride[part], min(left, 32u), p.cols - c0, lo);
        copy_pieces<LP, T, Left::SIZE>(source(p.l[part] + (uint64_t)t * p.l_stride[part] + c0), 0, lo, to, wave);
        if constexpr (TURN) {
            copy_pieces<RP, T, Right::SIZE>(source(p.d + (uint64_t)t * 2 * p.wide + r0), 0, ro, to + L, wave);
        } else {
            copy_pieces<RP, T, 512>(source(p.d + (uint64_t)r0 * 2 * p.wide), 2 * (t + (part ? p.wide : 0)), ro, to + L, wave);
        }
    };
    // Zeros in the tile of step s: rows past the part's end, all of a step past
    // the last (the steps go around in fours).
    auto clear = [&](uint16_t *at, uint32_t s) {
        const uint32_t t = (s >= each ? s - each : s) * 32, left = p.depth - t;
        if (s >= s1) {
            for (uint32_t i = thread(); i < ALL / 8; i += T) reinterpret_cast<u32x4 *>(at)[i] = u32x4{0, 0, 0, 0};
        } else {
            if (left >= 32) return;
            Left::template clear<T>(thread(), at, left);
        }
        __syncthreads();
    };
    // Until at most AHEAD tiles are under way, and all waves are here.
    auto meet = [](auto ahead) {
        wait_loads<decltype(ahead)::value * (LP + RP)>();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    struct Fragments {
        u32x4 l[NI], r[MI];
    };
    auto read = [&](const uint16_t *ll, Fragments &f) {
        const uint16_t *lr = ll + L;
#pragma unroll
        for (int j = 0; j < MI; j++) {
            if constexpr (TURN)
                f.r[j] = Right::read(lr, ra, j);
            else
                f.r[j] = *reinterpret_cast<const u32x4 *>(&lr[ra[0] + 16 * j * 32]);
        }
#pragma unroll
        for (int i = 0; i < NI; i++) f.l[i] = Left::read(ll, la, i);
    };
    // Step s: its products, from the registers `now`; the next step's tile,
    // which is here once all waves are, goes to `after` meanwhile; the buffer
    // of this step's, which all waves have read, takes the tile 4 steps on.
    // (Tiles past the last are that one again, until they are cleared: so as
    // many copies are under way at every step, and the compiler, which counts
    // them too, adds no waits of its own.)
    auto step = [&](uint32_t s, uint16_t *own, const uint16_t *next, Fragments &now, Fragments &after) {
        meet(std::integral_constant<int, 2>());
        clear(const_cast<uint16_t *>(next), s + 1);
        copy(own, min(s + 4, s1 - 1));
        read(next, after);
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
            for (int j = 0; j < MI; j++) acc[i][j] = mma16<DT>(now.l[i], now.r[j], acc[i][j]);
        // a read after every one or two products
        constexpr int reads = 2 * NI + (TURN ? 2 * MI : MI), products = NI * MI, few = products / reads, more = products % reads;
#pragma unroll
        for (int i = 0; i < reads; i++) {
            if (i < more)
                __builtin_amdgcn_sched_group_barrier(0x8, few + 1, 0);
            else
                __builtin_amdgcn_sched_group_barrier(0x8, few, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    if (s0 < s1) {
        Fragments a, b;
        copy(t0, s0);
        copy(t1, min(s0 + 1, s1 - 1));
        copy(t2, min(s0 + 2, s1 - 1));
        copy(t3, min(s0 + 3, s1 - 1));
        meet(std::integral_constant<int, 3>());
        clear(t0, s0);
        read(t0, a);
        for (uint32_t s = s0; s < s1; s += 4) {
            step(s, t0, t1, a, b);
            step(s + 1, t1, t2, b, a);
            step(s + 2, t2, t3, a, b);
            step(s + 3, t3, t0, b, a);
        }
    }
    // Sums go out by way of LDS, 16 rows x 64 columns of each wave at a time
    constexpr int Q = 16, PER = (TC + TR) * 64 / (16 * Q * 16);  // waves' pieces to a buffer
    static_assert(2 * PER >= WC * WR, "every wave's piece fits two buffers");
    f32x4 *own = reinterpret_cast<f32x4 *>(wave < PER ? t0 : t1) + wave % PER * 16 * Q;
#pragma unroll
    for (int j = 0; j < MI; j++)
#pragma unroll
        for (int h = 0; h < NI / 4; h++) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) own[r * Q + ((4 * i + g) ^ r)] = acc[4 * h + i][j];
            __syncthreads();
            uint32_t c = c0 + wc + 64 * h + r * 4, row = r0 + wr + 16 * j + g;
            asm volatile("" : "+v"(c), "+v"(row));  // no addresses of later pieces in registers meanwhile
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const f32x4 v = own[(4 * q + g) * Q + (r ^ (4 * q + g))];
                if (row + 4 * q < p.rows && c < p.cols) store_back<DT, TURN>(p, blockIdx.y, row + 4 * q, c, v);
            }
        }
}

// Any layout: tiles of S x S through registers, the next ones on their way
// while these are multiplied; 4 waves.
template <int DT, bool TURN, int S>
__global__ __launch_bounds__(256) void gated_back_any_kernel(const BackArgs p) {
    constexpr int F = S / 32, P = S / 32;  // fragments of a wave's side, pieces of 16 bytes a thread
    __shared__ __align__(16) uint16_t ll[S * 64], lr[S * 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, r = lane & 15u, g = lane >> 4;
    const Place at = place_of((p.rows + S - 1) / S, (p.cols + S - 1) / S);
    const uint32_t c0 = at.c * S, r0 = at.r * S, wc = (wave & 1u) * (S / 2), wr = (wave >> 1) * (S / 2);
    const uint32_t each = (p.depth + 63) / 64, all = TURN ? each : 2 * each;
    const uint32_t s0 = blockIdx.y * p.steps, s1 = min(all, s0 + p.steps);
    f32x4 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; i++)
#pragma unroll
        for (int j = 0; j < F; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    uint32_t la[F], ra[F];
    Turned<S>::places(lane, wc, la);
    if constexpr (TURN) Turned<S>::places(lane, wr, ra);
    u32x4 lv[P], rv[P];
    // Every load is done, at a place that is there, so that all of a step's are
    // under way at once; what is not this step's is put right on its way to LDS.
    // (Loads behind conditions wait for one another: 2048 x 14331 x 4093 2240
    // and 950 us with the slope, so 745 and 775.)  Columns and rows past C's hold
    // anything: only sums that are not stored take from them.
    auto fetch = [&](uint32_t s) {
        const uint32_t part = !TURN && s >= each, t0 = (s - (part ? each : 0)) * 64;
#pragma unroll
        for (int j = 0; j < P; j++) {
            const uint32_t slot = j * 256 + threadIdx.x, t = t0 + slot / (S / 8), c = c0 + slot % (S / 8) * 8;
            const uint16_t *from = p.l[part] + (uint64_t)min(t, p.depth - 1) * p.l_stride[part];
            if (p.cols >= 8) {
                lv[j] = *reinterpret_cast<const u32x4_any *>(from + min(c, p.cols - 8));
            } else {
                lv[j] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (uint32_t e = 0; e < 8; e++)
                    if (c + e < p.cols) lv[j][e >> 1] |= (uint32_t)from[e] << (16 * (e & 1));
            }
            if constexpr (TURN) {  // (D has whole steps of rows, and N whole pieces of 64 columns)
                rv[j] = *reinterpret_cast<const u32x4 *>(p.d + (uint64_t)t * 2 * p.wide + r0 + slot % (S / 8) * 8);
            } else {
                const uint32_t row = min(r0 + (slot >> 3), p.rows - 1);
                rv[j] = *reinterpret_cast<const u32x4 *>(p.d + (uint64_t)row * 2 * p.wide + (part ? p.wide : 0) + t0 + (slot & 7u) * 8);
            }
        }
    };
    auto stage = [&](uint32_t s) {
        const uint32_t t0 = (!TURN && s >= each ? s - each : s) * 64;
#pragma unroll
        for (int j = 0; j < P; j++) {
            const uint32_t slot = j * 256 + threadIdx.x, t = slot / (S / 8), piece = slot % (S / 8), row = slot >> 3;
            const uint32_t turned = t * S + (piece ^ (2 * twist(t, S / 16))) * 8;
            u32x4 v = lv[j];
            if (p.cols >= 8 && c0 + S > p.cols) {  // a row's last piece: read that much further left
                const uint32_t c = c0 + piece * 8, over = c + 8 > p.cols ? c + 8 - p.cols : 0;
                if (over & 4u) v = u32x4{v[2], v[3], 0, 0};
                if (over & 2u) v = u32x4{v[1], v[2], v[3], 0};
                if (over & 1u) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
            }
            if (t0 + t >= p.depth) v = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4 *>(&ll[turned]) = v;
            *reinterpret_cast<u32x4 *>(&lr[TURN ? turned : row * 64 + ((slot & 7u) ^ (row & 7u)) * 8]) = rv[j];
        }
    };
    if (s0 < s1) fetch(s0);
    for (uint32_t s = s0; s < s1; s++) {
        __syncthreads();
        stage(s);
        __syncthreads();
        if (s + 1 < s1) fetch(s + 1);
#pragma unroll
        for (uint32_t f = 0; f < 2; f++) {
            u32x4 rf[F];
#pragma unroll
            for (int j = 0; j < F; j++) {
                if constexpr (TURN)
                    rf[j] = Turned<S>::read(lr, ra[j], f);
                else
                    rf[j] = *reinterpret_cast<const u32x4 *>(&lr[(wr + 16 * j + r) * 64 + ((g + 4 * f) ^ (r & 7u)) * 8]);
            }
#pragma unroll
            for (int i = 0; i < F; i++) {
                const u32x4 lf = Turned<S>::read(ll, la[i], f);
#pragma unroll
                for (int j = 0; j < F; j++) acc[i][j] = mma16<DT>(lf, rf[j], acc[i][j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < F; j++)
#pragma unroll
        for (int i = 0; i < F; i++) {
            const uint32_t row = r0 + wr + 16 * j + r, c = c0 + wc + 16 * i + 4 * g;
            if (row < p.rows && c < p.cols) store_back<DT, TURN>(p, blockIdx.y, row, c, acc[i][j]);
        }
}

// The splits' sums, in order.
template <int DT, bool TURN>
__global__ __launch_bounds__(256) void gated_back_join_kernel(const BackArgs p, uint32_t splits) {
    const uint32_t quads = (p.cols + 3) / 4;
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (uint64_t)p.rows * quads) return;
    const uint32_t r = (uint32_t)(i / quads), c = (uint32_t)(i % quads) * 4;
    const uint64_t step = (uint64_t)p.rows * quads * 4;
    f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t j = 0; j < splits; j++) s += *reinterpret_cast<const f32x4 *>(p.partial + j * step + (uint64_t)r * quads * 4 + c);
    BackArgs q = p;
    q.partial = nullptr;
    store_back<DT, TURN>(q, 0, r, c, s);
}

// ---------------------------------------------------------------- host

// A tile shape (columns, rows), workgroups to a CU, microseconds per 64 t with
// all of them and with one alone.  These are the forward kernels' figures; of
// the kernels here, by a profiler, the weights' took 1.62, 0.88, 0.88, 0.97
// (alone 0.65), 0.96 (0.49), through registers 1.53 (1.12), 1.27 (0.72), and
// dx's 2.06, 1.40, 1.49, 1.41 (0.91), 1.60 (0.67), through registers 1.56
// (1.24), 1.52 (0.76).  So they rank the shapes of a product, within a fifth for
// most, and are no times of it; tables of their own were not tried.
struct Shape {
    uint32_t c, r, per_cu;
    double us, alone;
};
constexpr Shape kBackShapes[] = {{256, 256, 1, 1.65, 1.65}, {256, 128, 1, 1.0, 1.0}, {128, 256, 1, 1.0, 1.0},
                                 {128, 128, 2, 1.13, 0.67}, {128, 64, 3, 1.0, 0.45}};
constexpr Shape kBackAnyShapes[] = {{128, 128, 2, 2.0, 1.3}, {64, 64, 4, 1.6, 0.9}};
struct BackPlan {
    int shape;
    uint32_t splits, steps;
    uint64_t tiles;
    size_t room;  // bytes of the splits' sums
};
// The least of an estimate in microseconds: 4 for a tile's start and end; the
// splits' sums are written and read at 4 TB/s and joined by one more launch.
template <int N>
BackPlan plan_back(uint32_t rows, uint32_t cols, uint32_t steps, int cus, const Shape (&shapes)[N]) {
    BackPlan best = {0, 1, steps, 0, 0};
    double least = 1e30;
    const uint64_t sums = (uint64_t)rows * ((cols + 3) / 4 * 4);
    for (int i = 0; i < N; i++)
        for (uint32_t want = 1; want <= 16 && want <= steps; want *= 2) {
            const uint32_t each = (steps + want - 1) / want, splits = (steps + each - 1) / each;
            const uint64_t tiles = (uint64_t)((cols + shapes[i].c - 1) / shapes[i].c) * ((rows + shapes[i].r - 1) / shapes[i].r);
            const uint64_t slots = (uint64_t)cus * shapes[i].per_cu, work = tiles * splits;
            if (splits > 1 && sums > 1ull << 30) continue;  // 64 GiB at most, and one launch to join
            const double step = work <= (uint64_t)cus ? shapes[i].alone : shapes[i].us;
            double us = (double)((work + slots - 1) / slots) * (step * each + 4.0);
            if (splits > 1) us += 4.0 + (double)sums * 8.0 * splits / 4e6;
            if (us < least) least = us, best = {i, splits, each, tiles, splits > 1 ? splits * sums * sizeof(float) : 0};
        }
    return best;
}

template <int DT, bool TURN>
int32_t launch_back(BackArgs p, const BackPlan &plan, bool aligned, float *room, hipStream_t s) {
    p.steps = aligned ? 2 * plan.steps : plan.steps;
    p.partial = plan.splits > 1 ? room : nullptr;
    const dim3 grid((uint32_t)plan.tiles, plan.splits);
#define HH_BACK(TC, TR, WC, WR) hipLaunchKernelGGL((gated_back_kernel<DT, TURN, TC, TR, WC, WR>), grid, dim3(64 * WC * WR), 0, s, p)
    if (aligned) {
        switch (plan.shape) {
            case 0: HH_BACK(256, 256, 2, 4); break;
            case 1: HH_BACK(256, 128, 4, 2); break;
            case 2: HH_BACK(128, 256, 2, 4); break;
            case 3: HH_BACK(128, 128, 2, 2); break;
            default: HH_BACK(128, 64, 2, 2); break;
        }
    } else if (plan.shape == 0) {
        hipLaunchKernelGGL((gated_back_any_kernel<DT, TURN, 128>), grid, dim3(256), 0, s, p);
    } else {
        hipLaunchKernelGGL((gated_back_any_kernel<DT, TURN, 64>), grid, dim3(256), 0, s, p);
    }
#undef HH_BACK
    const int32_t rc = from_hip(hipGetLastError());
    if (rc != HH_OK || plan.splits == 1) return rc;
    hipLaunchKernelGGL((gated_back_join_kernel<DT, TURN>),
                       dim3((uint32_t)(((uint64_t)p.rows * ((p.cols + 3) / 4) + 255) / 256)), dim3(256), 0, s, p, plan.splits);
    return from_hip(hipGetLastError());
}

template <int DT>
int32_t gated_backward(hh_context *ctx, const hh_gated_args &a, const hh_gated_grads &d, hipStream_t s) {
    const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
    const uint32_t wide = (a.n + 63) / 64 * 64, rows = (a.m + 63) / 64 * 64;
    const bool dx = d.d_dx && a.k, dw = d.d_dgate && a.k, bias = d.d_dgate_bias || d.d_dup_bias;
    // offsets in a tile: 32 bits
    auto fits = [](const void *p, uint64_t stride) { return !((uintptr_t)p & 15u) && !(stride & 7u) && stride < 1u << 22; };
    const bool narrow = a.k % 8 == 0 && wide < 1u << 21;
    const bool x_aligned = narrow && fits(a.d_gate, a.gate_stride) && fits(a.d_up, a.up_stride);
    const bool w_aligned = narrow && fits(a.d_x, a.x_stride);
    BackPlan px = {}, pw = {};
    if (dx) px = x_aligned ? plan_back(a.m, a.k, 2 * (wide / 64), cus, kBackShapes) : plan_back(a.m, a.k, 2 * (wide / 64), cus, kBackAnyShapes);
    if (dw) pw = w_aligned ? plan_back(2 * wide, a.k, rows / 64, cus, kBackShapes) : plan_back(2 * wide, a.k, rows / 64, cus, kBackAnyShapes);
    // a launch has fewer than 2^32 threads
    // 32 rows to a workgroup, or 4 where that leaves CUs idle
    const uint32_t across = (wide + 255) / 256, block_rows = (uint64_t)(rows / 32) * across < 4 * (uint32_t)cus ? 4 : 32;
    const uint32_t blocks = rows / block_rows;
    if ((uint64_t)blocks * across >= 1u << 24 || px.tiles >= 1u << 23 || pw.tiles >= 1u << 23) return HH_ERR_UNSUPPORTED;
    // D (f16: one for each product, the largest magnitudes and their parts),
    // the biases' sums of row blocks, the larger of the products' sums
    const bool f16 = DT == HH_F16 && (dx || dw);
    const size_t one = (size_t)rows * 2 * wide * sizeof(uint16_t), tops = (size_t)rows + 2 * wide;
    const size_t words = tops + (dx ? (size_t)across * rows : 0) + (dw ? (size_t)blocks * 2 * wide : 0);  // (whole 64s)
    const size_t d_bytes = f16 ? one * (dx + dw) + words * sizeof(uint32_t) : one;
    const size_t b_bytes = bias ? ((size_t)blocks * 2 * a.n * sizeof(float) + 255) / 256 * 256 : 0;
    float *room = nullptr;
    const int32_t rc = op_room(ctx, s, d_bytes + b_bytes + (px.room > pw.room ? px.room : pw.room), &room);
    if (rc != HH_OK) return rc;
    uint8_t *at = reinterpret_cast<uint8_t *>(room);
    SlopeArgs sl = {};
    sl.dy = reinterpret_cast<const uint16_t *>(d.d_dy), sl.dy_stride = d.dy_stride;
    sl.saved = a.d_saved, sl.d = DT == HH_F16 && !dx ? nullptr : reinterpret_cast<uint16_t *>(at);
    sl.part = bias ? reinterpret_cast<float *>(at + d_bytes) : nullptr;
    sl.gate_bias = d.d_dgate_bias, sl.up_bias = d.d_dup_bias;
    sl.m = a.m, sl.n = a.n, sl.wide = wide, sl.rows = dw ? rows : a.m, sl.act = a.activation;
    sl.block_rows = block_rows;
    const dim3 grid(across * blocks);
    auto slope = [&](auto tops) {
        constexpr bool TOPS = decltype(tops)::value;
        if (block_rows == 4)
            hipLaunchKernelGGL((gated_slope_kernel<DT, 1, TOPS>), grid, dim3(256), 0, s, sl);
        else
            hipLaunchKernelGGL((gated_slope_kernel<DT, 4, TOPS>), grid, dim3(256), 0, s, sl);
        return from_hip(hipGetLastError());
    };
    int32_t e = HH_OK;
    if (f16) {
        uint8_t *d_cols = at + one * dx;
        uint32_t *next = reinterpret_cast<uint32_t *>(d_cols + one * dw);
        sl.row_top = next, sl.col_top = next + rows, next += tops;
        if (dx) sl.row_part = next, next += (size_t)across * rows;
        if (dw) sl.col_part = next;
        sl.d_cols = dw ? reinterpret_cast<uint16_t *>(d_cols) : nullptr;
        if constexpr (DT == HH_F16) e = slope(std::true_type());
        if (e == HH_OK) {
            hipLaunchKernelGGL(gated_tops_kernel, dim3((uint32_t)(tops / 32)), dim3(1024), 0, s, sl, rows, across, blocks);
            e = from_hip(hipGetLastError());
        }
    }
    if (e == HH_OK) e = slope(std::false_type());
    if (e == HH_OK && bias) {
        hipLaunchKernelGGL(gated_bias_kernel, dim3((a.n + 31) / 32, 2), dim3(1024), 0, s, sl, blocks);
        e = from_hip(hipGetLastError());
    }
    float *sums = reinterpret_cast<float *>(at + d_bytes + b_bytes);
    BackArgs p = {};
    p.cols = a.k, p.n = a.n, p.wide = wide;
    if (e == HH_OK && dx) {
        p.l[0] = reinterpret_cast<const uint16_t *>(a.d_gate), p.l[1] = reinterpret_cast<const uint16_t *>(a.d_up);
        p.l_stride[0] = a.gate_stride, p.l_stride[1] = a.up_stride;
        p.out[0] = reinterpret_cast<uint16_t *>(d.d_dx), p.out_stride[0] = d.dx_stride;
        p.d = sl.d, p.top = sl.row_top;
        p.rows = a.m, p.depth = a.n;
        e = launch_back<DT, false>(p, px, x_aligned, sums, s);
    }
    if (e == HH_OK && dw) {
        p.l[0] = reinterpret_cast<const uint16_t *>(a.d_x), p.l_stride[0] = a.x_stride;
        p.out[0] = reinterpret_cast<uint16_t *>(d.d_dgate), p.out[1] = reinterpret_cast<uint16_t *>(d.d_dup);
        p.out_stride[0] = d.dgate_stride, p.out_stride[1] = d.dup_stride;
        p.d = f16 ? sl.d_cols : sl.d, p.top = sl.col_top;
        p.rows = 2 * wide, p.depth = a.m;
        e = launch_back<DT, true>(p, pw, w_aligned, sums, s);
    }
    return e;
}

// Gradients of nothing: dx without weights' rows, the weights' without rows.
__global__ __launch_bounds__(256) void gated_zero_kernel(uint16_t *out, uint64_t stride, uint32_t rows, uint32_t cols) {
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (uint32_t c = blockIdx.x * 256 + threadIdx.x; c < cols; c += gridDim.x * 256) out[r * stride + c] = 0;
}
__global__ __launch_bounds__(256) void gated_zero_bias_kernel(float *out, uint32_t n) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) out[i] = 0.0f;
}
int32_t gated_zero(void *out, uint64_t stride, uint32_t rows, uint32_t cols, hipStream_t s) {
    if (!out || !rows || !cols) return HH_OK;
    hipLaunchKernelGGL(gated_zero_kernel, dim3(cols < 4096 ? (cols + 255) / 256 : 16, rows < 4096 ? rows : 4096), dim3(256), 0, s,
                       reinterpret_cast<uint16_t *>(out), stride, rows, cols);
    return from_hip(hipGetLastError());
}

}  // namespace
}  // namespace hh

extern "C" int32_t hh_gated_linear_backward(hh_context *ctx, const hh_gated_args *a, const hh_gated_grads *d, void *stream) {
    if (!ctx || !a || !d) return HH_ERR_INVALID_ARGUMENT;
    int32_t rc = hh::check_gated(a);
    if (rc != HH_OK) return rc;
    if (a->w_dtype == HH_INT4) return HH_ERR_UNSUPPORTED;
    if (!d->d_dgate != !d->d_dup) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)d->d_dy | (uintptr_t)d->d_dx | (uintptr_t)d->d_dgate | (uintptr_t)d->d_dup) & 1u) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)d->d_dgate_bias | (uintptr_t)d->d_dup_bias) & 3u) return HH_ERR_INVALID_ARGUMENT;
    if (a->m && a->n && (!d->d_dy || !a->d_saved || d->dy_stride < a->n)) return HH_ERR_INVALID_ARGUMENT;
    if ((d->d_dx && d->dx_stride < a->k) || (d->d_dgate && (d->dgate_stride < a->k || d->dup_stride < a->k)))
        return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (!a->m || !a->n) {
        rc = hh::gated_zero(d->d_dx, d->dx_stride, a->m, a->k, s);
        if (rc == HH_OK) rc = hh::gated_zero(d->d_dgate, d->dgate_stride, a->n, a->k, s);
        if (rc == HH_OK) rc = hh::gated_zero(d->d_dup, d->dup_stride, a->n, a->k, s);
        for (float *b : {d->d_dgate_bias, d->d_dup_bias})
            if (rc == HH_OK && b && a->n) {
                hipLaunchKernelGGL(hh::gated_zero_bias_kernel, dim3((a->n + 255) / 256), dim3(256), 0, s, b, a->n);
                rc = hh::from_hip(hipGetLastError());
            }
        return rc;
    }
    if ((!d->d_dx || !a->k) && (!d->d_dgate || !a->k) && !d->d_dgate_bias && !d->d_dup_bias) return HH_OK;
    return a->dtype == HH_BF16 ? hh::gated_backward<HH_BF16>(ctx, *a, *d, s) : hh::gated_backward<HH_F16>(ctx, *a, *d, s);
}
