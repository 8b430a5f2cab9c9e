// Layer norm and root mean square norm with their gradients (hh_norm,
// hh_norm_backward; rules: haagenti_hip.h).
//
// With g = dy w, h = (x - mean) rstd (mean 0 in the rms form):
//   y  = h w + b
//   dx = rstd (g - mean(g) - h mean(g h)) + add   (no mean(g) in the rms form)
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// Bound by memory: x in and y out; dy, x (and add) in and dx out.  A row lies
// in the registers of W waves, C pieces of 16 bytes a lane, so it is read once
// and its variance is summed about its mean, in f32.  The backward pass
// recomputes both from x, which it reads anyway: two sums over registers cost
// less than statistics kept, passed and checked.  W = 1 needs no LDS and no
// barrier; more waves take rows too long for one wave, and few rows.  Kernels'
// times, by a profiler: 8192 rows of 4096 bf16 24 us, 134 MB at 5.6 TB/s;
// gradients with add 57 us, 268 MB at 4.7 TB/s, and 6 us to join the workgroups'
// sums; 8 rows 3.6 us.
//
// The loops ask for the next row before they work on this one, but the compiler
// waits for it at once (the request is under a condition, and what comes after
// must hold either way): what hides a row's loads are the CU's other waves (at
// 4096 values 16 forward and 8 backward).
#include "layer_ops.hpp"

namespace hh {
namespace {

struct NormArgs {
    hh_norm_args a;
    const void *dy, *add;
    uint64_t dy_stride, add_stride;
    float *dw, *db;       // the sums' outputs, or null
    float *part;          // [workgroup][2][n]: dw's and db's sums, where rows are many
    int w32;              // weight and bias are f32
};

template <int XT>
struct Elem {
    static constexpr int V = XT == HH_F32 ? 4 : 8;      // values to 16 bytes
    static constexpr int S = XT == HH_F32 ? 4 : 2;
};
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));

// Value e of 16 bytes.
template <int XT>
__device__ __forceinline__ float value(const u32x4 &r, int e) {
    if constexpr (XT == HH_F32)
        return __uint_as_float(r[e]);
    else
        return half_to_f32<XT>((r[e >> 1] >> (16 * (e & 1))) & 0xffffu);
}
template <int XT>
__device__ __forceinline__ u32x4 packed(const float (&v)[Elem<XT>::V]) {
    u32x4 r;
    if constexpr (XT == HH_F32) {
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = __float_as_uint(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = f32_to_half<XT>(v[2 * e]) | f32_to_half<XT>(v[2 * e + 1]) << 16;
    }
    return r;
}
// 16 bytes of a row of n at value `at`, of which `left` are the row's.  In two
// parts: a load without a condition, of the row's last 16 bytes past their
// start, so that many are under way at once (with the ends loaded a value at a
// time 8192 rows of 4093 bfloat16 took 39 us and their gradients 87, so 32 and
// 65); and, once it is here, its values moved to their places, zeros past them.
template <int XT>
__device__ __forceinline__ u32x4 load16(const void *row, uint32_t at, uint32_t n) {
    const uint8_t *p = reinterpret_cast<const uint8_t *>(row) + (uint64_t)min(at, n - Elem<XT>::V) * Elem<XT>::S;
    return *reinterpret_cast<const u32x4_at2 *>(p);
}
template <int XT>
__device__ __forceinline__ u32x4 ended(u32x4 r, int32_t left) {
    constexpr int V = Elem<XT>::V;
    if (left >= V) return r;
    if (left <= 0) return u32x4{0, 0, 0, 0};
    const uint32_t halves = (V - left) * (8 / V);
    if (halves & 4u) r = u32x4{r[2], r[3], 0, 0};
    if (halves & 2u) r = u32x4{r[1], r[2], r[3], 0};
    if (halves & 1u) r = u32x4{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
    return r;
}
// A row of less than 16 bytes.
template <int XT>
__device__ __forceinline__ u32x4 load_few(const void *row, uint32_t at, int32_t left) {
    const uint8_t *p = reinterpret_cast<const uint8_t *>(row) + (uint64_t)at * Elem<XT>::S;
    u32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < Elem<XT>::V; e++)
        if (e < left) {
            if constexpr (XT == HH_F32)
                r[e] = reinterpret_cast<const uint32_t *>(p)[e];
            else
                r[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[e] << (16 * (e & 1));
        }
    return r;
}
template <int XT>
__device__ __forceinline__ u32x4 row16(const void *row, uint32_t at, int32_t left, uint32_t n) {
    return n < Elem<XT>::V ? load_few<XT>(row, at, left) : ended<XT>(load16<XT>(row, at, n), left);
}
template <int XT>
__device__ __forceinline__ void store16(void *row, uint32_t at, int32_t left, const u32x4 &r) {
    uint8_t *p = reinterpret_cast<uint8_t *>(row) + (uint64_t)at * Elem<XT>::S;
    if (left >= Elem<XT>::V) {
        *reinterpret_cast<u32x4_at2 *>(p) = r;
        return;
    }
#pragma unroll
    for (int e = 0; e < Elem<XT>::V; e++)
        if (e < left) {
            if constexpr (XT == HH_F32)
                reinterpret_cast<uint32_t *>(p)[e] = r[e];
            else
                reinterpret_cast<uint16_t *>(p)[e] = (uint16_t)(r[e >> 1] >> (16 * (e & 1)));
        }
}
// V parameters (weight or bias) from column `at` on, `none` where there are
// none and past the row.
template <int XT>
__device__ __forceinline__ void params(const void *p, int w32, uint32_t at, int32_t left, uint32_t n, float none,
                                       float (&v)[Elem<XT>::V]) {
    constexpr int V = Elem<XT>::V;
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = none;
    if (!p) return;
    if (XT != HH_F32 && !w32) {
        const u32x4 r = row16<XT>(p, at, left, n);
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = e < left ? value<XT>(r, e) : none;
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            const u32x4 r = row16<HH_F32>(p, at + 4 * i, left - 4 * i, n);
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * i + e] = 4 * i + e < left ? __uint_as_float(r[e]) : none;
        }
    }
}

// Sums over the W waves of a row (by way of `lds`, which takes turns: one
// barrier a sum).
template <int W, int G, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*lds)[W * G][3], int &turn) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
    if constexpr (W > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63u) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) lds[turn][wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) v[i] += lds[turn][wave / W * W + w][i];
        }
        turn ^= 1;
    }
}

// A row's values less its mean (0 in the rms form), zeros past the row.
template <int XT, int W, int G, int C>
__device__ __forceinline__ void off_mean(const NormArgs &p, const u32x4 (&x)[C], const int32_t (&left)[C], float inv,
                                         float (*lds)[W * G][3], int &turn, float (&d)[C][Elem<XT>::V]) {
    constexpr int V = Elem<XT>::V;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < V; e++) d[c][e] = value<XT>(x[c], e);
    if (p.a.kind != HH_NORM_LAYER) return;
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < V; e++) s[0] += d[c][e];
    row_sum<W, G>(s, lds, turn);
    const float mean = s[0] * inv;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < V; e++) d[c][e] -= mean;
    if (p.a.n == C * 64 * W * V) return;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < V; e++)
            if (e >= left[c]) d[c][e] = 0.0f;
}

// W waves to a row, G rows to a workgroup at a time.  All of a workgroup's
// waves go around together (they meet at barriers where W > 1); past the last
// row they read that row again and keep nothing of it.
template <int XT, int W, int G, int C>
__global__ __launch_bounds__(64 * W * G) void norm_kernel(const NormArgs p) {
    constexpr int V = Elem<XT>::V, T = 64 * W;
    __shared__ float lds[2][W * G][3];
    const uint32_t t = threadIdx.x % T, group = threadIdx.x / T, step = gridDim.x * G;
    const hh_norm_args &a = p.a;
    const float inv = 1.0f / (float)a.n;
    const bool few = C == 1 && W == 1 && a.n < V;
    int32_t left[C];
    float w[C][V], b[C][V];
#pragma unroll
    for (int c = 0; c < C; c++) {
        left[c] = (int32_t)a.n - (int32_t)((c * T + t) * V);
        params<XT>(a.d_weight, p.w32, (c * T + t) * V, left[c], a.n, 1.0f, w[c]);
        params<XT>(a.d_bias, p.w32, (c * T + t) * V, left[c], a.n, 0.0f, b[c]);
    }
    auto fetch = [&](uint32_t row, u32x4 (&x)[C]) {
        const uint8_t *at = reinterpret_cast<const uint8_t *>(a.d_x) + (uint64_t)min(row, a.rows - 1) * a.x_stride * Elem<XT>::S;
        if (few) {
            x[0] = load_few<XT>(at, t * V, left[0]);
            return;
        }
#pragma unroll
        for (int c = 0; c < C; c++) x[c] = load16<XT>(at, (c * T + t) * V, a.n);
    };
    u32x4 x[C], next[C];
    int turn = 0;
    fetch(blockIdx.x * G + group, x);
    for (uint32_t base = blockIdx.x * G; base < a.rows; base += step) {
        const uint32_t row = base + group;
        if (base + step < a.rows) fetch(row + step, next);
        if (!few)
#pragma unroll
            for (int c = 0; c < C; c++) x[c] = ended<XT>(x[c], left[c]);
        float d[C][V], s[1] = {0.0f};
        off_mean<XT, W, G, C>(p, x, left, inv, lds, turn, d);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < V; e++) s[0] = fmaf(d[c][e], d[c][e], s[0]);
        row_sum<W, G>(s, lds, turn);
        const float rstd = 1.0f / sqrtf(s[0] * inv + a.eps);
        uint8_t *to = reinterpret_cast<uint8_t *>(a.d_y) + (uint64_t)row * a.y_stride * Elem<XT>::S;
        if (row < a.rows)
#pragma unroll
            for (int c = 0; c < C; c++) {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; e++) y[e] = fmaf(d[c][e] * rstd, w[c][e], b[c][e]);
                store16<XT>(to, (c * T + t) * V, left[c], packed<XT>(y));
            }
#pragma unroll
        for (int c = 0; c < C; c++) x[c] = next[c];
    }
}

// The gradients; dw's and db's sums over the workgroup's rows stay in
// registers, are joined over its G rows in LDS and written to `part`.
template <int XT, int W, int G, int C>
__global__ __launch_bounds__(64 * W * G) void norm_backward_kernel(const NormArgs p) {
    constexpr int V = Elem<XT>::V, T = 64 * W;
    constexpr bool AHEAD = C * V <= 16;   // the next row asked for early and the weights in registers, where these allow
    __shared__ float lds[2][W * G][3];
    __shared__ __align__(16) float join[G > 1 ? G : 1][G > 1 ? T * 4 : 4];
    const uint32_t t = threadIdx.x % T, group = threadIdx.x / T, step = gridDim.x * G;
    const hh_norm_args &a = p.a;
    const float inv = 1.0f / (float)a.n;
    const bool few = C == 1 && W == 1 && a.n < V;
    int32_t left[C];
    float sw[C][V], sb[C][V], held[AHEAD ? C : 1][V];
#pragma unroll
    for (int c = 0; c < C; c++) {
        left[c] = (int32_t)a.n - (int32_t)((c * T + t) * V);
        if (AHEAD) params<XT>(a.d_weight, p.w32, (c * T + t) * V, left[c], a.n, 1.0f, held[AHEAD ? c : 0]);
#pragma unroll
        for (int e = 0; e < V; e++) sw[c][e] = 0.0f, sb[c][e] = 0.0f;
    }
    struct Row {
        u32x4 x[C], dy[C], add[C];
    };
    auto fetch = [&](uint32_t row, Row &r) {
        const uint64_t i = min(row, a.rows - 1);
        const uint8_t *xr = reinterpret_cast<const uint8_t *>(a.d_x) + i * a.x_stride * Elem<XT>::S;
        const uint8_t *dr = reinterpret_cast<const uint8_t *>(p.dy) + i * p.dy_stride * Elem<XT>::S;
        const uint8_t *ar = reinterpret_cast<const uint8_t *>(p.add) + i * p.add_stride * Elem<XT>::S;
        if (few) {
            r.x[0] = load_few<XT>(xr, t * V, left[0]), r.dy[0] = load_few<XT>(dr, t * V, left[0]);
            if (p.add) r.add[0] = load_few<XT>(ar, t * V, left[0]);
            return;
        }
#pragma unroll
        for (int c = 0; c < C; c++) r.x[c] = load16<XT>(xr, (c * T + t) * V, a.n);
#pragma unroll
        for (int c = 0; c < C; c++) r.dy[c] = load16<XT>(dr, (c * T + t) * V, a.n);
        if (p.add)
#pragma unroll
            for (int c = 0; c < C; c++) r.add[c] = load16<XT>(ar, (c * T + t) * V, a.n);
    };
    auto weights = [&](int c, float (&w)[V]) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int e = 0; e < V; e++) w[e] = held[c][e];
        } else {
            params<XT>(a.d_weight, p.w32, (c * T + t) * V, left[c], a.n, 1.0f, w);
        }
    };
    int turn = 0;
    Row now, next;
    if (AHEAD) fetch(blockIdx.x * G + group, now);
    for (uint32_t base = blockIdx.x * G; base < a.rows; base += step) {
        const uint32_t row = base + group;
        if (!AHEAD)
            fetch(row, now);
        else if (base + step < a.rows)
            fetch(row + step, next);
        if (!few)
#pragma unroll
            for (int c = 0; c < C; c++) {
                now.x[c] = ended<XT>(now.x[c], left[c]), now.dy[c] = ended<XT>(now.dy[c], left[c]);
                if (p.add) now.add[c] = ended<XT>(now.add[c], left[c]);
            }
        float d[C][V], dy[C][V];
        off_mean<XT, W, G, C>(p, now.x, left, inv, lds, turn, d);
        float s[3] = {0.0f, 0.0f, 0.0f};  // of (x - mean)^2, g, g (x - mean)
#pragma unroll
        for (int c = 0; c < C; c++) {
            float w[V];
            weights(c, w);
#pragma unroll
            for (int e = 0; e < V; e++) {
                dy[c][e] = value<XT>(now.dy[c], e);
                const float g = dy[c][e] * w[e];
                s[0] = fmaf(d[c][e], d[c][e], s[0]);
                s[1] += g;
                s[2] = fmaf(g, d[c][e], s[2]);
            }
        }
        row_sum<W, G>(s, lds, turn);
        // dx = g rstd - mean(g) rstd - (x - mean) rstd^3 mean(g (x - mean))
        const float rstd = 1.0f / sqrtf(s[0] * inv + a.eps);
        const float mg = a.kind == HH_NORM_LAYER ? s[1] * inv * rstd : 0.0f, mgd = s[2] * inv * rstd * rstd * rstd;
        uint8_t *to = reinterpret_cast<uint8_t *>(a.d_y) + (uint64_t)row * a.y_stride * Elem<XT>::S;
        if (row < a.rows)
#pragma unroll
            for (int c = 0; c < C; c++) {
                float w[V], v[V];
                weights(c, w);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    sw[c][e] = fmaf(dy[c][e] * rstd, d[c][e], sw[c][e]);
                    sb[c][e] += dy[c][e];
                    v[e] = fmaf(dy[c][e] * w[e], rstd, fmaf(-d[c][e], mgd, -mg));
                    if (p.add) v[e] += value<XT>(now.add[c], e);
                }
                store16<XT>(to, (c * T + t) * V, left[c], packed<XT>(v));
            }
        if (AHEAD) now = next;
    }
    if (!p.part) return;
    // sums of dw, then of db: joined over the groups in a fixed order
    float *out = p.part + (uint64_t)blockIdx.x * 2 * a.n;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (!(k ? p.db : p.dw)) continue;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int q = 0; q < V / 4; q++) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = k ? sb[c][4 * q + e] : sw[c][4 * q + e];
                if constexpr (G > 1) {
                    __syncthreads();
                    *reinterpret_cast<f32x4 *>(&join[group][t * 4]) = v;
                    __syncthreads();
                    if (group) continue;
#pragma unroll
                    for (int i = 1; i < G; i++) v += *reinterpret_cast<const f32x4 *>(&join[i][t * 4]);
                }
                const uint32_t at = (c * T + t) * V + 4 * q;
                float *o = out + (uint64_t)k * a.n + at;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (at + e < a.n) o[e] = v[e];
            }
    }
}

// The workgroups' sums, in order: 32 columns to a workgroup, its 32 rows of
// threads over every 32nd of them.
__global__ __launch_bounds__(1024) void norm_join_kernel(const NormArgs p, uint32_t parts) {
    __shared__ float sum[32][33];
    const uint32_t col = blockIdx.x * 32 + (threadIdx.x & 31u), q = threadIdx.x >> 5, k = blockIdx.y;
    float *out = k ? p.db : p.dw;
    if (!out) return;
    float s = 0.0f;
    if (col < p.a.n)
        for (uint32_t i = q; i < parts; i += 32) s += p.part[((uint64_t)i * 2 + k) * p.a.n + col];
    sum[q][threadIdx.x & 31u] = s;
    __syncthreads();
    if (q || col >= p.a.n) return;
    for (int i = 1; i < 32; i++) s += sum[i][threadIdx.x & 31u];
    out[col] = s;
}
// No rows: sums of nothing.
__global__ __launch_bounds__(256) void norm_zero_kernel(const NormArgs p) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= p.a.n) return;
    if (p.dw) p.dw[i] = 0.0f;
    if (p.db) p.db[i] = 0.0f;
}

// Waves to a row, rows to a workgroup at a time, pieces to a lane, workgroups
// to a CU.  Few pieces to a lane, so few registers and many waves: when this was
// chosen a call of layer norm of 8192 x 4096 bf16 took 25 us with 4 waves of 2
// pieces (30 with 2 of 4, 38 with one of 8), of its gradients 70 (96, 127; now
// 52, with add 62 to 67).  Rows of more than 1024 pieces need 16 waves, whose
// workgroups leave a lane 128 registers: too few for the gradients, which spill
// 44 to 624 bytes a lane there (the forward pass 24 with 4 pieces).  Calls with
// add: 8192 x 12288 bf16 710 us (1.1 TB/s; forward 97, 4.2 TB/s), 4096 x 16384
// 408 (51); 2048 x 16384 f32 without add 275 (46).
struct NormPlan {
    int w, g, c;
    uint32_t grid;
};
NormPlan plan_norm(const hh_norm_args &a, int cus, bool back) {
    const uint32_t v = a.dtype == HH_F32 ? 4 : 8, pieces = (a.n + v - 1) / v;
    NormPlan pl;
    uint32_t per_cu;
    if (pieces <= 128)
        pl.w = 1, pl.g = 4, pl.c = pieces <= 64 ? 1 : 2, per_cu = back ? 2 : 4;
    else if (pieces <= 512)
        pl.w = 4, pl.g = 1, pl.c = pieces <= 256 ? 1 : 2, per_cu = back ? 2 : 4;
    else if (pieces <= 1024)
        pl.w = 8, pl.g = 1, pl.c = 2, per_cu = back ? 1 : 2;
    else
        pl.w = 16, pl.g = 1, pl.c = pieces <= 2048 ? 2 : 4, per_cu = 1;
    const uint32_t need = (a.rows + pl.g - 1) / pl.g, most = (uint32_t)cus * per_cu;
    pl.grid = need < most ? need : most;
    return pl;
}
template <int XT, int W, int G, int C>
void launch_one(const NormArgs &p, const NormPlan &pl, bool back, hipStream_t s) {
    if (back)
        hipLaunchKernelGGL((norm_backward_kernel<XT, W, G, C>), dim3(pl.grid), dim3(64 * W * G), 0, s, p);
    else
        hipLaunchKernelGGL((norm_kernel<XT, W, G, C>), dim3(pl.grid), dim3(64 * W * G), 0, s, p);
}
template <int XT>
int32_t launch_norm(const NormArgs &p, const NormPlan &pl, bool back, hipStream_t s) {
    switch (pl.w * 10 + pl.c) {
        case 11: launch_one<XT, 1, 4, 1>(p, pl, back, s); break;
        case 12: launch_one<XT, 1, 4, 2>(p, pl, back, s); break;
        case 41: launch_one<XT, 4, 1, 1>(p, pl, back, s); break;
        case 42: launch_one<XT, 4, 1, 2>(p, pl, back, s); break;
        case 82: launch_one<XT, 8, 1, 2>(p, pl, back, s); break;
        case 162: launch_one<XT, 16, 1, 2>(p, pl, back, s); break;
        default: launch_one<XT, 16, 1, 4>(p, pl, back, s); break;
    }
    return from_hip(hipGetLastError());
}

int32_t check_norm(const hh_norm_args *a, uint32_t *size) {
    if (a->dtype != HH_F32 && a->dtype != HH_F16 && a->dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (a->kind != HH_NORM_LAYER && a->kind != HH_NORM_RMS) return HH_ERR_UNSUPPORTED;
    if (a->weight_dtype != a->dtype && a->weight_dtype != HH_F32) return HH_ERR_UNSUPPORTED;
    if (a->rows >= 1u << 31) return HH_ERR_INVALID_ARGUMENT;
    if (a->n > (a->dtype == HH_F32 ? 16384u : 32768u)) return HH_ERR_UNSUPPORTED;
    if (!(a->eps >= 0.0f)) return HH_ERR_INVALID_ARGUMENT;
    *size = a->dtype == HH_F32 ? 4 : 2;
    const uint32_t ws = a->weight_dtype == HH_F32 ? 4 : 2;
    if (a->rows && a->n && (!a->d_x || !a->d_y)) return HH_ERR_INVALID_ARGUMENT;
    if ((((uintptr_t)a->d_x | (uintptr_t)a->d_y) & (*size - 1)) || (((uintptr_t)a->d_weight | (uintptr_t)a->d_bias) & (ws - 1)))
        return HH_ERR_INVALID_ARGUMENT;
    if (a->x_stride < a->n || a->y_stride < a->n) return HH_ERR_INVALID_ARGUMENT;
    return HH_OK;
}

int32_t launch_type(const NormArgs &p, const NormPlan &pl, bool back, hipStream_t s) {
    switch (p.a.dtype) {
        case HH_F32: return launch_norm<HH_F32>(p, pl, back, s);
        case HH_F16: return launch_norm<HH_F16>(p, pl, back, s);
        default: return launch_norm<HH_BF16>(p, pl, back, s);
    }
}

}  // namespace
}  // namespace hh

extern "C" int32_t hh_norm(hh_context *ctx, const hh_norm_args *a, void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    uint32_t size;
    const int32_t rc = hh::check_norm(a, &size);
    if (rc != HH_OK) return rc;
    if (!a->rows || !a->n) return HH_OK;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hh::NormArgs p = {};
    p.a = *a;
    p.w32 = a->weight_dtype == HH_F32;
    return hh::launch_type(p, hh::plan_norm(*a, ctx->num_cus > 0 ? ctx->num_cus : 256, false), false,
                           reinterpret_cast<hipStream_t>(stream));
}

extern "C" int32_t hh_norm_backward(hh_context *ctx, const hh_norm_args *a, const hh_norm_grads *d, void *stream) {
    if (!ctx || !a || !d) return HH_ERR_INVALID_ARGUMENT;
    uint32_t size;
    const int32_t rc = hh::check_norm(a, &size);
    if (rc != HH_OK) return rc;
    if (!a->n) return HH_OK;
    if (a->rows && !d->d_dy) return HH_ERR_INVALID_ARGUMENT;
    if ((((uintptr_t)d->d_dy | (uintptr_t)d->d_add) & (size - 1)) || (((uintptr_t)d->d_dweight | (uintptr_t)d->d_dbias) & 3u))
        return HH_ERR_INVALID_ARGUMENT;
    if (d->dy_stride < a->n || (d->d_add && d->add_stride < a->n)) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    hh::NormArgs p = {};
    p.a = *a;
    p.w32 = a->weight_dtype == HH_F32;
    p.dy = d->d_dy, p.add = d->d_add, p.dy_stride = d->dy_stride, p.add_stride = d->add_stride;
    p.dw = reinterpret_cast<float *>(d->d_dweight), p.db = reinterpret_cast<float *>(d->d_dbias);
    const bool sums = p.dw || p.db;
    if (!a->rows) {
        if (sums) hipLaunchKernelGGL(hh::norm_zero_kernel, dim3((a->n + 255) / 256), dim3(256), 0, s, p);
        return hh::from_hip(hipGetLastError());
    }
    const hh::NormPlan pl = hh::plan_norm(*a, ctx->num_cus > 0 ? ctx->num_cus : 256, true);
    if (sums) {
        const int32_t e = hh::op_room(ctx, s, (size_t)pl.grid * 2 * a->n * sizeof(float), &p.part);
        if (e != HH_OK) return e;
    }
    const int32_t e = hh::launch_type(p, pl, true, s);
    if (e != HH_OK || !sums) return e;
    hipLaunchKernelGGL(hh::norm_join_kernel, dim3((a->n + 31) / 32, 2), dim3(1024), 0, s, p, pl.grid);
    return hh::from_hip(hipGetLastError());
}
