// Attention over the paged 8-bit cache (layout and rules: haagenti_hip.h).
//
// With column c = (new row i, head g of the group), i = c / group, both
// kernels compute, per cache head,
//   S^T = K Q^T     codes (exact in f16) times f16 queries, f32
//   z   = S^T (scale of K's block) (softmax scale) log2(e)
//   w   = z + log2(scale of V's block)
//   m, l, M: running maximum of z, sum of 2^(z - m), running maximum of w,
//   O^T += V^T P^T  codes times f16 P = 2^(w - M), O in units of 2^M, f32,
// and the output is 2^(M - m) O / l.  Both maxima are the column's own, over
// tokens that it sees, so whatever the scales are, its largest P is at least 1:
// a P keeps f16's 11 bits down to 2^-14 and is off by at most 2^-25 below (of
// terms that small beside the column's largest).  The step kernel, which
// memory bounds, adds the rest of P as a second f16 (22 bits; 48 requests 93.1
// us, 92.2 without it, 131,001 tokens 52.3 and 51.8); for the tile kernel that
// is half as much again of the matrix products (two prompts 573 us, 440
// without) for errors below half a unit of its outputs.
// P's exponent is z - m + share, share = log2(scale of V's block) - rise, rise
// standing for M - m; the sum l takes the share out again per 16 tokens (a
// share below 2^-40 counts as 2^-40: such a P is 0 in f16 anyway, and l keeps
// its tokens).  m and M follow their maxima only when these pass them by 8, so
// P < 256 and the accumulators are seldom rescaled.  Powers of two are the
// hardware's, to a unit in the last place.
// Tokens lie on the first product's rows, so its accumulators hold, for one
// column per lane, just the tokens that the lane supplies to the second
// product's P^T operand: P never moves between lanes.  Which token a row
// stands for is free as long as V's operand agrees, and is chosen so that V's
// operands are contiguous bytes of the cache.  The cache's codes c become the
// f16 numbers 1024 + c by byte permutation, less 1152 by one packed add.
//
// bf16 queries are scaled by a power of two, to a largest magnitude of 2^14 to
// 2^15 per row, before they become f16: exact down to 2^-31 of the largest, off
// by at most 2^-39 of it below.
#include "layer_ops.hpp"

namespace hh {
namespace {

struct AttnArgs {
    hh_kv_cache cache;
    hh_kv_attention_args a;
    uint32_t group;      // q heads per cache head
    uint32_t bs_log;     // block_size = 1 << bs_log
    uint32_t block_step; // bytes of a block: kv_heads * block_size * head_dim
    uint32_t splits;     // of a request's tokens, in chunks of:
    uint32_t chunk;      // a multiple of 256
    uint32_t tiles;      // column tiles per request (tile kernel)
    uint32_t small;      // requests with at most this many columns are the step kernel's
    uint32_t cols;       // most columns of such a request
    float *part_o;       // [request][head][split][cols][dim]
    float *part_ml;      // [request][head][split][cols][m, l, rise]
};

constexpr float kLog2e = 1.44269504088896340736f;

// 4 codes as 4 f16 numbers -127..127.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias);
}
__device__ __forceinline__ f16x8 codes8_to_f16(uint32_t a, uint32_t b) {
    u32x4 v;
    uint32_t x, y;
    codes_to_f16(a, x, y);
    v[0] = x, v[1] = y;
    codes_to_f16(b, x, y);
    v[2] = x, v[3] = y;
    return __builtin_bit_cast(f16x8, v);
}

// One request's part of the call.
struct Request {
    int32_t q0, rows, kv_len, seen;  // seen: tokens within the call's bounds
};
__device__ __forceinline__ Request request_of(const AttnArgs &p, uint32_t r) {
    Request q;
    q.q0 = p.a.d_start[r];
    q.rows = p.a.d_start[r + 1] - q.q0;
    q.kv_len = p.a.d_kv_len[r];
    const uint64_t room = min((uint64_t)p.a.max_kv, (uint64_t)p.a.table_width * p.cache.block_size);
    q.seen = (int32_t)min((uint64_t)max(q.kv_len, 0), room);
    if (q.q0 < 0 || q.rows < 0 || (uint32_t)q.q0 > p.a.tokens || (uint32_t)q.rows > p.a.tokens - (uint32_t)q.q0) q.rows = 0;
    return q;
}
__device__ __forceinline__ uint32_t columns_of(const AttnArgs &p, const Request &q) {
    return min((uint32_t)q.rows, p.a.max_q) * p.group;
}
// Tokens that new row i sees.
__device__ __forceinline__ int32_t limit_of(const Request &q, int32_t i) {
    return max(0, min(q.seen, q.kv_len - q.rows + i + 1));
}

// The table's entry for a token, or -1 past the end.
__device__ __forceinline__ int32_t block_of(const AttnArgs &p, const int32_t *table, int32_t tok, int32_t end) {
    if (tok >= end) return -1;
    return table[(uint32_t)tok >> p.bs_log];
}
__device__ __forceinline__ bool held(const AttnArgs &p, int32_t id) { return (uint32_t)id < p.cache.num_blocks; }
constexpr float kSlack = 8.0f, kNear = 20.0f;

// What a V scale does to the exponent.  Shares of scales that the column
// doesn't see may be large: of no use, but finite.
__device__ __forceinline__ float share_of(float log_vs, float rise) {
    const float s = log_vs - rise;
    return s > -40.0f ? fminf(s, 300.0f) : -40.0f;
}

// The larger of lanes 32 (16) apart, by a swap of register halves (rows).
__device__ __forceinline__ float max_across_32(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float max_across_16(float v) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// A maximum to subtract, where there may be none.
__device__ __forceinline__ float base_of(float top) { return top == -__builtin_inff() ? 0.0f : top; }

// O's unit in units of 2^top, a common m; -inf where there is none.
__device__ __forceinline__ float unit_of(float m, float rise, float top) {
    return rise < __builtin_inff() ? m - top + rise : -__builtin_inff();
}

// A column's running maxima.  rise is infinite while no token seen has a scale
// above 0; O's unit is 2^(m + rise), and big is that sum for comparing.
struct Tops {
    float m = -__builtin_inff(), big = -__builtin_inff(), rise = __builtin_inff();
    __device__ __forceinline__ bool passed(float zm, float wm) const { return zm > m + kSlack || wm > big + kSlack; }
    // Takes new maxima where they pass; what that does to l and to O.
    __device__ __forceinline__ void take(float zm, float wm, float &of_l, float &of_o) {
        const float mn = zm > m + kSlack ? zm : m, bn = wm > big + kSlack ? wm : big;
        const float rn = bn > -__builtin_inff() ? bn - mn : __builtin_inff();
        of_l = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
        of_o = big > -__builtin_inff() ? __builtin_amdgcn_exp2f((m - mn) + (rise - rn)) : 1.0f;
        m = mn, big = bn, rise = rn;
    }
    // Moves both to a new M, as far as that lies above the old.
    __device__ __forceinline__ float move(float wm) {
        const float mn = wm > big + kSlack ? m + (wm - big) : m, of = __builtin_amdgcn_exp2f(m - mn);
        if (wm > big + kSlack) big = wm;
        m = mn;
        return of;
    }
};
// The root of 2^rise (the power itself may leave f32's range where the output
// doesn't); 0 where there is none.
__device__ __forceinline__ float half_rise(float rise) {
    return rise < __builtin_inff() ? __builtin_amdgcn_exp2f(0.5f * rise) : 0.0f;
}

// N f16 fragments of 8 dimensions of a query row, fragment f at dimension
// dim(f), as f16 scaled by a power of two of the row; returns what undoes the
// scaling.  `join` makes a lane's largest magnitude the row's; `sign` (of the
// softmax scale) goes into the row, so that scores are scaled by positives.
template <int DT, int N, typename Dim, typename Join>
__device__ __forceinline__ float load_query(const uint16_t *row, bool wide, float sign, f16x8 (&q)[N], Dim dim, Join join) {
    u32x4 raw[N];
    float top = 0.0f;
#pragma unroll
    for (int f = 0; f < N; f++) {
        raw[f] = u32x4{};
        if (row) {
            const uint16_t *at = row + dim(f);
            if (wide) {
                raw[f] = *reinterpret_cast<const u32x4 *>(at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) raw[f][e] = (uint32_t)at[2 * e] | (uint32_t)at[2 * e + 1] << 16;
            }
        }
        if constexpr (DT == HH_F16) q[f] = __builtin_bit_cast(f16x8, raw[f]) * (_Float16)sign;
    }
    if constexpr (DT == HH_F16) return 1.0f;
#pragma unroll
    for (int f = 0; f < N; f++)
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(half_to_f32<DT>((raw[f][e >> 1] >> (16 * (e & 1))) & 0xffffu)));
    const int ex = (int)(__float_as_uint(join(top)) >> 23);
    const int by = ex == 255 ? 0 : min(127 + 14 - ex, 127);  // infinities stay; 2^127 is the largest factor
    const float down = ldexpf(sign, by), up = ldexpf(1.0f, -by);
#pragma unroll
    for (int f = 0; f < N; f++)
#pragma unroll
        for (int e = 0; e < 8; e++)
            q[f][e] = (_Float16)(half_to_f32<DT>((raw[f][e >> 1] >> (16 * (e & 1))) & 0xffffu) * down);
    return up;
}

// Zeros to rows from .. to - 1 of `heads` heads from h on (a workgroup's work).
template <int D>
__device__ __forceinline__ void zero_rows(const AttnArgs &p, uint32_t from, uint32_t to, uint32_t h, uint32_t heads) {
    for (uint32_t t = from; t < to; t++) {
        uint16_t *row = reinterpret_cast<uint16_t *>(p.a.d_out) + t * p.a.out_token_stride + h * p.a.out_head_stride;
        for (uint32_t e = threadIdx.x; e < heads * D; e += blockDim.x) row[e / D * p.a.out_head_stride + e % D] = 0;
    }
}
// Rows before the first request's and past the last one's.
template <int D>
__device__ __forceinline__ void zero_ends(const AttnArgs &p) {
    zero_rows<D>(p, 0, (uint32_t)min((int64_t)p.a.tokens, max((int64_t)0, (int64_t)p.a.d_start[0])), 0, p.a.q_heads);
    zero_rows<D>(p, (uint32_t)max(0, p.a.d_start[p.a.requests]), p.a.tokens, 0, p.a.q_heads);
}
// A call without requests.
template <int D>
__global__ __launch_bounds__(256) void attn_zero_kernel(const AttnArgs p) {
    for (uint32_t t = blockIdx.x; t < p.a.tokens; t += gridDim.x) zero_rows<D>(p, t, t + 1, 0, p.a.q_heads);
}

// 4 consecutive dimensions of an output row.
template <int DT>
__device__ __forceinline__ void store4(uint16_t *to, bool wide, const float *v) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = f32_to_half<DT>(v[i]);
    if (wide) {
        *reinterpret_cast<u32x2 *>(to) = u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) to[i] = (uint16_t)h[i];
    }
}

// ---------------------------------------------------------------- few columns
//
// A step of a running request: at most 16 columns, one 16 x 16 x 32 tile
// wide.  Bound by reading the codes once: 131,001 tokens of 8 heads of 128
// dimensions (268 MB) take 43 us (6.2 TB/s) and 8 to join, 48 requests of 100
// to 8000 tokens (424 MB) 87 and 5 (chunks end unevenly).  A workgroup takes one chunk of a
// request's tokens for one cache head, its 4 waves every fourth 64 tokens
// straight from memory to registers; their results are joined in LDS, the
// chunks' by attn_join_kernel.
//
// In a wave's 64 tokens, run u (16 tokens, in one block) supplies rows
// 4u..4u+3 of each of the 4 row tiles: tile t's row 4u + i is token
// 16u + 4t + i, so that lane (column, u) ends with tokens 16u..16u+15 of its
// column, and V's operand is 16 contiguous codes of a dimension.

template <int DT, int D>
__global__ __launch_bounds__(256, D <= 128 ? 3 : 1) void attn_step_kernel(const AttnArgs p) {
    constexpr int KS = D / 32, VT = D / 16, KW = D / 16;  // k steps, V tiles, 4-byte words of K per lane and row
    __shared__ __align__(16) float lds_o[2][16][D + 4];
    __shared__ float lds_ml[4][16][3];
    const uint32_t r = blockIdx.x / p.splits, split = blockIdx.x % p.splits, h = blockIdx.y;
    if (r == p.a.requests - 1 && split == 0 && h == 0) zero_ends<D>(p);
    const Request rq = request_of(p, r);
    if (split == 0 && (uint32_t)rq.rows > p.a.max_q)  // rows beyond the call's bound
        zero_rows<D>(p, (uint32_t)rq.q0 + p.a.max_q, (uint32_t)(rq.q0 + rq.rows), h * p.group, p.group);
    const uint32_t cols = columns_of(p, rq);
    if (cols == 0 || cols > p.small) return;
    const int32_t begin = (int32_t)(split * p.chunk), end = min(rq.seen, begin + (int32_t)p.chunk);
    if (split && begin >= rq.seen) return;
    const bool whole = rq.seen <= (int32_t)p.chunk;  // no other chunk

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, u = lane >> 4;
    const int32_t bs = (int32_t)p.cache.block_size;
    const int32_t *table = p.a.d_table + (uint64_t)r * p.a.table_stride;
    const bool live = (uint32_t)col < cols;
    const uint32_t qi = (uint32_t)col / p.group, qh = h * p.group + (uint32_t)col % p.group;
    const int32_t limit = live ? min(end, limit_of(rq, (int32_t)qi)) : end;  // unused columns mask nothing

    f16x8 q[KS];
    float zs;
    {
        const uint16_t *row = live ? reinterpret_cast<const uint16_t *>(p.a.d_q) +
                                         ((uint64_t)rq.q0 + qi) * p.a.q_token_stride + qh * p.a.q_head_stride
                                   : nullptr;
        const bool wide = !((uintptr_t)p.a.d_q & 15u) && !((p.a.q_token_stride | p.a.q_head_stride) & 7u);
        zs = load_query<DT, KS>(
            row, wide, p.a.scale < 0.0f ? -1.0f : 1.0f, q, [&](int f) { return u * (D / 4) + f * 8; },
            [](float v) { v = fmaxf(v, __shfl_xor(v, 16)); return fmaxf(v, __shfl_xor(v, 32)); });
        zs *= fabsf(p.a.scale) * kLog2e;
    }

    f32x4 o[VT];
#pragma unroll
    for (int t = 0; t < VT; t++) o[t] = f32x4{0, 0, 0, 0};
    Tops tops;
    float l = 0.0f;

    // K rows: this lane's rows are in run col >> 2; V and the scales: run u
    const int32_t kr = 16 * (col >> 2), vr = 16 * u, mask = bs - 1;
    const uint8_t *kh = p.cache.d_k + (uint64_t)h * bs * D + (col & 3) * D + u * (D / 4);
    const uint8_t *vh = p.cache.d_v + (uint64_t)h * bs * D + col * bs;
    int32_t bk = block_of(p, table, begin + 64 * wave + kr, end), bv = block_of(p, table, begin + 64 * wave + vr, end);
    for (int32_t base = begin + 64 * wave; base < end; base += 256) {
        const uint32_t ik = held(p, bk) ? bk : 0, iv = held(p, bv) ? bv : 0;
        const bool hv = held(p, bv);
        uint32_t kw[4][KW];
        u32x4 vw[VT];
        const uint8_t *kp = kh + (uint64_t)ik * p.block_step + (uint32_t)(((base + kr) & mask) * D);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if constexpr (KW % 4 == 0) {
#pragma unroll
                for (int w = 0; w < KW; w += 4) {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(kp + t * 4 * D + w * 4);
#pragma unroll
                    for (int e = 0; e < 4; e++) kw[t][w + e] = x[e];
                }
            } else {
#pragma unroll
                for (int w = 0; w < KW; w += 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2 *>(kp + t * 4 * D + w * 4);
                    kw[t][w] = x[0], kw[t][w + 1] = x[1];
                }
            }
        }
        const uint32_t bh = iv * p.cache.kv_heads + h;
        const float ks = p.cache.d_k_scale[bh], log_vs = log2f(hv ? p.cache.d_v_scale[bh] : 0.0f);
        const uint8_t *vp = vh + (uint64_t)iv * p.block_step + (uint32_t)((base + vr) & mask);
#pragma unroll
        for (int t = 0; t < VT; t++) vw[t] = *reinterpret_cast<const u32x4 *>(vp + t * 16 * bs);
        // the next tokens' blocks, before anything waits for these
        bk = block_of(p, table, base + 256 + kr, end), bv = block_of(p, table, base + 256 + vr, end);

        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < KS; f++)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8_to_f16(kw[t][2 * f], kw[t][2 * f + 1]), q[f], s[t], 0, 0, 0);
        }
        float c = ks * zs;
        const int32_t seen = hv ? limit - (base + vr) : 0;  // of this lane's 16 tokens
        if (!__all(seen >= 16)) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i >> 2][i & 3] = i < seen ? s[i >> 2][i & 3] * c : -__builtin_inff();
            c = 1.0f;
        }
        float zm = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; i++) zm = fmaxf(zm, s[i >> 2][i & 3]);
        zm *= c;
        float wm = zm + log_vs;  // -inf where nothing is seen
        zm = max_across_32(max_across_16(zm)), wm = max_across_32(max_across_16(wm));
        if (__any(tops.passed(zm, wm))) {
            float of_l, of_o;
            tops.take(zm, wm, of_l, of_o);
            l *= of_l;
#pragma unroll
            for (int t = 0; t < VT; t++) o[t] *= of_o;
        }
        const float share = share_of(log_vs, tops.rise), less = share - base_of(tops.m);
        f16x8 pv[2], rest[2];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float e = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], c, less));
            sum += e;
            pv[i >> 3][i & 7] = (_Float16)e;
            rest[i >> 3][i & 7] = (_Float16)(e - (float)pv[i >> 3][i & 7]);
        }
        l = fmaf(sum, __builtin_amdgcn_exp2f(-share), l);
#pragma unroll
        for (int t = 0; t < VT; t++) {
            const f16x8 a = codes8_to_f16(vw[t][0], vw[t][1]), b = codes8_to_f16(vw[t][2], vw[t][3]);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, rest[0], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, rest[1], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pv[0], o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pv[1], o[t], 0, 0, 0);
        }
    }

    // join the 4 waves: the common maxima, then the sums in a fixed order
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (u == 0) lds_ml[wave][col][0] = tops.m, lds_ml[wave][col][1] = l, lds_ml[wave][col][2] = tops.rise;
    __syncthreads();
    float mm = -__builtin_inff(), ll = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) mm = fmaxf(mm, lds_ml[w][col][0]);
#pragma unroll
    for (int w = 0; w < 4; w++) ll += lds_ml[w][col][1] * __builtin_amdgcn_exp2f(lds_ml[w][col][0] - base_of(mm));
    float rise = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < 4; w++) rise = fmaxf(rise, unit_of(lds_ml[w][col][0], lds_ml[w][col][2], mm));
    const float f = __builtin_amdgcn_exp2f(unit_of(tops.m, tops.rise, mm) - base_of(rise));
    if (rise == -__builtin_inff()) rise = __builtin_inff();
#pragma unroll
    for (int t = 0; t < VT; t++) o[t] *= f;
    if (wave >= 2) {
#pragma unroll
        for (int t = 0; t < VT; t++) *reinterpret_cast<f32x4 *>(&lds_o[wave - 2][col][16 * t + 4 * u]) = o[t];
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int t = 0; t < VT; t++) o[t] += *reinterpret_cast<const f32x4 *>(&lds_o[wave][col][16 * t + 4 * u]);
    }
    __syncthreads();
    if (wave == 1) {
#pragma unroll
        for (int t = 0; t < VT; t++) *reinterpret_cast<f32x4 *>(&lds_o[0][col][16 * t + 4 * u]) = o[t];
    }
    __syncthreads();
    if (wave != 0 || !live) return;
#pragma unroll
    for (int t = 0; t < VT; t++) o[t] += *reinterpret_cast<const f32x4 *>(&lds_o[0][col][16 * t + 4 * u]);
    if (whole) {
        uint16_t *out = reinterpret_cast<uint16_t *>(p.a.d_out) + ((uint64_t)rq.q0 + qi) * p.a.out_token_stride +
                        qh * p.a.out_head_stride;
        const bool wide = !((uintptr_t)p.a.d_out & 7u) && !((p.a.out_token_stride | p.a.out_head_stride) & 3u);
        const float inv = ll != 0.0f ? 1.0f / ll : 0.0f, root = half_rise(rise);
#pragma unroll
        for (int t = 0; t < VT; t++) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = o[t][i] * inv * root * root;
            store4<DT>(out + 16 * t + 4 * u, wide, v);
        }
        return;
    }
    const uint64_t at = (((uint64_t)r * p.cache.kv_heads + h) * p.splits + split) * p.cols + col;
#pragma unroll
    for (int t = 0; t < VT; t++) *reinterpret_cast<f32x4 *>(p.part_o + at * D + 16 * t + 4 * u) = o[t];
    if (u == 0) p.part_ml[3 * at] = mm, p.part_ml[3 * at + 1] = ll, p.part_ml[3 * at + 2] = rise;
}

// Joins the chunks of a request's column: one workgroup per request, head and
// column, its threads over 4 dimensions and every W-th chunk.
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs p) {
    constexpr int W = 256 / (D / 4);
    __shared__ __align__(16) float sum[W][D];
    const uint32_t r = blockIdx.x, h = blockIdx.y / p.cols, col = blockIdx.y % p.cols;
    const Request rq = request_of(p, r);
    const uint32_t cols = columns_of(p, rq);
    if (col >= cols || cols > p.small || rq.seen <= (int32_t)p.chunk) return;
    const uint32_t n = ((uint32_t)rq.seen + p.chunk - 1) / p.chunk;
    const uint64_t at = ((uint64_t)r * p.cache.kv_heads + h) * p.splits * p.cols + col;
    // l in units of 2^own, the largest of O's units in the same
    float own = -__builtin_inff(), rise = -__builtin_inff(), l = 0.0f;
    for (uint32_t s = threadIdx.x & 63u; s < n; s += 64) {
        const float *ml = p.part_ml + 3 * (at + (uint64_t)s * p.cols);
        const float now = fmaxf(own, ml[0]), down = own - base_of(now);
        l = fmaf(ml[1], __builtin_amdgcn_exp2f(ml[0] - base_of(now)), l * __builtin_amdgcn_exp2f(down));
        rise = fmaxf(rise + down, unit_of(ml[0], ml[2], now));
        own = now;
    }
    const float m = wave_max(own);
    l *= __builtin_amdgcn_exp2f(own - base_of(m));
    rise = wave_max(rise + (own - base_of(m)));
#pragma unroll
    for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
    const uint32_t part = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    if (part < W) {
        f32x4 o = {0, 0, 0, 0};
#pragma unroll 8
        for (uint32_t s = part; s < n; s += W) {
            const uint64_t i = at + (uint64_t)s * p.cols;
            o += __builtin_amdgcn_exp2f(unit_of(p.part_ml[3 * i], p.part_ml[3 * i + 2], m) - base_of(rise)) *
                 *reinterpret_cast<const f32x4 *>(p.part_o + i * D + d);
        }
        *reinterpret_cast<f32x4 *>(&sum[part][d]) = o;
    }
    __syncthreads();
    if (threadIdx.x >= D) return;
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) o += sum[w][threadIdx.x];
    uint16_t *out = reinterpret_cast<uint16_t *>(p.a.d_out) + ((uint64_t)rq.q0 + col / p.group) * p.a.out_token_stride +
                    (h * p.group + col % p.group) * p.a.out_head_stride;
    const float root = half_rise(rise > -__builtin_inff() ? rise : __builtin_inff());
    out[threadIdx.x] = (uint16_t)f32_to_half<DT>(l != 0.0f ? o / l * root * root : 0.0f);
}

// ---------------------------------------------------------------- many columns
//
// Bound by the two products' reads of LDS (each wave reads a tile's 32 KiB)
// and the softmax's vector instructions, about half of the time each beside
// a third for the matrix pipes: two prompts of 1900 to 2048 rows over 3000 to
// 4100 cached tokens, 32 heads on 8, 440 to 455 us (740 TFLOP/s).  4 waves of 32
// columns instead of 8 take 780 us there (each tile's codes are converted for
// half the columns).
//
// Where all of a tile's V scales lie within 2^20 of the column's rise, m and M
// move together by w alone: m is then within 28 of the largest z, which costs
// l nothing.
//
// Rows of a prompt: NW waves of 32 columns (32 x 32 x 16 tiles) share tiles of
// 64 tokens, which the workgroup turns into f16 once, in LDS.  Rows of LDS
// are padded by 16 bytes (an odd number of 16-byte units: rows read together
// lie in different banks).  A column's accumulators in S^T hold tokens
// 8 (i / 4) + 4 (lane / 32) + i % 4; V's tokens are stored in the order that
// makes a lane's 8 of them contiguous (4-7 and 8-11 of 16 change places).

template <int DT, int D, int NW>
__global__ __launch_bounds__(64 * NW) void attn_tile_kernel(const AttnArgs p) {
    constexpr int KS = D / 16, VT = D / 32, T = 64 * NW;
    constexpr int KP = D + 8, VP = 64 + 8;  // pitches in f16
    constexpr int CODES = 64 * D / 16, PER = (CODES + T - 1) / T;  // 16-byte pieces of a tile's codes
    __shared__ __align__(16) _Float16 lk[2][64 * KP];
    __shared__ __align__(16) _Float16 lv[2][D * VP];
    __shared__ __align__(16) float lks[2][4], lvs[2][4];  // K's scales, logarithms of V's
    const uint32_t r = blockIdx.x / p.tiles, tile = p.tiles - 1 - blockIdx.x % p.tiles, h = blockIdx.y;
    const Request rq = request_of(p, r);
    const uint32_t cols = columns_of(p, rq);
    if (cols <= p.small || tile * (32 * NW) >= cols) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hl = lane >> 5;
    const uint32_t c0 = tile * (32 * NW) + wave * 32 + (lane & 31);
    const bool live = c0 < cols;
    const uint32_t qi = c0 / p.group, qh = h * p.group + c0 % p.group;
    const int32_t limit = live ? limit_of(rq, (int32_t)qi) : 0;
    const uint32_t last = min(cols, (tile + 1) * (32 * NW)) - 1;
    const int32_t end = limit_of(rq, (int32_t)(last / p.group));
    const int32_t all = limit_of(rq, (int32_t)(tile * (32 * NW) / p.group));  // tokens that every column sees
    const int32_t bs = (int32_t)p.cache.block_size, mask = bs - 1;
    const int32_t *table = p.a.d_table + (uint64_t)r * p.a.table_stride;

    f16x8 q[KS];
    float zs;
    {
        const uint16_t *row = live ? reinterpret_cast<const uint16_t *>(p.a.d_q) +
                                         ((uint64_t)rq.q0 + qi) * p.a.q_token_stride + qh * p.a.q_head_stride
                                   : nullptr;
        const bool wide = !((uintptr_t)p.a.d_q & 15u) && !((p.a.q_token_stride | p.a.q_head_stride) & 7u);
        zs = load_query<DT, KS>(
            row, wide, p.a.scale < 0.0f ? -1.0f : 1.0f, q, [&](int f) { return f * 16 + hl * 8; },
            [](float v) { return fmaxf(v, __shfl_xor(v, 32)); });
        zs *= fabsf(p.a.scale) * kLog2e;
    }
    f32x16 o[VT];
#pragma unroll
    for (int t = 0; t < VT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[t][i] = 0.0f;
    Tops tops;
    float l = 0.0f;

    // A tile's codes on the way: pieces of 16 dimensions of a token, of 16
    // tokens of a dimension.  The blocks' ids come a tile ahead of the codes,
    // the codes a tile ahead of their use.
    u32x4 kc[PER], vc[PER];
    int32_t ik[PER], iv[PER], is = -1;
    float ksc = 0.0f, vsc = 0.0f;
    const uint8_t *kh = p.cache.d_k + (uint64_t)h * bs * D, *vh = p.cache.d_v + (uint64_t)h * bs * D;
    auto ids = [&](int32_t base) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int x = j * T + tid;
            ik[j] = block_of(p, table, base + x / (D / 16), end), iv[j] = block_of(p, table, base + 16 * (x % 4), end);
        }
        if (tid < 4) is = block_of(p, table, base + 16 * tid, end);
    };
    auto fetch = [&](int32_t base) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int x = j * T + tid;
            if (CODES % T && x >= CODES) break;
            const int kt = x / (D / 16), kd = x % (D / 16), vd = x / 4, vu = x % 4;
            kc[j] = *reinterpret_cast<const u32x4 *>(kh + (uint64_t)(held(p, ik[j]) ? ik[j] : 0) * p.block_step +
                                                     (uint32_t)(((base + kt) & mask) * D + kd * 16));
            vc[j] = *reinterpret_cast<const u32x4 *>(vh + (uint64_t)(held(p, iv[j]) ? iv[j] : 0) * p.block_step +
                                                     (uint32_t)(vd * bs + ((base + 16 * vu) & mask)));
        }
        if (tid < 4) {
            const bool in = held(p, is);
            const uint32_t bh = (in ? is : 0) * p.cache.kv_heads + h;
            // a run without a block: marked by a negative scale
            ksc = in ? p.cache.d_k_scale[bh] : -1.0f;
            vsc = log2f(in ? p.cache.d_v_scale[bh] : 0.0f);
        }
    };
    auto stage = [&](int b) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int x = j * T + tid;
            if (CODES % T && x >= CODES) break;
            const int kt = x / (D / 16), kd = x % (D / 16), vd = x / 4, vu = x % 4;
            *reinterpret_cast<f16x8 *>(&lk[b][kt * KP + kd * 16]) = codes8_to_f16(kc[j][0], kc[j][1]);
            *reinterpret_cast<f16x8 *>(&lk[b][kt * KP + kd * 16 + 8]) = codes8_to_f16(kc[j][2], kc[j][3]);
            *reinterpret_cast<f16x8 *>(&lv[b][vd * VP + vu * 16]) = codes8_to_f16(vc[j][0], vc[j][2]);
            *reinterpret_cast<f16x8 *>(&lv[b][vd * VP + vu * 16 + 8]) = codes8_to_f16(vc[j][1], vc[j][3]);
        }
        if (tid < 4) lks[b][tid] = ksc, lvs[b][tid] = vsc;
    };

    if (end > 0) {
        ids(0);
        fetch(0);
        ids(64);
        stage(0);
        fetch(64);
        ids(128);
    }
    for (int32_t base = 0; base < end; base += 64) {
        const int b = (base >> 6) & 1;
        // the one barrier of a tile: its codes are in LDS, and the tile
        // before, whose buffer the next one takes, is done with
        __syncthreads();
        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
#pragma unroll
            for (int f = 0; f < KS; f++) {
                const f16x8 a = *reinterpret_cast<const f16x8 *>(&lk[b][(t * 32 + (lane & 31)) * KP + f * 16 + hl * 8]);
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[f], s[t], 0, 0, 0);
            }
        }
        float c[4], log_vs[4];
        bool masked = base + 64 > all;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float ks = lks[b][i];
            log_vs[i] = lvs[b][i];
            c[i] = ks * zs;
            masked = masked || ks < 0.0f;
        }
        if (base + 64 < end) {
            stage(b ^ 1);
            fetch(base + 128);
            ids(base + 192);
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int u = 2 * t + (i >> 3);
                    const int32_t tok = base + 32 * t + 8 * (i >> 2) + 4 * hl + (i & 3);
                    s[t][i] = tok < limit && lks[b][u] >= 0.0f ? s[t][i] * c[u] : -__builtin_inff();
                }
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = 1.0f;
        }
        float um[4], share[4], zm = -__builtin_inff(), wm = -__builtin_inff();
        bool close = true;  // not for NaN
#pragma unroll
        for (int u = 0; u < 4; u++) {
            um[u] = s[u >> 1][8 * (u & 1)];
#pragma unroll
            for (int i = 1; i < 8; i++) um[u] = fmaxf(um[u], s[u >> 1][8 * (u & 1) + i]);
            wm = fmaxf(wm, fmaf(um[u], c[u], log_vs[u]));
            share[u] = log_vs[u] - tops.rise;
            close = close && fabsf(share[u]) <= kNear;
        }
        wm = max_across_32(wm);
        const bool near = __all(close);
        if (!near) {
#pragma unroll
            for (int u = 0; u < 4; u++) zm = fmaxf(zm, um[u] * c[u]);
            zm = max_across_32(zm);
        }
        if (__any(tops.passed(zm, wm))) {
            float of_l, of_o;
            if (near)
                of_l = of_o = tops.move(wm);
            else
                tops.take(zm, wm, of_l, of_o);
            l *= of_l;
#pragma unroll
            for (int t = 0; t < VT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[t][i] *= of_o;
        }
        if (!near) {
#pragma unroll
            for (int u = 0; u < 4; u++) share[u] = share_of(log_vs[u], tops.rise);
        }
        const float ref = base_of(tops.m);
        f16x8 pv[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const float less = share[u] - ref;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + i], c[u], less));
                sum += e;
                pv[u][i] = (_Float16)e;
            }
            l = fmaf(sum, __builtin_amdgcn_exp2f(-share[u]), l);
        }
#pragma unroll
        for (int t = 0; t < VT; t++)
#pragma unroll
            for (int f = 0; f < 4; f++) {
                const f16x8 a = *reinterpret_cast<const f16x8 *>(&lv[b][(t * 32 + (lane & 31)) * VP + f * 16 + hl * 8]);
                o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pv[f], o[t], 0, 0, 0);
            }
    }
    l += __shfl_xor(l, 32);
    if (!live) return;
    uint16_t *out = reinterpret_cast<uint16_t *>(p.a.d_out) + ((uint64_t)rq.q0 + qi) * p.a.out_token_stride +
                    qh * p.a.out_head_stride;
    const bool wide = !((uintptr_t)p.a.d_out & 7u) && !((p.a.out_token_stride | p.a.out_head_stride) & 3u);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f, root = half_rise(tops.rise);
#pragma unroll
    for (int t = 0; t < VT; t++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = o[t][i + e] * inv * root * root;
            store4<DT>(out + 32 * t + 2 * i + 4 * hl, wide, v);
        }
}

// 8 waves (two to a SIMD, each tile's codes converted for 256 columns) where
// their registers fit.
template <int D>
constexpr int kTileWaves = D <= 128 ? 8 : 4;

template <int DT, int D>
hipError_t launch_attention(const AttnArgs &p, hipStream_t s) {
    if (!p.a.requests) {
        hipLaunchKernelGGL((attn_zero_kernel<D>), dim3(p.a.tokens < 4096 ? p.a.tokens : 4096), dim3(256), 0, s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((attn_step_kernel<DT, D>), dim3(p.a.requests * p.splits, p.cache.kv_heads), dim3(256), 0, s, p);
    if (p.splits > 1)
        hipLaunchKernelGGL((attn_join_kernel<DT, D>), dim3(p.a.requests, p.cache.kv_heads * p.cols), dim3(256), 0, s, p);
    if (p.tiles)
        hipLaunchKernelGGL((attn_tile_kernel<DT, D, kTileWaves<D>>), dim3(p.a.requests * p.tiles, p.cache.kv_heads),
                           dim3(64 * kTileWaves<D>), 0, s, p);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_dim(const AttnArgs &p, hipStream_t s) {
    switch (p.cache.head_dim) {
        case 64: return launch_attention<DT, 64>(p, s);
        case 96: return launch_attention<DT, 96>(p, s);
        case 128: return launch_attention<DT, 128>(p, s);
        case 192: return launch_attention<DT, 192>(p, s);
        default: return launch_attention<DT, 256>(p, s);
    }
}

// Whether two rows of `dim` elements, `tokens` of them `ts` apart for each of
// `heads` heads `hs` apart, share an element.
bool rows_meet(uint64_t tokens, uint64_t heads, uint64_t ts, uint64_t hs, uint64_t dim) {
    typedef unsigned __int128 u128;
    if (tokens > 1 && ts < dim) return true;
    if (heads > 1 && hs < dim) return true;
    if (tokens == 1 || heads == 1 || ts >= (u128)(heads - 1) * hs + dim || hs >= (u128)(tokens - 1) * ts + dim) return false;
    // neither stride spans the other: heads j apart against the tokens next to that
    for (uint64_t j = 1; j < heads; j++) {
        const u128 d = (u128)j * hs, below = d / ts, rest = d % ts;
        if (below < tokens && rest < dim) return true;
        if (below + 1 < tokens && ts - rest < dim) return true;
    }
    return false;
}

}  // namespace
}  // namespace hh

extern "C" int32_t hh_kv_attention(hh_context *ctx, const hh_kv_cache *cache, const hh_kv_attention_args *a,
                                   void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    const int32_t rc = hh::check_kv_cache(cache);
    if (rc != HH_OK) return rc;
    if (a->dtype != HH_F16 && a->dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (a->q_heads == 0 || a->q_heads % cache->kv_heads) return HH_ERR_INVALID_ARGUMENT;
    if (a->tokens == 0) return HH_OK;
    if (!a->d_q || !a->d_out || (a->requests && (!a->d_start || !a->d_kv_len || (!a->d_table && a->table_width))))
        return HH_ERR_INVALID_ARGUMENT;
    if ((((uintptr_t)a->d_q | (uintptr_t)a->d_out) & 1u) || a->table_stride < a->table_width) return HH_ERR_INVALID_ARGUMENT;
    if (hh::rows_meet(a->tokens, a->q_heads, a->out_token_stride, a->out_head_stride, cache->head_dim))
        return HH_ERR_INVALID_ARGUMENT;
    if (a->requests > 65536 || a->tokens >= 1u << 24) return HH_ERR_INVALID_ARGUMENT;
    const uint32_t group = a->q_heads / cache->kv_heads;
    const uint64_t most = (uint64_t)(a->max_q < a->tokens ? a->max_q : a->tokens) * group;
    if (most >= 1ull << 31) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hh::AttnArgs p = {};
    p.cache = *cache;
    p.a = *a;
    p.group = group;
    p.bs_log = (uint32_t)__builtin_ctz(cache->block_size);
    p.block_step = cache->kv_heads * cache->block_size * cache->head_dim;
    p.small = 16;
    p.cols = (uint32_t)(most < 1 ? 1 : most < 16 ? most : 16);
    const uint64_t room = (uint64_t)a->table_width * cache->block_size;
    const uint64_t kv = a->max_kv < room ? a->max_kv : room;
    if (kv > 1ull << 30) return HH_ERR_UNSUPPORTED;  // tokens are counted in 31 bits
    // chunks: enough workgroups for 8 per CU, none below 512 tokens (48
    // requests of up to 8001 tokens, 131,001 tokens of one: 93 and 52 us; 4 per
    // CU 106 and 50, 16 per CU 100 and 52, 24 per CU 93 and 52)
    const uint64_t lanes = (uint64_t)(a->requests ? a->requests : 1) * cache->kv_heads;
    const uint64_t want = (8ull * (uint64_t)(ctx->num_cus > 0 ? ctx->num_cus : 256) + lanes - 1) / lanes;
    uint64_t chunk = (kv + want - 1) / want;
    chunk = (chunk + 255) / 256 * 256;
    if (chunk < 512) chunk = 512;
    p.chunk = (uint32_t)chunk;
    p.splits = (uint32_t)((kv + chunk - 1) / chunk);
    if (p.splits < 1) p.splits = 1;
    // Workgroups go around the 8 XCDs: with an odd number of chunks to a
    // request each XCD gets early and late ones (of ragged requests the late
    // ones are empty; those 48 in 6 chunks each 106 us, in 7 93).
    if (p.splits > 1) p.splits |= 1;
    const uint32_t waves = cache->head_dim <= 128 ? hh::kTileWaves<128> : hh::kTileWaves<256>, tile = 32 * waves;
    p.tiles = most > p.small ? (uint32_t)((most + tile - 1) / tile) : 0;
    // a launch has fewer than 2^32 threads a dimension (chunks are a few
    // thousand, or a few to a request)
    if ((uint64_t)a->requests * p.tiles * 64 * waves >= 1ull << 32) return HH_ERR_UNSUPPORTED;
    if (cache->kv_heads * 16ull > 65535) return HH_ERR_UNSUPPORTED;
    if (a->requests && p.splits > 1) {
        const uint64_t n = lanes * p.splits * p.cols;
        const int32_t e = hh::op_room(ctx, reinterpret_cast<hipStream_t>(stream), n * (cache->head_dim + 3) * sizeof(float),
                                      &p.part_o);
        if (e != HH_OK) return e;
        p.part_ml = p.part_o + n * cache->head_dim;
    }
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    return hh::from_hip(a->dtype == HH_BF16 ? hh::launch_dim<HH_BF16>(p, s) : hh::launch_dim<HH_F16>(p, s));
}
