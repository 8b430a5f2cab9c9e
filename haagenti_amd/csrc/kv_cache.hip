// The paged 8-bit key / value cache: a step's plan, appending rows, reading
// blocks back.  Layout and rules are in include/haagenti_hip.h.
#include "layer_ops.hpp"

namespace hh {
namespace {

constexpr uint32_t kMaxRequests = 65536;

// ---------------------------------------------------------------- plan
//
// Every workgroup scans all requests' lengths (8 bytes each, from L2) for the
// running sums of rows, blocks taken and blocks freed, and keeps what it
// needs of its own requests: request r belongs to the workgroups of column
// r % gridDim.x, whose gridDim.y rows share its table entries and slots.
// Nothing passes between workgroups, so one launch does it.  What bounds it
// is the launch and the scan's chain of two loads and two block scans: 8
// requests 5.5 us, 1024 with 64,000 new rows 11.7.

constexpr uint32_t kPlanThreads = 256, kPlanItems = 4, kPlanChunk = kPlanThreads * kPlanItems, kPlanColumns = 1024;

struct PlanOwn {
    uint32_t start, rows, len, have, take, first, give, back;
    int32_t served;
};

// Exclusive sums over the workgroup of each thread's a and b; totals in ta, tb.
__device__ __forceinline__ void block_scan2(uint64_t &a, uint64_t &b, uint64_t &ta, uint64_t &tb, uint64_t (*part)[2]) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t a0 = a, b0 = b;
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) {
        const uint64_t ua = __shfl_up(a, d), ub = __shfl_up(b, d);
        if (lane >= d) a += ua, b += ub;
    }
    __syncthreads();  // the last call's readers are done with part
    if (lane == 63) part[wave][0] = a, part[wave][1] = b;
    __syncthreads();
    a -= a0, b -= b0, ta = tb = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanThreads / 64; w++) {
        if (w < wave) a += part[w][0], b += part[w][1];
        ta += part[w][0], tb += part[w][1];
    }
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(const hh_kv_plan_args p) {
    __shared__ PlanOwn own[kMaxRequests / kPlanColumns];
    __shared__ uint64_t part[kPlanThreads / 64][2];
    __shared__ uint32_t taken;
    const uint32_t tid = threadIdx.x, bs = p.block_size, cap = p.ring_capacity;
    const uint32_t column = blockIdx.x, columns = gridDim.x;
    if (tid == 0) taken = 0;
    const uint32_t count = (uint32_t)min((int64_t)cap, max((int64_t)0, (int64_t)p.d_state[1]));
    const uint32_t head = cap ? (uint32_t)p.d_state[0] % cap : 0;
    uint64_t rows_at = 0, take_at = 0, give_at = 0;  // sums over the chunks before
    for (uint32_t c = 0; c < p.requests; c += kPlanChunk) {
        int32_t len[kPlanItems], add[kPlanItems];
        uint64_t sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPlanItems; j++) {
            const uint32_t r = c + tid * kPlanItems + j;
            len[j] = r < p.requests ? p.d_len[r] : 0;
            add[j] = r < p.requests ? p.d_new[r] : 0;
            sum += (uint64_t)max(add[j], 0);
        }
        uint64_t at = sum, zero = 0, total, none;
        block_scan2(at, zero, total, none, part);
        uint64_t want[kPlanItems], give[kPlanItems], start[kPlanItems], sw = 0, sg = 0;
        int32_t status[kPlanItems];
        at += rows_at;
#pragma unroll
        for (uint32_t j = 0; j < kPlanItems; j++) {
            const uint64_t l = (uint64_t)max(len[j], 0), a = (uint64_t)max(add[j], 0);
            const uint64_t have = (l + bs - 1) / bs, need = (l + a + bs - 1) / bs;
            start[j] = at;
            at += a;
            status[j] = len[j] < 0 ? HH_ERR_INVALID_ARGUMENT
                        : add[j] >= 0 && (need > p.table_width || l + a > 0x7fffffffu || (a && at > p.tokens))
                            ? HH_ERR_BUFFER_TOO_SMALL
                            : HH_OK;
            const bool sound = status[j] == HH_OK;
            want[j] = sound && add[j] > 0 ? need - have : 0;
            give[j] = sound && add[j] < 0 ? min(have, (uint64_t)p.table_width) : 0;
            sw += want[j], sg += give[j];
        }
        uint64_t wat = sw, gat = sg, tw, tg;
        block_scan2(wat, gat, tw, tg, part);
        wat += take_at, gat += give_at;
        uint32_t most = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPlanItems; j++) {
            const uint32_t r = c + tid * kPlanItems + j;
            // in order: a request that finds too few blocks stops all after
            // it that need any, so what a served one takes starts at the sum
            // of all wants before it
            const uint64_t first = wat;
            wat += want[j];
            if (status[j] == HH_OK && want[j] && wat > count) status[j] = HH_ERR_OUT_OF_MEMORY;
            const bool served = status[j] == HH_OK && add[j] >= 0;
            if (served && want[j]) most = (uint32_t)wat;
            if (r < p.requests && r % columns == column) {
                const uint32_t a = (uint32_t)max(add[j], 0), l = (uint32_t)max(len[j], 0);
                own[r / columns] = {(uint32_t)min(start[j], (uint64_t)p.tokens), a, l, (uint32_t)(((uint64_t)l + bs - 1) / bs),
                                    served ? (uint32_t)want[j] : 0u, (uint32_t)first, (uint32_t)give[j], (uint32_t)gat, served};
                if (blockIdx.y == 0) {
                    p.d_start[r] = (int32_t)min(start[j], (uint64_t)p.tokens);
                    p.d_kv_len[r] = served ? (int32_t)(l + a) : 0;
                    p.d_status[r] = status[j];
                }
            }
            gat += give[j];
        }
        if (most) atomicMax(&taken, most);
        rows_at += total, take_at += tw, give_at += tg;
    }
    __syncthreads();
    const uint32_t rows = (uint32_t)min(rows_at, (uint64_t)p.tokens);
    if (column == 0 && blockIdx.y == 0 && tid == 0) {
        const uint64_t after = (uint64_t)count - taken + give_at;
        p.d_start[p.requests] = (int32_t)rows;
        p.d_state_out[0] = cap ? (int32_t)((head + (uint64_t)taken) % cap) : 0;
        p.d_state_out[1] = (int32_t)min(after, (uint64_t)cap);
    }
    const uint32_t at0 = blockIdx.y * kPlanThreads + tid, step = gridDim.y * kPlanThreads;
    for (uint32_t r = column, o = 0; r < p.requests; r += columns, o++) {
        const PlanOwn w = own[o];
        int32_t *table = p.d_table + (uint64_t)r * p.table_stride;
        auto fresh = [&](uint32_t e) {
            const uint64_t i = (uint64_t)head + w.first + e;  // first + e < count <= cap
            return p.d_ring[i < cap ? i : i - cap];
        };
        for (uint32_t e = at0; e < w.take; e += step) table[w.have + e] = fresh(e);
        for (uint32_t i = at0; i < w.rows && w.start + i < p.tokens; i += step) {
            const uint32_t pos = w.len + i, b = pos / bs;
            int32_t slot = -1;
            if (w.served) {
                // an id whose slots pass 31 bits is no block of any cache
                const uint32_t id = (uint32_t)(b < w.have ? table[b] : fresh(b - w.have));
                if (id < 0x80000000u / bs) slot = (int32_t)(id * bs + pos % bs);
            }
            p.d_slots[w.start + i] = slot;
        }
        // entries past the free ones: nobody else reads or writes them
        for (uint32_t e = at0; e < w.give; e += step) {
            const uint64_t n = (uint64_t)count + w.back + e;
            if (n < cap) p.d_ring[head + n < cap ? head + n : head + n - cap] = table[e];
        }
    }
    for (uint64_t i = (uint64_t)rows + (uint64_t)column * step + at0; i < p.tokens; i += (uint64_t)columns * step)
        p.d_slots[i] = -1;
}

// The plan's inputs where its results go over them: to[0..1] the state, then
// the lengths, then the new rows.
__global__ __launch_bounds__(kPlanThreads) void plan_inputs_kernel(const int32_t *state, const int32_t *len, const int32_t *add,
                                                                   uint32_t requests, int32_t *to) {
    const uint32_t i = blockIdx.x * kPlanThreads + threadIdx.x;
    if (i < 2) to[i] = state[i];
    if (i < requests) to[2 + i] = len[i], to[2 + requests + i] = add[i];
}

// ---------------------------------------------------------------- append
//
// A run is the rows of one block: consecutive slots.  A workgroup takes the
// runs that begin in its span of rows, for one head and side (keys, values):
// it holds a run's rows in registers (PER pieces of 8 values per thread),
// finds their largest magnitude and writes their codes, the keys' at once,
// the values' through LDS, where they become 16 tokens per dimension.  Bound
// by reading the rows and, for single rows, by the chain slot, row, maximum,
// scale, code: 8388 rows of 8 heads of 128 dimensions 21 us (2.4 TB/s), 67
// rows that are runs of their own 6.7.  Reading the rows twice instead of
// holding them took 109.

struct AppendArgs {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    const uint16_t *rows_k, *rows_v;
    uint64_t tk, hk, tv, hv;
    const int32_t *slots;
    uint32_t tokens, heads, dim, bs, slots_end, span;
};

// amax / 127, rounded up to 8 significant bits: a / 127 of an 11-bit a is no
// nearer than 2^-18 (relative) to such a number without being one, so the
// f32 quotient decides as the exact one does.
__device__ __forceinline__ float scale_for(float amax) {
    return __uint_as_float((__float_as_uint(amax / 127.0f) + 0xffffu) & 0xffff0000u);
}
// x / scale rounded to a code.  The quotient of an x of at most 16 bits by a
// scale of 8 is a tie or 2^-18 (relative) away from one; with one correction
// the product by the reciprocal is within 2^-22 and exact where the quotient
// is a tie (its correction is the error of the first product, to 2^-23).
// Scales whose reciprocal leaves f32's normal range are divided by.
struct Divider {
    float scale, inverse;
    __device__ __forceinline__ explicit Divider(float s) : scale(s), inverse(1.0f / s) {}
    __device__ __forceinline__ float quotient(float x) const {
        if (scale < 0x1p-120f) return x / scale;
        const float q = x * inverse;
        return fmaf(fmaf(-q, scale, x), inverse, q);
    }
    // values: infinities give the last codes, NaN that of 0
    __device__ __forceinline__ uint32_t code(float x) const {
        const float q = fabsf(x) < __builtin_inff() ? quotient(x) : x;
        return (uint32_t)(int32_t)(q != q ? 0.0f : fminf(fmaxf(rintf(q), -127.0f), 127.0f)) + 128u;
    }
    // The low byte of the result, for a value of at most 127 scales (a whole
    // run without infinities and NaN) and a scale that is not tiny: the sum
    // is rounded at its units.
    __device__ __forceinline__ uint32_t code_in_byte(float x) const {
        const float q = x * inverse;
        return __float_as_uint(fmaf(fmaf(-q, scale, x), inverse, q) + 12583040.0f);  // 1.5 * 2^23 + 128
    }
};
// The low bytes of four numbers.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}
// A word of codes at another scale.
__device__ __forceinline__ uint32_t recode(uint32_t w, float old, const Divider &now) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) v |= now.code((float)((int32_t)((w >> (8 * i)) & 255u) - 128) * old) << (8 * i);
    return v;
}

// 8 values of a row.  WIDE: 16-byte aligned.
template <bool WIDE>
__device__ __forceinline__ u32x4 load8(const uint16_t *p) {
    if constexpr (WIDE) return *reinterpret_cast<const u32x4 *>(p);
    typedef u32x4 u32x4_any __attribute__((aligned(2)));
    return *reinterpret_cast<const u32x4_any *>(p);
}
template <int DT>
__device__ __forceinline__ float elem(const u32x4 &v, int i) {
    return half_to_f32<DT>((v[i >> 1] >> (16 * (i & 1))) & 0xffffu);
}

template <int DT, bool WIDE, int PER>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs p) {
    extern __shared__ __align__(16) uint8_t tile[];
    __shared__ float tops[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, h = blockIdx.y >> 1, bs = p.bs, t0 = blockIdx.x * p.span;
    const bool values = blockIdx.y & 1u;
    // 64 slots from the span's first row on: where runs begin, where they go on
    const int32_t mine = t0 + lane < p.tokens ? p.slots[t0 + lane] : -1;
    const int32_t ahead = t0 ? p.slots[t0 - 1] : -1;
    const int32_t below = __shfl_up(mine, 1), prev = lane ? below : ahead;  // every lane takes part in the shuffle
    const bool sound = mine >= 0 && (uint32_t)mine < p.slots_end, on = sound && (uint32_t)mine % bs && prev == mine - 1;
    const uint64_t goes_on = __ballot(on);
    uint64_t first = __ballot(sound && !on && lane < p.span);
    const uint32_t chunks = p.dim / 8, pitch = bs + 20;
    // i / chunks of i < 4096: exact, as the error i / 2^16 stays below 1 / chunks
    const uint32_t inv = 65536u / chunks + (65536u % chunks != 0);
    for (; first; first &= first - 1) {
        const uint32_t l0 = (uint32_t)__builtin_ctzll(first), t = t0 + l0;
        const int32_t slot = __builtin_amdgcn_readlane(mine, (int)l0);
        const uint32_t off = (uint32_t)slot % bs;
        const uint64_t rest = ~(goes_on >> l0 >> 1);
        uint32_t n = 1 + (uint32_t)__builtin_ctzll(rest);  // a bit is set: zeros came in from above
        if (l0 + n == 64) {
            // as far as was read: 64 more slots at a time
            for (uint32_t i = n; off + i < bs; i += 64) {
                const uint32_t j = i + lane;
                const bool in = off + j < bs && (uint64_t)t + j < p.tokens && p.slots[t + j] == slot + (int32_t)j;
                const uint64_t out = ~__ballot(in);
                n += out ? (uint32_t)__builtin_ctzll(out) : 64u;
                if (out) break;
            }
        }
        const uint64_t bh = (uint64_t)((uint32_t)slot / bs) * p.heads + h, ts = values ? p.tv : p.tk;
        const uint16_t *rows = values ? p.rows_v + t * p.tv + h * p.hv : p.rows_k + t * p.tk + h * p.hk;
        uint8_t *codes = (values ? p.v : p.k) + bh * bs * p.dim;
        float *scale = (values ? p.v_scale : p.k_scale) + bh;
        const float old = off ? *scale : 0.0f;

        u32x4 x[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const uint32_t i = j * 256 + tid;
            x[j] = i < n * chunks ? load8<WIDE>(rows + (i * inv >> 16) * ts + (i - (i * inv >> 16) * chunks) * 8) : u32x4{0, 0, 0, 0};
        }
        // magnitudes order as their bits do, infinities and NaN above all
        u16x2 most = {0, 0};
#pragma unroll
        for (int j = 0; j < PER; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[j][e] & 0x7fff7fffu));
        float amax = half_to_f32<DT>(max(most[0], most[1]));
        const bool fine = __syncthreads_and(amax < __builtin_inff());
        if (!fine) {
            amax = 0.0f;
#pragma unroll
            for (int j = 0; j < PER; j++)
#pragma unroll 1
                for (int e = 0; e < 8; e++) {
                    const float v = fabsf(elem<DT>(x[j], e));
                    amax = fmaxf(amax, v < __builtin_inff() ? v : 0.0f);
                }
        }
        amax = wave_max(amax);
        if (lane == 0) tops[tid >> 6] = amax;
        __syncthreads();
        amax = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float now = fmaxf(old, scale_for(amax));
        const Divider div(now > 0.0f ? now : 1.0f);
        const bool grown = off && now > old, plain = fine && div.scale >= 0x1p-120f;
        const uint32_t lead = off % 16;  // tile's columns are tokens from the run's first 16 on
        if (tid == 0) *scale = now;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const uint32_t i = j * 256 + tid, r = i * inv >> 16, c = (i - r * chunks) * 8;
            if (i >= n * chunks) break;
            u32x2 w;
            if (plain) {
                uint32_t b[8];
#pragma unroll
                for (int e = 0; e < 8; e++) b[e] = div.code_in_byte(elem<DT>(x[j], e));
                w = u32x2{low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
            } else {
                w = u32x2{0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; e++) w[e >> 2] |= div.code(elem<DT>(x[j], e)) << (8 * (e & 3));
            }
            if (values) {
#pragma unroll
                for (int e = 0; e < 8; e++) tile[(c + e) * pitch + lead + r] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
            } else {
                *reinterpret_cast<u32x2 *>(codes + (uint64_t)(off + r) * p.dim + c) = w;
            }
        }
        if (values) {
            // 16 tokens of a dimension at a time, with what is there of
            // tokens before (at the new scale) and after the run
            __syncthreads();
            const uint32_t g0 = grown ? 0 : off / 16, groups = (off + n + 15) / 16 - g0;
            for (uint32_t i = tid; i < groups * p.dim; i += 256) {
                const uint32_t d = i / groups, at = (g0 + i % groups) * 16;
                u32x4 *to = reinterpret_cast<u32x4 *>(codes + (uint64_t)d * bs + at);
                u32x4 w;
                if (at >= off && at + 16 <= off + n) {
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = reinterpret_cast<const uint32_t *>(tile + d * pitch + (at - off + lead))[e];
                } else {
                    w = *to;
                    for (uint32_t j = 0; j < 16; j++) {
                        const uint32_t r = at + j - off;  // wraps below the run
                        uint32_t c = (w[j >> 2] >> (8 * (j & 3))) & 255u;
                        if (r < n)
                            c = tile[d * pitch + lead + r];
                        else if (grown && at + j < off)
                            c = div.code((float)((int32_t)c - 128) * old);
                        w[j >> 2] = (w[j >> 2] & ~(255u << (8 * (j & 3)))) | c << (8 * (j & 3));
                    }
                }
                *to = w;
            }
        } else if (grown) {
            for (uint32_t i = tid; i < off * p.dim / 16; i += 256) {
                u32x4 *at = reinterpret_cast<u32x4 *>(codes) + i;
                u32x4 w = *at;
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = recode(w[e], old, div);
                *at = w;
            }
        }
        __syncthreads();  // tops and tile are read
    }
}

template <int DT, bool WIDE>
void launch_append(const AppendArgs &p, hipStream_t s) {
    // pieces of 8 values in a full block, over 256 threads
    const uint32_t per = (p.bs * p.dim / 8 + 255) / 256;
    auto kernel = per <= 1   ? kv_append_kernel<DT, WIDE, 1>
                  : per <= 2 ? kv_append_kernel<DT, WIDE, 2>
                  : per <= 4 ? kv_append_kernel<DT, WIDE, 4>
                  : per <= 8 ? kv_append_kernel<DT, WIDE, 8>
                             : kv_append_kernel<DT, WIDE, 16>;
    hipLaunchKernelGGL(kernel, dim3((p.tokens + p.span - 1) / p.span, 2 * p.heads), dim3(256), p.dim * (p.bs + 20), s, p);
}

// ---------------------------------------------------------------- read
//
// One workgroup per block, head and side; bound by memory: 140 blocks of 64
// tokens, 8 heads of 128 dimensions to bf16 11 us (5 TB/s).  Values go through LDS, their rows
// of tokens padded by 4 bytes against bank conflicts, to come out token by
// token.

template <int OUT>
__device__ __forceinline__ void store8(void *out, uint64_t at, const float *v) {
    if constexpr (OUT == HH_F32) {
        f32x4 *o = reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(out) + at);
        o[0] = f32x4{v[0], v[1], v[2], v[3]};
        o[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = f32_to_half<OUT>(v[2 * i]) | f32_to_half<OUT>(v[2 * i + 1]) << 16;
        *reinterpret_cast<u32x4 *>(reinterpret_cast<uint16_t *>(out) + at) = w;
    }
}

template <int OUT>
__global__ __launch_bounds__(256) void kv_read_kernel(const hh_kv_cache cache, const int32_t *__restrict__ blocks,
                                                      void *__restrict__ out_k, void *__restrict__ out_v) {
    extern __shared__ uint32_t words[];
    const uint32_t bs = cache.block_size, dim = cache.head_dim, heads = cache.kv_heads, h = blockIdx.y;
    const bool values = blockIdx.z, held = (uint32_t)blocks[blockIdx.x] < cache.num_blocks;
    const uint64_t bh = (uint64_t)(held ? blocks[blockIdx.x] : 0) * heads + h;
    const uint8_t *codes = (values ? cache.d_v : cache.d_k) + bh * bs * dim;
    const float scale = held ? (values ? cache.d_v_scale : cache.d_k_scale)[bh] : 0.0f;
    void *out = values ? out_v : out_k;
    const uint64_t base = (uint64_t)blockIdx.x * bs * heads * dim + (uint64_t)h * dim;
    const uint32_t chunks = dim / 8, pitch = bs + 4;
    if (values) {
        for (uint32_t i = threadIdx.x; i < dim * bs / 16; i += 256) {
            const uint32_t d = i / (bs / 16), g = i % (bs / 16);
            const u32x4 w = held ? *reinterpret_cast<const u32x4 *>(codes + (uint64_t)i * 16) : u32x4{};
#pragma unroll
            for (int j = 0; j < 4; j++) words[(d * pitch + 16 * g) / 4 + j] = w[j];
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < bs * chunks; i += 256) {
        const uint32_t t = i / chunks, c = i % chunks * 8;
        float v[8];
        if (values) {
            const uint8_t *b = reinterpret_cast<const uint8_t *>(words);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float)((int32_t)b[(c + e) * pitch + t] - 128) * scale;
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(codes + (uint64_t)i * 8);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float)((int32_t)((w[e >> 2] >> (8 * (e & 3))) & 255u) - 128) * scale;
        }
        if (!held) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = 0.0f;
        }
        store8<OUT>(out, base + (uint64_t)t * heads * dim + c, v);
    }
}

}  // namespace

int32_t check_kv_cache(const hh_kv_cache *c) {
    if (!c || !c->d_k || !c->d_v || !c->d_k_scale || !c->d_v_scale) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)c->d_k | (uintptr_t)c->d_v) & 15u) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)c->d_k_scale | (uintptr_t)c->d_v_scale) & 3u) return HH_ERR_INVALID_ARGUMENT;
    if (c->block_size != 16 && c->block_size != 32 && c->block_size != 64 && c->block_size != 128)
        return HH_ERR_UNSUPPORTED;
    const uint32_t d = c->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 192 && d != 256) return HH_ERR_UNSUPPORTED;
    if (c->num_blocks == 0 || c->kv_heads == 0 || c->kv_heads > 32767) return HH_ERR_INVALID_ARGUMENT;
    if ((uint64_t)c->num_blocks * c->block_size >= 1ull << 31) return HH_ERR_INVALID_ARGUMENT;
    return HH_OK;
}

}  // namespace hh

extern "C" {

int32_t hh_kv_plan(hh_context *ctx, const hh_kv_plan_args *a, void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    if (a->requests > hh::kMaxRequests) return HH_ERR_UNSUPPORTED;
    if (a->block_size != 16 && a->block_size != 32 && a->block_size != 64 && a->block_size != 128)
        return HH_ERR_UNSUPPORTED;
    if (!a->d_state || !a->d_start || !a->d_state_out || (a->ring_capacity && !a->d_ring) || (a->tokens && !a->d_slots))
        return HH_ERR_INVALID_ARGUMENT;
    if (a->requests && (!a->d_len || !a->d_new || !a->d_kv_len || !a->d_status || (a->table_width && !a->d_table)))
        return HH_ERR_INVALID_ARGUMENT;
    if (a->table_stride < a->table_width || a->tokens >= 1u << 31 || a->ring_capacity >= 1u << 31)
        return HH_ERR_INVALID_ARGUMENT;
    if (a->d_state < a->d_state_out + 2 && a->d_state_out < a->d_state + 2) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    // every workgroup reads the state and all lengths while others write
    // their results: inputs that these go over are set aside first
    const uint64_t n = a->requests;
    const struct {
        const int32_t *at;
        uint64_t n;
    } in[] = {{a->d_len, n}, {a->d_new, n}, {a->d_state, 2}},
      out[] = {{a->d_start, n + 1}, {a->d_kv_len, n}, {a->d_slots, a->tokens}, {a->d_status, n}, {a->d_state_out, 2}};
    bool over = false;
    for (const auto &i : in)
        for (const auto &o : out) over = over || (i.n && o.n && i.at < o.at + o.n && o.at < i.at + i.n);
    hh_kv_plan_args p = *a;
    if (over) {
        float *room = nullptr;
        const int32_t rc = hh::op_room(ctx, s, (2 * n + 2) * sizeof(int32_t), &room);
        if (rc != HH_OK) return rc;
        int32_t *to = reinterpret_cast<int32_t *>(room);
        hipLaunchKernelGGL(hh::plan_inputs_kernel, dim3((uint32_t)(n / hh::kPlanThreads) + 1), dim3(hh::kPlanThreads), 0, s,
                           a->d_state, a->d_len, a->d_new, a->requests, to);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return hh::from_hip(e);
        p.d_state = to, p.d_len = to + 2, p.d_new = to + 2 + n;
    }
    const uint32_t columns = a->requests < 1 ? 1 : a->requests < hh::kPlanColumns ? a->requests : hh::kPlanColumns;
    // prompts of thousands of rows: up to 8 workgroups to a request
    const uint32_t per = a->tokens / columns / (4 * hh::kPlanThreads);
    const uint32_t rows = per < 1 ? 1 : per > 8 ? 8 : per;
    hipLaunchKernelGGL(hh::kv_plan_kernel, dim3(columns, rows), dim3(hh::kPlanThreads), 0, s, p);
    return hh::from_hip(hipGetLastError());
}

int32_t hh_kv_append(hh_context *ctx, const hh_kv_cache *cache, const void *d_rows_k, const void *d_rows_v,
                     int32_t dtype, uint64_t tk, uint64_t hk, uint64_t tv, uint64_t hv, const int32_t *d_slots,
                     uint32_t tokens, void *stream) {
    if (!ctx) return HH_ERR_INVALID_ARGUMENT;
    const int32_t rc = hh::check_kv_cache(cache);
    if (rc != HH_OK) return rc;
    if (dtype != HH_F16 && dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (tokens == 0) return HH_OK;
    if (!d_rows_k || !d_rows_v || !d_slots || tokens >= 1u << 24) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)d_rows_k | (uintptr_t)d_rows_v) & 1u) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    // Rows in a workgroup's span: one while the grid is small (each row of a
    // step is a run), up to 16 for prompts, most of whose rows begin none.
    // Runs of one span follow one another, so rows that are runs of their own
    // want few: 8 heads of 128 dimensions, 4096 single rows take 208 us at 8,
    // 218 at 16, 244 at 64, 2048 of them after 4192 rows of prompts 105, 116
    // and 171, 8384 rows of prompts 24, 20 and 22.
    const uint64_t grid = (uint64_t)tokens * 2 * cache->kv_heads / 2048;
    const hh::AppendArgs p = {cache->d_k, cache->d_v, cache->d_k_scale, cache->d_v_scale,
                              reinterpret_cast<const uint16_t *>(d_rows_k), reinterpret_cast<const uint16_t *>(d_rows_v),
                              tk, hk, tv, hv, d_slots, tokens, cache->kv_heads, cache->head_dim, cache->block_size,
                              cache->num_blocks * cache->block_size, (uint32_t)(grid < 1 ? 1 : grid > 16 ? 16 : grid)};
    const bool wide = !(((uintptr_t)d_rows_k | (uintptr_t)d_rows_v) & 15u) && !((tk | hk | tv | hv) & 7u);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == HH_BF16)
        wide ? hh::launch_append<HH_BF16, true>(p, s) : hh::launch_append<HH_BF16, false>(p, s);
    else
        wide ? hh::launch_append<HH_F16, true>(p, s) : hh::launch_append<HH_F16, false>(p, s);
    return hh::from_hip(hipGetLastError());
}

int32_t hh_kv_read(hh_context *ctx, const hh_kv_cache *cache, const int32_t *d_blocks, uint32_t nblocks,
                   int32_t out_dtype, void *d_out_k, void *d_out_v, void *stream) {
    if (!ctx) return HH_ERR_INVALID_ARGUMENT;
    const int32_t rc = hh::check_kv_cache(cache);
    if (rc != HH_OK) return rc;
    if (out_dtype != HH_F32 && out_dtype != HH_F16 && out_dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (nblocks == 0) return HH_OK;
    if (!d_blocks || !d_out_k || !d_out_v || nblocks >= 1u << 24) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)d_out_k | (uintptr_t)d_out_v) & 15u) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    auto kernel = out_dtype == HH_F32   ? hh::kv_read_kernel<HH_F32>
                  : out_dtype == HH_F16 ? hh::kv_read_kernel<HH_F16>
                                        : hh::kv_read_kernel<HH_BF16>;
    hipLaunchKernelGGL(kernel, dim3(nblocks, cache->kv_heads, 2), dim3(256), cache->head_dim * (cache->block_size + 4),
                       reinterpret_cast<hipStream_t>(stream), *cache, d_blocks, d_out_k, d_out_v);
    return hh::from_hip(hipGetLastError());
}

}  // extern "C"
