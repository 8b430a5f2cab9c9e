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
// is the launch and the scan's chain of two loads and two block scans.

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
            if (w.served) slot = (int32_t)((uint32_t)(b < w.have ? table[b] : fresh(b - w.have)) * bs + pos % bs);
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

// ---------------------------------------------------------------- append
//
// One wave per row, head and side (keys, values): the wave of a run's first
// row (its predecessor's slot is not the one before in the same block) takes
// the whole run, the others end.  It reads the run twice (largest magnitude,
// then codes; the second time from cache).  Values are transposed on the way:
// a lane takes 8 dimensions of 16 tokens and writes each dimension's 16 codes
// at once.

struct AppendArgs {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    const uint16_t *rows_k, *rows_v;
    uint64_t tk, hk, tv, hv;
    const int32_t *slots;
    uint32_t tokens, heads, dim, bs, slots_end;
};

// amax / 127, rounded up to 8 significant bits: a / 127 of an 11-bit a is no
// nearer than 2^-18 (relative) to such a number without being one, so the
// f32 quotient decides as the exact one does.
__device__ __forceinline__ float scale_for(float amax) {
    return __uint_as_float((__float_as_uint(amax / 127.0f) + 0xffffu) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t code_of(float x, float scale) {
    const float q = x != x ? 0.0f : fminf(fmaxf(rintf(x / scale), -127.0f), 127.0f);
    return (uint32_t)(int32_t)q + 128u & 255u;
}

// 8 values of a row.  WIDE: 16-byte aligned.
template <bool WIDE>
__device__ __forceinline__ u32x4 load8(const uint16_t *p) {
    if constexpr (WIDE) return *reinterpret_cast<const u32x4 *>(p);
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    return v;
}
template <int DT>
__device__ __forceinline__ float elem(const u32x4 &v, int i) {
    return half_to_f32<DT>((v[i >> 1] >> (16 * (i & 1))) & 0xffffu);
}

template <int DT, bool WIDE>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs p) {
    const uint32_t lane = threadIdx.x & 63u, task = blockIdx.y * 4 + (threadIdx.x >> 6);
    const uint32_t h = task >> 1, t = blockIdx.x, bs = p.bs;
    if (h >= p.heads) return;
    const int32_t slot = p.slots[t];
    if (slot < 0 || (uint32_t)slot >= p.slots_end) return;
    const uint32_t off = (uint32_t)slot % bs;
    if (off && t && p.slots[t - 1] == slot - 1) return;
    // the run: consecutive slots of this block (at most 128 rows)
    uint32_t n = 1;
    for (uint32_t i = 1; off + i < bs; i += 64) {
        const uint32_t j = i + lane;
        const bool in = off + j < bs && (uint64_t)t + j < p.tokens && p.slots[t + j] == slot + (int32_t)j;
        const uint64_t out = ~__ballot(in);
        if (out) {
            n += (uint32_t)__builtin_ctzll(out);
            break;
        }
        n += 64;
    }
    const bool values = task & 1u;
    const uint64_t bh = (uint64_t)((uint32_t)slot / bs) * p.heads + h;
    const uint64_t ts = values ? p.tv : p.tk;
    const uint16_t *rows = values ? p.rows_v + t * p.tv + h * p.hv : p.rows_k + t * p.tk + h * p.hk;
    uint8_t *codes = (values ? p.v : p.k) + bh * bs * p.dim;
    float *scale = (values ? p.v_scale : p.k_scale) + bh;
    const float old = off ? *scale : 0.0f;

    const uint32_t chunks = p.dim / 8;
    float amax = 0.0f;
    for (uint32_t i = lane; i < n * chunks; i += 64) {
        const u32x4 x = load8<WIDE>(rows + i / chunks * ts + i % chunks * 8);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float a = fabsf(elem<DT>(x, e));
            amax = fmaxf(amax, a < __builtin_inff() ? a : 0.0f);
        }
    }
    amax = wave_max(amax);
    const float now = fmaxf(old, scale_for(amax)), div = now > 0.0f ? now : 1.0f;
    if (off && now > old) {
        // the block's tokens before: off * dim codes, keys in one piece,
        // values in rows of bs
        for (uint32_t i = lane; i < off * p.dim; i += 64) {
            uint8_t *c = codes + (values ? (uint64_t)(i / off) * bs + i % off : i);
            *c = (uint8_t)code_of((float)((int32_t)*c - 128) * old, div);
        }
    }
    if (lane == 0) *scale = now;
    if (!values) {
        for (uint32_t i = lane; i < n * chunks; i += 64) {
            const uint32_t r = i / chunks, c = i % chunks * 8;
            const u32x4 x = load8<WIDE>(rows + r * ts + c);
            u32x2 w = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; e++) w[e >> 2] |= code_of(elem<DT>(x, e), div) << (8 * (e & 3));
            *reinterpret_cast<u32x2 *>(codes + (uint64_t)(off + r) * p.dim + c) = w;
        }
        return;
    }
    const uint32_t g0 = off / 16, groups = (off + n - 1) / 16 - g0 + 1;
    for (uint32_t i = lane; i < groups * chunks; i += 64) {
        const uint32_t g = g0 + i / chunks, c = i % chunks * 8;
        uint8_t *to = codes + (uint64_t)c * bs + 16 * g;
        u32x4 w[8] = {};
        bool whole = true;
#pragma unroll
        for (uint32_t j = 0; j < 16; j++) {
            const uint32_t r = 16 * g + j - off;  // wraps below the run
            if (r < n) {
                const u32x4 x = load8<WIDE>(rows + r * ts + c);
#pragma unroll
                for (int e = 0; e < 8; e++) w[e][j >> 2] |= code_of(elem<DT>(x, e), div) << (8 * (j & 3));
            } else {
                whole = false;
            }
        }
        if (whole) {
#pragma unroll
            for (int e = 0; e < 8; e++) *reinterpret_cast<u32x4 *>(to + (uint64_t)e * bs) = w[e];
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) {
                if (16 * g + j - off >= n) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) to[(uint64_t)e * bs + j] = (uint8_t)(w[e][j >> 2] >> (8 * (j & 3)));
            }
        }
    }
}

// ---------------------------------------------------------------- read
//
// One workgroup per block, head and side.  Values go through LDS, their rows
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
    extern __shared__ uint32_t tile[];
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
            for (int j = 0; j < 4; j++) tile[(d * pitch + 16 * g) / 4 + j] = w[j];
        }
        __syncthreads();
    }
    for (uint32_t i = threadIdx.x; i < bs * chunks; i += 256) {
        const uint32_t t = i / chunks, c = i % chunks * 8;
        float v[8];
        if (values) {
            const uint8_t *b = reinterpret_cast<const uint8_t *>(tile);
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
    // a step reads the state in every workgroup and writes the next one
    if (a->d_state < a->d_state_out + 2 && a->d_state_out < a->d_state + 2) return HH_ERR_INVALID_ARGUMENT;
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    const uint32_t columns = a->requests < 1 ? 1 : a->requests < hh::kPlanColumns ? a->requests : hh::kPlanColumns;
    // prompts of thousands of rows: up to 8 workgroups to a request
    const uint32_t per = a->tokens / columns / (4 * hh::kPlanThreads);
    const uint32_t rows = per < 1 ? 1 : per > 8 ? 8 : per;
    hipLaunchKernelGGL(hh::kv_plan_kernel, dim3(columns, rows), dim3(hh::kPlanThreads), 0,
                       reinterpret_cast<hipStream_t>(stream), *a);
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
    const hh::AppendArgs p = {cache->d_k, cache->d_v, cache->d_k_scale, cache->d_v_scale,
                              reinterpret_cast<const uint16_t *>(d_rows_k), reinterpret_cast<const uint16_t *>(d_rows_v),
                              tk, hk, tv, hv, d_slots, tokens, cache->kv_heads, cache->head_dim, cache->block_size,
                              cache->num_blocks * cache->block_size};
    const bool wide = !(((uintptr_t)d_rows_k | (uintptr_t)d_rows_v) & 15u) && !((tk | hk | tv | hv) & 7u);
    auto kernel = dtype == HH_BF16 ? (wide ? hh::kv_append_kernel<HH_BF16, true> : hh::kv_append_kernel<HH_BF16, false>)
                                   : (wide ? hh::kv_append_kernel<HH_F16, true> : hh::kv_append_kernel<HH_F16, false>);
    hipLaunchKernelGGL(kernel, dim3(tokens, (2 * cache->kv_heads + 3) / 4), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), p);
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
