// y = act(x W^T + bias) * mul + residual (hh_linear, include/haagenti_hip.h).
//
// The kernels are in linear_kernels.hpp; here is which of them a shape takes.
#define HH_GATED 0
#include "linear_kernels.hpp"

namespace hh {
namespace {

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

// Room for the splits' sums.
int32_t split_room(hh_context *ctx, const LinearArgs &p, const TilePlan &plan, hipStream_t s, Split *split) {
    *split = {plan.steps, nullptr, 0};
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
