// y = act(x G^T + gate bias) * (x U^T + up bias) in one launch
// (hh_gated_linear, include/haagenti_hip.h): the kernels of
// linear_kernels.hpp with both weights' rows in turns of 16.  Its gradients
// are in gated_backward.hip.
//
// Beside two products (up, then gate with the product as epilogue) x is read
// once, up's output not written and read between, and one launch less.  bf16,
// 14336 x 4096: a token 40 us (235 MB of weights at 5.9 TB/s); 16 tokens of
// INT4 33 us (66 MB at 2 TB/s: loads of 64 bytes a row, and their scales), both
// the kernel's by a profiler; a call of 2048 tokens 429 us, with what is kept 454
// (1060 TFLOP/s; the library's bare product in the same run 334), bound by LDS
// beside the matrix pipes.  INT4 of 2048 tokens, in tiles through registers 1082
// us; of rows of 4097 values, whose groups cross rows, 1 to 16 tokens 166 to 170.
#define HH_GATED 1
#include "linear_kernels.hpp"

namespace hh {
namespace {

// Both weights' 16 rows to a workgroup; 8 waves while there are at most two
// workgroups to a CU, else 4, as in linear.hip, where both are measured.
template <int DT, int YT, int MT, bool INT4>
hipError_t launch_gated_rows(const GatedArgs &p, int cus, hipStream_t s) {
    const uint32_t tiles = (p.a.n + 15) / 16;
    if (tiles <= 2 * (uint32_t)cus)
        hipLaunchKernelGGL((gated_rows_kernel<DT, YT, MT, 2, 8, INT4>), dim3(tiles), dim3(512), 0, s, p);
    else
        hipLaunchKernelGGL((gated_rows_kernel<DT, YT, MT, 2, 4, INT4>), dim3(tiles), dim3(256), 0, s, p);
    return hipGetLastError();
}

// The tiles' plan, of a product with both weights' rows (n outputs to 2 n
// rows, in whole turns).
template <int N>
TilePlan plan_gated(const hh_linear_args &a, int cus, const Shape (&shapes)[N]) {
    hh_linear_args both = a;
    both.n = (a.n + 15) / 16 * 32;
    return plan_tiles(both, cus, shapes);
}
// Where a last round of tiles leaves CUs idle, whole rounds and then a launch
// of smaller tiles for the other columns, if that is expected to be faster: the
// first launch's columns (all of them: n) and the second's shape.  The estimate
// is the plain product's; what is kept, 8 bytes an output beside y's, isn't in
// it.  Calls: 2048 x 14336 x 4096 in 896 tiles of 256 x 256 on 256 CUs 446 us
// (470 with what is kept), in 768 and 256 of 256 x 128 428 (454); 3000 x 5504 x
// 2048 169 (170), so 143 (144).
uint32_t whole_rounds(const hh_linear_args &a, int cus, const TilePlan &plan, int *rest_shape) {
    if (plan.splits > 1) return a.n;
    const Shape &s = kLargeShapes[plan.shape];
    const uint64_t mt = (a.m + s.m - 1) / s.m, slots = (uint64_t)cus * s.per_cu;
    const uint64_t nt = ((uint64_t)a.n * 2 + s.n - 1) / s.n, first = nt * mt / slots * slots / mt;  // tiles of columns
    if (!first || first >= nt) return a.n;
    auto time = [&](const Shape &t, uint64_t cols) {
        const uint64_t tiles = (2 * cols + t.n - 1) / t.n * ((a.m + t.m - 1) / t.m), all = (uint64_t)cus * t.per_cu;
        return (double)((tiles + all - 1) / all) * ((tiles <= (uint64_t)cus ? t.alone : t.us) * plan.steps + 4.0);
    };
    const uint32_t cols = (uint32_t)(first * s.n / 2);
    double least = time(s, a.n) - time(s, cols) - 4.0;  // (a launch)
    uint32_t whole = a.n;
    for (int i = 0; i < (int)(sizeof(kLargeShapes) / sizeof(Shape)); i++) {
        const double rest = time(kLargeShapes[i], a.n - cols);
        if (rest < least) least = rest, whole = cols, *rest_shape = i;
    }
    return whole;
}
int32_t gated_room(hh_context *ctx, const GatedArgs &p, const TilePlan &plan, hipStream_t s, Split *split) {
    *split = {plan.steps, nullptr, 0};
    if (plan.splits == 1) return HH_OK;
    return op_room(ctx, s, (size_t)plan.splits * p.a.m * partial_row(p.a.n) * sizeof(float), &split->partial);
}
template <int DT, int YT>
int32_t join_gated(const GatedArgs &p, const TilePlan &plan, const Split &split, hipStream_t s) {
    if (split.partial)
        hipLaunchKernelGGL((gated_join_kernel<DT, YT>),
                           dim3((uint32_t)(((uint64_t)p.a.m * ((p.a.n + 3) / 4) + 255) / 256)), dim3(256), 0, s, p,
                           (const float *)split.partial, plan.splits);
    return from_hip(hipGetLastError());
}

template <int DT, int YT, int MODE>
int32_t launch_gated_any(hh_context *ctx, const GatedArgs &p, int cus, hipStream_t s) {
    const TilePlan plan = plan_gated(p.a, cus, kAnyShapes);
    Split split;
    const int32_t rc = gated_room(ctx, p, plan, s, &split);
    if (rc != HH_OK) return rc;
    const uint32_t S = kAnyShapes[plan.shape].n;
    const dim3 grid((p.a.n + S / 2 - 1) / (S / 2), (p.a.m + S - 1) / S, plan.splits);
    if (S == 128)
        hipLaunchKernelGGL((gated_tile_kernel<DT, YT, MODE, 128>), grid, dim3(256), 0, s, p, split);
    else
        hipLaunchKernelGGL((gated_tile_kernel<DT, YT, MODE, 64>), grid, dim3(256), 0, s, p, split);
    return join_gated<DT, YT>(p, plan, split, s);
}
template <int DT, int YT, int TN, int TM, int WN, int WM>
void launch_gated_tiles(const GatedArgs &p, const Split &split, uint32_t cols, uint32_t splits, hipStream_t s) {
    const uint32_t tiles = ((cols + TN / 2 - 1) / (TN / 2)) * ((p.a.m + TM - 1) / TM);
    hipLaunchKernelGGL((gated_large_kernel<DT, YT, TN, TM, WN, WM>), dim3(tiles, splits), dim3(64 * WN * WM), 0, s, p,
                       split);
}

template <int DT, int YT>
int32_t launch_gated(hh_context *ctx, const GatedArgs &p, hipStream_t s) {
    const hh_linear_args &a = p.a;
    const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
    const bool int4 = a.w_dtype == HH_INT4;
    if (int4 && a.k % 32) return launch_gated_any<DT, YT, kInt4Any>(ctx, p, cus, s);
    const bool aligned = !int4 && !(((uintptr_t)a.d_x | (uintptr_t)a.d_w | (uintptr_t)p.up) & 15u) &&
                         !((a.x_stride | a.w_stride | p.up_stride) & 7u) && a.k % 64 == 0 && a.k && a.x_stride < 1u << 22 &&
                         a.w_stride < 1u << 22 && p.up_stride < 1u << 22;  // offsets in a tile: 32 bits
    if (a.m <= (aligned ? 32u : 64u)) {  // as hh_linear
        const int rows = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
        return from_hip(int4 ? (rows == 1   ? launch_gated_rows<DT, YT, 1, true>(p, cus, s)
                                : rows == 2 ? launch_gated_rows<DT, YT, 2, true>(p, cus, s)
                                            : launch_gated_rows<DT, YT, 4, true>(p, cus, s))
                             : (rows == 1   ? launch_gated_rows<DT, YT, 1, false>(p, cus, s)
                                : rows == 2 ? launch_gated_rows<DT, YT, 2, false>(p, cus, s)
                                            : launch_gated_rows<DT, YT, 4, false>(p, cus, s)));
    }
    if (int4) return launch_gated_any<DT, YT, kInt4>(ctx, p, cus, s);
    if (!aligned) return launch_gated_any<DT, YT, kHalf>(ctx, p, cus, s);
    const TilePlan plan = plan_gated(a, cus, kLargeShapes);
    Split split;
    const int32_t rc = gated_room(ctx, p, plan, s, &split);
    if (rc != HH_OK) return rc;
    int rest_shape = 0;
    const uint32_t whole = whole_rounds(a, cus, plan, &rest_shape);
    auto launch = [&](int shape, uint32_t cols) {
        switch (shape) {
            case 0: launch_gated_tiles<DT, YT, 256, 256, 2, 4>(p, split, cols, plan.splits, s); break;
            case 1: launch_gated_tiles<DT, YT, 256, 128, 4, 2>(p, split, cols, plan.splits, s); break;
            case 2: launch_gated_tiles<DT, YT, 128, 256, 2, 4>(p, split, cols, plan.splits, s); break;
            case 3: launch_gated_tiles<DT, YT, 128, 128, 2, 2>(p, split, cols, plan.splits, s); break;
            default: launch_gated_tiles<DT, YT, 128, 64, 2, 2>(p, split, cols, plan.splits, s); break;
        }
    };
    launch(plan.shape, whole);
    if (whole < a.n) {
        const int32_t e = from_hip(hipGetLastError());
        if (e != HH_OK) return e;
        split.first = whole;
        launch(rest_shape, a.n - whole);
    }
    return join_gated<DT, YT>(p, plan, split, s);
}

}  // namespace

int32_t check_gated(const hh_gated_args *a) {
    if (a->dtype != HH_F16 && a->dtype != HH_BF16) return HH_ERR_UNSUPPORTED;
    if (a->w_dtype != a->dtype && a->w_dtype != HH_INT4) return HH_ERR_UNSUPPORTED;
    if (a->activation < HH_ACT_NONE || a->activation > HH_ACT_SILU) return HH_ERR_UNSUPPORTED;
    if (a->m >= 1u << 21 || a->n >= 1u << 25 || a->k >= 1u << 31) return HH_ERR_INVALID_ARGUMENT;
    if (a->m && a->n && a->k && (!a->d_x || !a->d_gate || !a->d_up)) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)a->d_x | (uintptr_t)a->d_gate | (uintptr_t)a->d_up | (uintptr_t)a->d_gate_bias | (uintptr_t)a->d_up_bias) & 1u)
        return HH_ERR_INVALID_ARGUMENT;
    if ((uintptr_t)a->d_saved & 15u) return HH_ERR_INVALID_ARGUMENT;
    if (a->x_stride < a->k) return HH_ERR_INVALID_ARGUMENT;
    if (a->w_dtype != HH_INT4 && (a->gate_stride < a->k || a->up_stride < a->k)) return HH_ERR_INVALID_ARGUMENT;
    return HH_OK;
}

}  // namespace hh

extern "C" int32_t hh_gated_linear(hh_context *ctx, const hh_gated_args *a, void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    const int32_t rc = hh::check_gated(a);
    if (rc != HH_OK) return rc;
    if (a->y_dtype != a->dtype && a->y_dtype != HH_F32) return HH_ERR_UNSUPPORTED;
    if (a->m == 0 || a->n == 0) return HH_OK;
    if (!a->d_y || ((uintptr_t)a->d_y & (a->y_dtype == HH_F32 ? 3u : 1u)) || a->y_stride < a->n) return HH_ERR_INVALID_ARGUMENT;
    hh::GatedArgs p = {};
    p.a.d_x = a->d_x, p.a.d_w = a->d_gate, p.a.d_bias = a->d_gate_bias, p.a.d_y = a->d_y;
    p.a.x_stride = a->x_stride, p.a.w_stride = a->gate_stride, p.a.y_stride = a->y_stride;
    p.a.m = a->m, p.a.n = a->n, p.a.k = a->k;
    p.a.dtype = a->dtype, p.a.w_dtype = a->w_dtype, p.a.y_dtype = a->y_dtype, p.a.activation = a->activation;
    p.up = a->d_up, p.up_bias = a->d_up_bias, p.up_stride = a->up_stride, p.saved = a->d_saved;
    if (a->w_dtype == HH_INT4) {
        const uint64_t count = (uint64_t)a->n * a->k, scales = (count + 31) / 32 * 2, bytes = scales + (count + 1) / 2;
        if (a->gate_bytes < bytes || a->up_bytes < bytes) return HH_ERR_UNEXPECTED_EOF;
        p.scales = reinterpret_cast<const uint16_t *>(a->d_gate);
        p.nibbles = reinterpret_cast<const uint8_t *>(a->d_gate) + scales;
        p.up_scales = reinterpret_cast<const uint16_t *>(a->d_up);
        p.up_nibbles = reinterpret_cast<const uint8_t *>(a->d_up) + scales;
    }
    p.vec = !(((uintptr_t)a->d_gate_bias | (uintptr_t)a->d_up_bias) & 7u) &&
            !((uintptr_t)a->d_y & (a->y_dtype == HH_F32 ? 15u : 7u)) && !(a->y_stride & 3u) && !(a->d_saved && (a->n & 3u));
    hh::DeviceGuard guard(ctx->device);
    if (guard.status() != hipSuccess) return hh::from_hip(guard.status());
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (a->dtype == HH_BF16)
        return a->y_dtype == HH_F32 ? hh::launch_gated<HH_BF16, HH_F32>(ctx, p, s)
                                    : hh::launch_gated<HH_BF16, HH_BF16>(ctx, p, s);
    return a->y_dtype == HH_F32 ? hh::launch_gated<HH_F16, HH_F32>(ctx, p, s) : hh::launch_gated<HH_F16, HH_F16>(ctx, p, s);
}
