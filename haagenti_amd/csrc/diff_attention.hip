// o = softmax(scale q1 K1^T) V - lambda softmax(scale q2 K2^T) V over the paged
// 8-bit cache, with a norm over each head's dimensions (hh_kv_diff_attention,
// include/haagenti_hip.h).
#define HH_DIFF 1
#include "attention_kernels.hpp"

extern "C" int32_t hh_kv_diff_attention(hh_context *ctx, const hh_kv_cache *cache, const hh_kv_attention_args *a,
                                        const hh_kv_diff_args *diff, void *stream) {
    if (!ctx || !a || !diff) return HH_ERR_INVALID_ARGUMENT;
    if (a->tokens && !diff->d_lambda) return HH_ERR_INVALID_ARGUMENT;
    if (((uintptr_t)diff->d_lambda | (uintptr_t)diff->d_norm_weight) & 3u) return HH_ERR_INVALID_ARGUMENT;
    if (!(diff->eps >= 0.0f)) return HH_ERR_INVALID_ARGUMENT;
    hh::AttnArgs p = {};
    p.diff = *diff;
    return hh::run_attention(ctx, cache, a, p, stream);
}
