// o = softmax(scale q K^T) V over the paged 8-bit cache (hh_kv_attention,
// include/haagenti_hip.h).
#define HH_DIFF 0
#include "attention_kernels.hpp"

extern "C" int32_t hh_kv_attention(hh_context *ctx, const hh_kv_cache *cache, const hh_kv_attention_args *a,
                                   void *stream) {
    if (!ctx || !a) return HH_ERR_INVALID_ARGUMENT;
    return hh::run_attention(ctx, cache, a, hh::AttnArgs{}, stream);
}
