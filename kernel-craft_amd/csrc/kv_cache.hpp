// kv_cache.hpp -- the quantized paged key/value cache: argument checks shared
// by the kernels that write it (qk_norm_rope.hip) and read it (kv_cache_read.hip).
#pragma once

#include "fp8_common.hpp"
#include "mxfp4.hpp"

namespace kc {
namespace kv {

constexpr int kMaxHeadDim = 1024;
constexpr int64_t kMaxGrid = (1 << 24) - 1;  // workgroups of 256: a launch holds fewer than 2^32 threads

inline int check_cache(const char* fn, const kc_kv_cache* c) {
    if (!c) return set_error(KC_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
    if (c->format != KC_KV_FP8 && c->format != KC_KV_MXFP4)
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: unknown cache format %d", fn, c->format);
    if (c->num_pages < 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->head_dim <= 0)
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: bad cache shape pages=%lld page_size=%d heads=%d head_dim=%d", fn,
                         (long long)c->num_pages, c->page_size, c->kv_heads, c->head_dim);
    if (c->head_dim > kMaxHeadDim)
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: head_dim=%d is over %d", fn, c->head_dim, kMaxHeadDim);
    if (c->format == KC_KV_MXFP4 && c->head_dim % mx::kBlock != 0)
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: head_dim=%d must be a multiple of 32 for MXFP4", fn, c->head_dim);
    if (c->num_pages > INT32_MAX || c->kv_heads > (1 << 16))
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: cache too large", fn);
    if (c->num_pages > 0 && (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales))
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: null cache pointer", fn);
    return KC_SUCCESS;
}

}  // namespace kv
}  // namespace kc
