// The paged key-value cache as the kernels see it, and its 8-bit codes.
#pragma once

#include <cstdio>

#include "vectors.cuh"

namespace chm {

// Checks a cache's layout (host); what is wrong goes to chm_last_error.
inline chm_status check_cache(const chm_kv_cache* c, const char* who) {
    auto bad = [&](const char* why) {
        char msg[160];
        snprintf(msg, sizeof(msg), "%s: %s", who, why);
        set_last_message(msg);
        return CHM_ERR_INVALID;
    };
    if (!c) return bad("null cache");
    if (c->type != CHM_FP16 && c->type != CHM_BF16 && c->type != CHM_INT8 && c->type != CHM_E4M3)
        return bad("a cache is fp16, bf16, int8 or e4m3");
    if (c->num_pages < 0 || c->page_size < 1 || c->heads < 1 || c->heads > (1 << 16))
        return bad("page_size and heads must be positive");
    if (c->num_pages > (INT64_MAX >> 8) / c->page_size / c->heads) return bad("too many pages");
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) return bad("dim must be a multiple of 16, at most 256");
    const int run = 16 / type_bytes(c->type);
    if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0) return bad("cache strides must not be negative");
    if (c->page_stride % run || c->head_stride % run || c->token_stride % run)
        return bad("cache strides must be multiples of 16 bytes");
    if (!aligned16(c->k) || !aligned16(c->v)) return bad("cache memory must be 16-byte aligned");
    const bool scaled = c->type == CHM_INT8 || c->type == CHM_E4M3;
    if (c->num_pages > 0 && (!c->k || !c->v)) return bad("null pages");
    if (c->num_pages > 0 && scaled && (!c->k_scale || !c->v_scale)) return bad("an 8-bit cache needs its scales");
    return CHM_OK;
}

}  // namespace chm
