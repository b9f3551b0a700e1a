// paged_cache.h -- host checks of a paged key/value cache, shared by its writer
// and its reader.
#pragma once

#include <stdint.h>

#include "kda_abi.h"

namespace kda {

// Types and sizes that the kernels assume. An empty pool (num_pages = 0) is valid: nothing is
// addressed in it.
inline int check_cache_sizes(const KdaPagedCache &c) {
    if (c.head_dim != 64 && c.head_dim != 128) {
        return KDA_ERR_UNSUPPORTED;
    }
    if (c.dtype != KDA_BF16 && c.dtype != KDA_FP8_E4M3) {
        return KDA_ERR_UNSUPPORTED;
    }
    // kv_heads: a head's number times its row stays in range
    if (c.kv_heads <= 0 || c.kv_heads > 65535 || c.page_size <= 0 || c.num_pages < 0 ||
        c.num_pages > INT32_MAX / c.page_size) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    return KDA_OK;
}

// The same, and the pointers, strides and alignment.
inline int check_cache(const KdaPagedCache &c) {
    if (const int rc = check_cache_sizes(c); rc != KDA_OK) {
        return rc;
    }
    if (c.num_pages == 0) {
        return KDA_OK;
    }
    const int64_t unit = c.dtype == KDA_BF16 ? 8 : 16;  // elements of 16 bytes
    for (const int64_t s : {c.k_stride_page, c.k_stride_token, c.k_stride_head, c.v_stride_page, c.v_stride_token,
                            c.v_stride_head}) {
        if (s % unit != 0) {
            return KDA_ERR_INVALID_ARGUMENT;
        }
    }
    for (const void *p : {c.k, c.v}) {
        if (p == nullptr || reinterpret_cast<uintptr_t>(p) % 16 != 0) {
            return KDA_ERR_INVALID_ARGUMENT;
        }
    }
    for (const float *p : {c.k_scale, c.v_scale}) {
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0 || (p != nullptr && c.dtype != KDA_FP8_E4M3)) {
            return KDA_ERR_INVALID_ARGUMENT;
        }
    }
    return KDA_OK;
}

}  // namespace kda
