// linear_device.h -- what the two forms of linear attention share: metadata as the kernels read it, host checks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kda_abi.h"
#include "kda_device.h"

namespace kda {

struct LinearParams : KdaLinearArgs {
    // An entry of the metadata, whole: two words of an int64 one, the same word twice of an int32 one. Without a branch,
    // so that the loads of several arrays are in flight together.
    __device__ __forceinline__ int64_t entry(const void *p, int n, int bit) const {
        const int both = (wide & bit) != 0 ? 1 : 0;
        const char *at = static_cast<const char *>(p) + (static_cast<uint64_t>(static_cast<uint32_t>(n)) << (2 + both));
        const int32_t low = *reinterpret_cast<const int32_t *>(at);
        const int32_t high = *reinterpret_cast<const int32_t *>(at + 4 * both);
        return both != 0 ? static_cast<int64_t>(high) << 32 | static_cast<uint32_t>(low) : low;
    }
    // Token offsets cut to the tensors, whatever the metadata says.
    __device__ __forceinline__ int cu(int n) const {
        return static_cast<int>(
            min(max(entry(cu_seqlens, n, KDA_WIDE_CU_SEQLENS), INT64_C(0)), static_cast<int64_t>(num_tokens)));
    }
    __device__ __forceinline__ int64_t inside(int64_t slot) const { return slot > 0 && slot < num_slots ? slot : 0; }
    __device__ __forceinline__ int64_t slot(int n) const { return inside(entry(state_indices, n, KDA_WIDE_STATE_INDICES)); }
    // The slot that request n's tracked prefix goes to (0: none), and the prefix's length.
    __device__ __forceinline__ int64_t track_slot(int n) const {
        return track_indices == nullptr ? 0 : inside(entry(track_indices, n, KDA_WIDE_TRACK_INDICES));
    }
    __device__ __forceinline__ int64_t track_len(int n) const { return entry(track_lens, n, KDA_WIDE_TRACK_LENS); }
    __device__ __forceinline__ float *pool(int64_t slot, int head) const {
        return state + slot * state_stride_slot + head * state_stride_head;
    }
};

// Tokens that no request covers: zeros, spread over a grid.
template <int D, typename T, int THREADS>
__device__ __forceinline__ void linear_zero_uncovered(const LinearParams &a, int64_t block, int64_t blocks) {
    const int64_t begin = a.cu(0), end = max(a.cu(a.num_seqs), a.cu(0));
    const int64_t count = begin + (a.num_tokens - end);
    const int64_t row = static_cast<int64_t>(a.num_heads) * D;
    for (int64_t i = block; i < count; i += blocks) {
        T *out = static_cast<T *>(a.out) + (i < begin ? i : end + (i - begin)) * row;
        for (int64_t e = threadIdx.x; e < row; e += THREADS) {
            out[e] = T(0);
        }
    }
}

// Sizes that the kernels assume.
inline int check_linear_sizes(const KdaLinearArgs &a) {
    if (a.head_dim != 64 && a.head_dim != 128) {
        return KDA_ERR_UNSUPPORTED;
    }
    if (a.dtype != KDA_BF16 && a.dtype != KDA_F32) {
        return KDA_ERR_UNSUPPORTED;
    }
    if (a.num_heads <= 0 || a.num_heads > (1 << 20) || a.num_seqs < 0 || a.num_tokens < 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    return KDA_OK;
}

// The same, and pointers, strides and alignment.
inline int check_linear(const KdaLinearArgs &a) {
    if (const int rc = check_linear_sizes(a); rc != KDA_OK) {
        return rc;
    }
    const auto off = [](const void *p, uintptr_t m) { return reinterpret_cast<uintptr_t>(p) % m != 0; };
    const int64_t unit = a.dtype == KDA_BF16 ? 8 : 4;  // elements of 16 bytes
    if ((a.wide & ~kWideAll) != 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    if (a.num_tokens > 0) {
        for (const void *p : {a.q, a.k, a.v, static_cast<const void *>(a.out)}) {
            if (p == nullptr || off(p, 16)) {
                return KDA_ERR_INVALID_ARGUMENT;
            }
        }
        if (a.g == nullptr || off(a.g, 4)) {
            return KDA_ERR_INVALID_ARGUMENT;
        }
        for (const int64_t s : {a.q_stride_token, a.q_stride_head, a.k_stride_token, a.k_stride_head, a.v_stride_token,
                                a.v_stride_head}) {
            if (s % unit != 0) {
                return KDA_ERR_INVALID_ARGUMENT;
            }
        }
    }
    if (a.cu_seqlens == nullptr || off(a.cu_seqlens, (a.wide & KDA_WIDE_CU_SEQLENS) != 0 ? 8 : 4)) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    if (a.num_seqs == 0) {
        return KDA_OK;
    }
    if (a.num_slots < 0 || (a.num_slots > 0 && a.state == nullptr) || off(a.state, 16) || a.state_stride_slot % 4 != 0 ||
        a.state_stride_head % 4 != 0 || a.state_indices == nullptr ||
        off(a.state_indices, (a.wide & KDA_WIDE_STATE_INDICES) != 0 ? 8 : 4)) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    if (a.track_indices != nullptr &&
        (a.track_lens == nullptr || off(a.track_indices, (a.wide & KDA_WIDE_TRACK_INDICES) != 0 ? 8 : 4) ||
         off(a.track_lens, (a.wide & KDA_WIDE_TRACK_LENS) != 0 ? 8 : 4))) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    return KDA_OK;
}

}  // namespace kda
