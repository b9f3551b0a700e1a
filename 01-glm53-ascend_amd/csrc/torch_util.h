// torch_util.h -- what the torch operators' checks and launches share.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <utility>

#include "kda_abi.h"

namespace {

using NamedTensor = std::pair<const char *, const at::Tensor &>;

inline void check_same_device(const at::Tensor &x, const char *name, const at::Tensor &t, const char *x_name = "q") {
    TORCH_CHECK(t.device() == x.device(), name, " must be on the same device as ", x_name);
}

inline void check_ok(int status, const char *op) {
    TORCH_CHECK(status == KDA_OK, op, ": ", kda_status_string(status), " (status ", status, ")");
}

inline void *stream_of(const at::Tensor &t) {
    return static_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// The kernels run on a HIP device only; a host tensor is an error, never a
// fallback. Checked after the shape/layout rules so those are testable on a
// machine without a GPU.
inline void check_on_gpu(const char *name, const at::Tensor &t) {
    TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA (HIP) tensor");
}

// One packed token batch [1, T, H, D] (the sglang contract; a leading batch
// above one would otherwise be ignored), with T and the request count in the
// kernels' int32 range.
inline void check_packed(const char *op, const at::Tensor &q, const at::Tensor &indices) {
    TORCH_CHECK(q.size(0) == 1, op, " expects one packed token batch [1, T, H, D], got batch ",
                q.size(0));
    TORCH_CHECK(q.size(1) <= INT32_MAX && indices.numel() < INT32_MAX, op,
                " supports at most 2^31-1 tokens and requests");
}

inline void check_index_tensors(const char *op, const at::Tensor &q, const at::Tensor &indices,
                         const at::Tensor &cu_seqlens) {
    for (const auto &named : {NamedTensor{"initial_state_indices", indices},
                              NamedTensor{"cu_seqlens", cu_seqlens}}) {
        TORCH_CHECK(named.second.scalar_type() == at::kInt ||
                        named.second.scalar_type() == at::kLong,
                    named.first, " must be int32 or int64");
        TORCH_CHECK(named.second.is_contiguous(), named.first, " must be contiguous");
        TORCH_CHECK(named.second.device() == q.device(), named.first,
                    " must be on the same device as q");
    }
    TORCH_CHECK(cu_seqlens.numel() == indices.numel() + 1, op,
                ": cu_seqlens must have numReq+1 entries, got ", cu_seqlens.numel(), " for ",
                indices.numel(), " requests");
}

inline void check_track(const at::Tensor &q, const at::Tensor &indices,
                 const std::optional<at::Tensor> &track_indices,
                 const std::optional<at::Tensor> &track_lens) {
    if (!track_indices.has_value()) {
        return;
    }
    TORCH_CHECK(track_lens.has_value(), "track_state_indices requires track_state_lens");
    for (const auto &named : {NamedTensor{"track_state_indices", *track_indices},
                              NamedTensor{"track_state_lens", *track_lens}}) {
        TORCH_CHECK(named.second.scalar_type() == at::kInt ||
                        named.second.scalar_type() == at::kLong,
                    named.first, " must be int32 or int64");
        TORCH_CHECK(named.second.numel() == indices.numel(), named.first,
                    " must have one entry per request");
        TORCH_CHECK(named.second.device() == q.device(), named.first,
                    " must be on the same device as q");
    }
}

// The state pool: 4-D fp32 [slots, H, K, V] with K contiguous
// (kda_varlen_recurrent.cpp:60-74).
inline void check_pool(const at::Tensor &pool, int64_t H, int64_t D) {
    TORCH_CHECK(pool.dim() == 4 && pool.scalar_type() == at::kFloat,
                "state must be a 4-D fp32 [slots,HV,K,V] pool");
    TORCH_CHECK(pool.size(1) == H && pool.size(2) == D && pool.size(3) == D,
                "state must be [slots,HV,K,V] matching the head and feature dims");
    TORCH_CHECK(pool.stride(2) == 1 && pool.stride(3) == D,
                "state must be K-contiguous (stride(2)==1, stride(3)==", D, "), got strides (",
                pool.stride(2), ", ", pool.stride(3), ")");
}

struct PoolRef {
    float *base;
    int64_t stride_slot;
    int64_t stride_head;
    int64_t num_slots;
};

inline PoolRef pool_ref(at::Tensor &pool) {
    return PoolRef{pool.data_ptr<float>(), pool.stride(0), pool.stride(1), pool.size(0)};
}

}  // namespace
