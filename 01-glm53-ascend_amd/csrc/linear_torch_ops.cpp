// linear_torch_ops.cpp -- torch operators of linear attention with a decay for each head.
//
// The plain member of the KDA operators' family (no delta rule, one decay a head), in their namespace
// and manner and on their state pool: each op validates what its kernels index against, allocates its
// output and scratch through the caching allocator and enqueues on the current stream; metadata may be int32
// or int64 and is read on the device only. No counterpart in the reference package.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <optional>

#include "kda_abi.h"
#include "torch_util.h"

namespace {

// Metadata that the arguments point into: kept until the launch.
struct LinearCall {
    KdaLinearArgs args{};
    at::Tensor track_indices, track_lens;
};

// The stride of a dimension, 0 where it has a single entry (torch leaves such strides at any number).
int64_t stride_at(const at::Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

LinearCall linear_args(const char *op, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g,
                       at::Tensor &pool, const at::Tensor &indices, const at::Tensor &cu_seqlens, double scale,
                       const std::optional<at::Tensor> &track_indices, const std::optional<at::Tensor> &track_lens) {
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, op, " expects q, k, v as [1, T, H, D]");
    check_packed(op, q, indices);
    const auto dt = q.scalar_type();
    TORCH_CHECK(dt == at::kBFloat16 || dt == at::kFloat, op, ": q must be bf16 or fp32");
    TORCH_CHECK(k.sizes() == q.sizes() && v.sizes() == q.sizes(), op, " expects q, k, v all [1, T, H, D] with K == V");
    const int64_t T = q.size(1), H = q.size(2), D = q.size(3);
    TORCH_CHECK(D == 64 || D == 128, op, " requires K == V in {64, 128}, got ", D);
    TORCH_CHECK(H > 0 && H <= (1 << 20), op, " supports 1 to 2^20 heads");
    const int64_t unit = dt == at::kFloat ? 4 : 8;
    for (const auto &named : {NamedTensor{"q", q}, NamedTensor{"k", k}, NamedTensor{"v", v}}) {
        const at::Tensor &t = named.second;
        TORCH_CHECK(t.scalar_type() == dt, named.first, " must have q's dtype");
        TORCH_CHECK(t.stride(3) == 1, op, ": ", named.first, " must be contiguous in D");
        TORCH_CHECK(t.numel() == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && stride_at(t, 1) % unit == 0 &&
                                       stride_at(t, 2) % unit == 0),
                    op, ": rows of ", named.first, " must be 16-byte aligned");
        check_same_device(q, named.first, t);
    }
    TORCH_CHECK(g.scalar_type() == at::kFloat, "g must be fp32");
    TORCH_CHECK((g.dim() == 1 && g.size(0) == H) || (g.dim() == 3 && g.size(0) == 1 && g.size(1) == T && g.size(2) == H), op,
                " expects g as [H] (a log decay for each head) or [1, T, H] (for each token and head)");
    check_same_device(q, "g", g);
    check_pool(pool, H, D);
    TORCH_CHECK(pool.numel() == 0 || (reinterpret_cast<uintptr_t>(pool.data_ptr()) % 16 == 0 && stride_at(pool, 0) % 4 == 0 &&
                                      stride_at(pool, 1) % 4 == 0),
                op, ": rows of state must be 16-byte aligned");
    check_same_device(q, "initial_state_source", pool);
    check_index_tensors(op, q, indices, cu_seqlens);
    check_track(q, indices, track_indices, track_lens);
    LinearCall call;
    KdaLinearArgs &a = call.args;
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.q_stride_token = stride_at(q, 1);
    a.q_stride_head = stride_at(q, 2);
    a.k_stride_token = stride_at(k, 1);
    a.k_stride_head = stride_at(k, 2);
    a.v_stride_token = stride_at(v, 1);
    a.v_stride_head = stride_at(v, 2);
    a.g = g.data_ptr<float>();
    a.g_stride_token = g.dim() == 3 ? stride_at(g, 1) : 0;
    a.g_stride_head = stride_at(g, g.dim() - 1);
    const PoolRef pr = pool_ref(pool);
    a.state = pr.base;
    a.state_stride_slot = pr.num_slots > 1 ? pr.stride_slot : 0;
    a.state_stride_head = H > 1 ? pr.stride_head : 0;
    a.num_slots = pr.num_slots;
    a.state_indices = indices.data_ptr();
    a.cu_seqlens = cu_seqlens.data_ptr();
    a.wide = (indices.scalar_type() == at::kLong ? KDA_WIDE_STATE_INDICES : 0) |
             (cu_seqlens.scalar_type() == at::kLong ? KDA_WIDE_CU_SEQLENS : 0);
    if (track_indices.has_value()) {
        call.track_indices = track_indices->contiguous();
        call.track_lens = track_lens->contiguous();
        a.track_indices = call.track_indices.data_ptr();
        a.track_lens = call.track_lens.data_ptr();
        a.wide |= (call.track_indices.scalar_type() == at::kLong ? KDA_WIDE_TRACK_INDICES : 0) |
                  (call.track_lens.scalar_type() == at::kLong ? KDA_WIDE_TRACK_LENS : 0);
    }
    a.scale = static_cast<float>(scale);
    a.num_seqs = static_cast<int32_t>(indices.numel());
    a.num_tokens = static_cast<int32_t>(T);
    a.num_heads = static_cast<int32_t>(H);
    a.head_dim = static_cast<int32_t>(D);
    a.dtype = dt == at::kFloat ? KDA_F32 : KDA_BF16;
    return call;
}

at::Tensor linear_varlen_recurrent(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g,
                                   at::Tensor &initial_state_source, const at::Tensor &initial_state_indices,
                                   const at::Tensor &cu_seqlens, double scale,
                                   const std::optional<at::Tensor> &intermediate_state,
                                   const std::optional<at::Tensor> &track_state_indices,
                                   const std::optional<at::Tensor> &track_state_lens) {
    const char *op = "linear_varlen_recurrent";
    LinearCall call = linear_args(op, q, k, v, g, initial_state_source, initial_state_indices, cu_seqlens, scale,
                                  track_state_indices, track_state_lens);
    KdaLinearArgs &a = call.args;
    if (intermediate_state.has_value()) {
        const at::Tensor &mid = *intermediate_state;
        TORCH_CHECK(mid.dim() == 5 && mid.scalar_type() == at::kFloat,
                    "intermediate_state must be a 5-D fp32 [slots,steps,HV,K,V] buffer");
        TORCH_CHECK(mid.size(2) == a.num_heads && mid.size(3) == a.head_dim && mid.size(4) == a.head_dim,
                    "intermediate_state must be [slots,steps,HV,K,V] matching the head and feature dims");
        TORCH_CHECK(mid.stride(3) == 1 && mid.stride(4) == a.head_dim,
                    "intermediate_state must be K-contiguous (stride(3)==1, stride(4)==", a.head_dim, "), got strides (",
                    mid.stride(3), ", ", mid.stride(4), ")");
        TORCH_CHECK(mid.numel() == 0 || (reinterpret_cast<uintptr_t>(mid.data_ptr()) % 16 == 0 && stride_at(mid, 0) % 4 == 0 &&
                                         stride_at(mid, 1) % 4 == 0 && stride_at(mid, 2) % 4 == 0),
                    op, ": rows of intermediate_state must be 16-byte aligned");
        check_same_device(q, "intermediate_state", mid);
        TORCH_CHECK(mid.size(0) >= a.num_seqs, "intermediate_state needs a row per request, got ", mid.size(0), " for ",
                    a.num_seqs, " requests");
        TORCH_CHECK(mid.size(1) * a.num_seqs >= a.num_tokens || a.num_seqs == 0, "intermediate_state has ", mid.size(1),
                    " step rows, too few for ", a.num_tokens, " tokens across ", a.num_seqs, " requests");
        a.intermediate = mid.data_ptr<float>();
        a.mid_stride_req = stride_at(mid, 0);
        a.mid_stride_step = stride_at(mid, 1);
        a.mid_stride_head = stride_at(mid, 2);
        a.mid_rows = mid.size(0);
        a.mid_steps = mid.size(1);
    }
    check_on_gpu("q", q);
    const c10::DeviceGuard device_guard(q.device());
    at::Tensor out = at::empty(q.sizes(), q.options());
    if (a.num_seqs == 0) {
        return out.zero_();
    }
    a.out = out.data_ptr();
    check_ok(kda_linear_recurrent_launch(&a, stream_of(q)), op);
    return out;
}

at::Tensor linear_varlen_chunk(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &g,
                               at::Tensor &initial_state_source, const at::Tensor &initial_state_indices,
                               const at::Tensor &cu_seqlens, double scale,
                               const std::optional<at::Tensor> &track_state_indices,
                               const std::optional<at::Tensor> &track_state_lens) {
    const char *op = "linear_varlen_chunk";
    LinearCall call = linear_args(op, q, k, v, g, initial_state_source, initial_state_indices, cu_seqlens, scale,
                                  track_state_indices, track_state_lens);
    KdaLinearArgs &a = call.args;
    TORCH_CHECK(a.dtype == KDA_BF16, op, " takes bf16 q, k, v (bf16 MFMA operands)");
    check_on_gpu("q", q);
    const c10::DeviceGuard device_guard(q.device());
    at::Tensor out = at::empty(q.sizes(), q.options());
    if (a.num_seqs == 0) {
        return out.zero_();
    }
    a.out = out.data_ptr();
    const size_t bytes = kda_linear_chunk_workspace_bytes(&a);
    at::Tensor workspace;
    if (bytes > 0) {
        workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    }
    check_ok(kda_linear_chunk_launch(&a, bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)), op);
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sgl_glm53_ascend, m) {
    m.def(
        "linear_varlen_recurrent(Tensor q, Tensor k, Tensor v, Tensor g, *, Tensor(a!) initial_state_source, "
        "Tensor initial_state_indices, Tensor cu_seqlens, float scale, Tensor(b!)? intermediate_state=None, "
        "Tensor? track_state_indices=None, Tensor? track_state_lens=None) -> Tensor");
    m.def(
        "linear_varlen_chunk(Tensor q, Tensor k, Tensor v, Tensor g, *, Tensor(a!) initial_state_source, "
        "Tensor initial_state_indices, Tensor cu_seqlens, float scale, "
        "Tensor? track_state_indices=None, Tensor? track_state_lens=None) -> Tensor");
}

#define LINEAR_REGISTER_IMPLS(m)                                 \
    m.impl("linear_varlen_recurrent", &linear_varlen_recurrent); \
    m.impl("linear_varlen_chunk", &linear_varlen_chunk)

TORCH_LIBRARY_IMPL(sgl_glm53_ascend, CUDA, m) { LINEAR_REGISTER_IMPLS(m); }

// Host tensors reach the same validation and then fail at the device check.
TORCH_LIBRARY_IMPL(sgl_glm53_ascend, CPU, m) { LINEAR_REGISTER_IMPLS(m); }
