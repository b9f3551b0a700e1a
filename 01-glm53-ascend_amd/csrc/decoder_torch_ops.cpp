// decoder_torch_ops.cpp -- torch operators of a decoder's norms and paged attention.
//
// The parts of a hybrid decoder that stand beside its KDA layers, in the same
// operator namespace and manner as those: each op validates what its kernel indexes
// against, allocates its output and scratch through the caching allocator and
// enqueues on the current stream; metadata may be int32 or int64 and is read on
// the device only. No counterpart in the reference package.

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <utility>

#include "kda_abi.h"
#include "torch_util.h"

namespace {

// ---------------------------------------------------------------------------
// add_rms_norm, add_rms_norm_fp8
// ---------------------------------------------------------------------------

bool bf16_or_fp32(const at::Tensor &t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
int32_t dtype_of(const at::Tensor &t) { return t.scalar_type() == at::kFloat ? KDA_F32 : KDA_BF16; }

// [..., width] as rows: the elements between them. Leading dimensions have to
// collapse into one (any slice of columns of a contiguous tensor does).
int64_t row_stride(const char *op, const char *name, const at::Tensor &t) {
    TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, op, ": ", name, " must be contiguous in its last dimension");
    std::optional<int64_t> stride;  // of a row
    int64_t next = 0;               // stride of the next outer dimension
    for (int64_t d = t.dim() - 2; d >= 0 && t.numel() > 0; --d) {
        if (t.size(d) == 1) {
            continue;
        }
        TORCH_CHECK(!stride.has_value() || t.stride(d) == next, op, ": ", name,
                    " must have rows at one stride, got strides ", t.strides());
        stride = stride.value_or(t.stride(d));
        next = t.stride(d) * t.size(d);
    }
    return stride.value_or(t.size(-1));
}

// The same of x, whose rows may lie in groups at a second stride.
void x_strides(const char *op, const at::Tensor &x, KdaRmsNormArgs &a) {
    TORCH_CHECK(x.size(-1) <= 1 || x.stride(-1) == 1, op, ": x must be contiguous in its last dimension");
    int64_t size[2] = {1, 1}, stride[2] = {x.size(-1), 0};
    int levels = 0;
    for (int64_t d = x.dim() - 2; d >= 0 && x.numel() > 0; --d) {
        if (x.size(d) == 1) {
            continue;
        }
        if (levels > 0 && x.stride(d) == stride[levels - 1] * size[levels - 1]) {
            size[levels - 1] *= x.size(d);
            continue;
        }
        TORCH_CHECK(levels < 2, op, ": x must have rows at one stride, or groups of rows at two, got strides ", x.strides());
        size[levels] = x.size(d);
        stride[levels] = x.stride(d);
        ++levels;
    }
    TORCH_CHECK(levels < 2 || size[0] < (1 << 22), op, " supports fewer than 2^22 rows in a group");
    a.x_stride = stride[0];
    a.x_inner = levels < 2 ? 0 : static_cast<int32_t>(size[0]);
    a.x_outer_stride = stride[1];
}

KdaRmsNormArgs norm_args(const char *op, const at::Tensor &x, const at::Tensor &weight, double eps,
                         const std::optional<at::Tensor> &residual) {
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, op, " expects x as [..., width]");
    TORCH_CHECK(bf16_or_fp32(x), op, ": x must be bf16 or fp32");
    const int64_t width = x.size(-1);
    TORCH_CHECK(width <= (1 << 30), op, " supports a width of at most 2^30");
    const int64_t rows = x.numel() / width;
    TORCH_CHECK(rows <= INT32_MAX, op, " supports at most 2^31-1 rows");
    TORCH_CHECK(bf16_or_fp32(weight), op, ": weight must be bf16 or fp32");
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == width && weight.is_contiguous(), op,
                " expects a contiguous weight of the width ", width);
    check_same_device(x, "weight", weight, "x");
    KdaRmsNormArgs a{};
    a.x = x.data_ptr();
    a.weight = weight.data_ptr();
    x_strides(op, x, a);
    a.out_stride = width;
    a.rows = rows;
    a.width = static_cast<int32_t>(width);
    a.eps = static_cast<float>(eps);
    a.x_dtype = dtype_of(x);
    a.weight_dtype = dtype_of(weight);
    a.out_dtype = a.x_dtype;
    if (residual.has_value()) {
        TORCH_CHECK(bf16_or_fp32(*residual), op, ": residual must be bf16 or fp32");
        TORCH_CHECK(residual->sizes() == x.sizes(), op, " expects residual in x's shape");
        check_same_device(x, "residual", *residual, "x");
        a.residual = residual->data_ptr();
        a.residual_stride = row_stride(op, "residual", *residual);
        a.residual_dtype = dtype_of(*residual);
        TORCH_CHECK(rows <= 1 || a.residual_stride >= width, op, ": residual is updated in place, its rows must not overlap");
    }
    return a;
}

at::Tensor add_rms_norm(const at::Tensor &x, const at::Tensor &weight, double eps,
                        const std::optional<at::Tensor> &residual) {
    const char *op = "add_rms_norm";
    KdaRmsNormArgs a = norm_args(op, x, weight, eps, residual);
    check_on_gpu("x", x);
    const c10::DeviceGuard device_guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options());
    a.out = out.data_ptr();
    check_ok(kda_rms_norm_launch(&a, stream_of(x)), op);
    return out;
}

std::tuple<at::Tensor, at::Tensor> add_rms_norm_fp8(const at::Tensor &x, const at::Tensor &weight, double eps,
                                                    const std::optional<at::Tensor> &residual, int64_t group_size) {
    const char *op = "add_rms_norm_fp8";
    KdaRmsNormArgs a = norm_args(op, x, weight, eps, residual);
    TORCH_CHECK(group_size == 0 || group_size == 128, op, " supports group_size 0 (a scale per row) or 128, got ",
                group_size);
    check_on_gpu("x", x);
    const c10::DeviceGuard device_guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = group_size == 0 ? 1 : (a.width + group_size - 1) / group_size;
    at::Tensor scale = at::empty(shape, x.options().dtype(at::kFloat));
    a.out = out.data_ptr();
    a.scale = scale.data_ptr<float>();
    a.out_dtype = KDA_FP8_E4M3;
    a.group = static_cast<int32_t>(group_size);
    check_ok(kda_rms_norm_launch(&a, stream_of(x)), op);
    return {out, scale};
}

// ---------------------------------------------------------------------------
// paged_kv_store, paged_attention
// ---------------------------------------------------------------------------

// The stride of a dimension, 0 where it has a single entry (torch leaves such strides at any number).
int64_t stride_of(const at::Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

KdaPagedCache cache_of(const char *op, const char *of, const at::Tensor &x, const at::Tensor &k_cache,
                       const at::Tensor &v_cache, const std::optional<at::Tensor> &k_scale,
                       const std::optional<at::Tensor> &v_scale) {
    TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(), op,
                " expects k_cache and v_cache as [pages, page_size, kv_heads, D]");
    const bool fp8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK((fp8 || k_cache.scalar_type() == at::kBFloat16) && v_cache.scalar_type() == k_cache.scalar_type(), op,
                ": k_cache and v_cache must both be bf16 or both float8_e4m3fn");
    const int64_t D = k_cache.size(3);
    TORCH_CHECK(D == 64 || D == 128, op, " requires D in {64, 128}, got ", D);
    TORCH_CHECK(k_cache.size(1) > 0 && k_cache.size(2) > 0 && k_cache.size(2) <= 65535, op,
                " expects pages of at least one token and 1 to 65535 kv_heads");
    TORCH_CHECK(k_cache.size(0) <= INT32_MAX / k_cache.size(1), op, " supports pools of fewer than 2^31 tokens");
    const int64_t unit = fp8 ? 16 : 8;
    for (const auto &named : {NamedTensor{"k_cache", k_cache}, NamedTensor{"v_cache", v_cache}}) {
        const at::Tensor &t = named.second;
        check_same_device(x, named.first, t, of);
        TORCH_CHECK(t.stride(3) == 1, op, ": ", named.first, " must be contiguous in D");
        TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && stride_of(t, 0) % unit == 0 &&
                        stride_of(t, 1) % unit == 0 && stride_of(t, 2) % unit == 0,
                    op, ": rows of ", named.first, " must be 16-byte aligned");
    }
    for (const auto &named : {std::pair<const char *, const std::optional<at::Tensor> &>{"k_scale", k_scale},
                              std::pair<const char *, const std::optional<at::Tensor> &>{"v_scale", v_scale}}) {
        if (named.second.has_value()) {
            const at::Tensor &t = *named.second;
            TORCH_CHECK(fp8, op, ": ", named.first, " belongs to a float8_e4m3fn cache");
            TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == k_cache.size(2) && t.is_contiguous(), op, ": ",
                        named.first, " must be contiguous fp32 with an entry per kv head");
            check_same_device(x, named.first, t, of);
        }
    }
    KdaPagedCache c{};
    c.k = k_cache.data_ptr();
    c.v = v_cache.data_ptr();
    c.k_stride_page = stride_of(k_cache, 0);
    c.k_stride_token = stride_of(k_cache, 1);
    c.k_stride_head = stride_of(k_cache, 2);
    c.v_stride_page = stride_of(v_cache, 0);
    c.v_stride_token = stride_of(v_cache, 1);
    c.v_stride_head = stride_of(v_cache, 2);
    c.k_scale = k_scale.has_value() ? k_scale->data_ptr<float>() : nullptr;
    c.v_scale = v_scale.has_value() ? v_scale->data_ptr<float>() : nullptr;
    c.num_pages = k_cache.size(0);
    c.page_size = static_cast<int32_t>(k_cache.size(1));
    c.kv_heads = static_cast<int32_t>(k_cache.size(2));
    c.head_dim = static_cast<int32_t>(D);
    c.dtype = fp8 ? KDA_FP8_E4M3 : KDA_BF16;
    return c;
}

// Token tensors [1, T, heads, D] in bf16; tokens and heads at any stride.
void check_tokens(const char *op, const char *name, const at::Tensor &t, int64_t D) {
    TORCH_CHECK(t.dim() == 4 && t.size(0) == 1 && t.size(3) == D, op, " expects ", name,
                " as one packed token batch [1, T, heads, D] with the cache's D");
    TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bf16");
    TORCH_CHECK(t.stride(3) == 1, op, ": ", name, " must be contiguous in D");
    TORCH_CHECK(t.size(1) <= INT32_MAX, op, " supports at most 2^31-1 tokens");
}

void check_index(const char *op, const char *name, const char *of, const at::Tensor &x, const at::Tensor &t, int64_t dim) {
    TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
    TORCH_CHECK(t.dim() == dim, op, " expects ", name, " with ", dim, " dimensions, got ", t.dim());
    TORCH_CHECK(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, op, ": ", name,
                " must be contiguous in its last dimension");
    check_same_device(x, name, t, of);
}

void paged_kv_store(const at::Tensor &k, const at::Tensor &v, at::Tensor &k_cache, at::Tensor &v_cache,
                    const at::Tensor &slot_indices, const std::optional<at::Tensor> &k_scale,
                    const std::optional<at::Tensor> &v_scale) {
    const char *op = "paged_kv_store";
    KdaPagedStoreArgs a{};
    a.cache = cache_of(op, "k", k, k_cache, v_cache, k_scale, v_scale);
    check_tokens(op, "k", k, a.cache.head_dim);
    check_tokens(op, "v", v, a.cache.head_dim);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(2) == a.cache.kv_heads, op,
                " expects k and v as [1, T, kv_heads, D] with the cache's kv_heads");
    check_same_device(k, "v", v, "k");
    check_index(op, "slot_indices", "k", k, slot_indices, 1);
    TORCH_CHECK(slot_indices.numel() == k.size(1), op, ": slot_indices must have an entry per token, got ",
                slot_indices.numel(), " for ", k.size(1), " tokens");
    check_on_gpu("k", k);
    const c10::DeviceGuard device_guard(k.device());
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.k_stride_token = k.stride(1);
    a.k_stride_head = k.stride(2);
    a.v_stride_token = v.stride(1);
    a.v_stride_head = v.stride(2);
    a.slots = slot_indices.data_ptr();
    a.slots_int64 = slot_indices.scalar_type() == at::kLong ? 1 : 0;
    a.num_tokens = static_cast<int32_t>(k.size(1));
    check_ok(kda_paged_store_launch(&a, stream_of(k)), op);
}

at::Tensor paged_attention(const at::Tensor &q, const at::Tensor &k_cache, const at::Tensor &v_cache,
                           const at::Tensor &page_table, const at::Tensor &kv_lens, const at::Tensor &cu_seqlens,
                           double scale, int64_t max_query_len, int64_t window, double logit_cap,
                           const std::optional<at::Tensor> &k_scale, const std::optional<at::Tensor> &v_scale) {
    const char *op = "paged_attention";
    KdaPagedAttentionArgs a{};
    a.cache = cache_of(op, "q", q, k_cache, v_cache, k_scale, v_scale);
    check_tokens(op, "q", q, a.cache.head_dim);
    const int64_t T = q.size(1), H = q.size(2), N = kv_lens.numel();
    TORCH_CHECK(H > 0 && H % a.cache.kv_heads == 0 && H <= INT32_MAX, op, " requires query heads in a multiple of kv_heads, got ", H,
                " and ", a.cache.kv_heads);
    check_index(op, "page_table", "q", q, page_table, 2);
    check_index(op, "kv_lens", "q", q, kv_lens, 1);
    check_index(op, "cu_seqlens", "q", q, cu_seqlens, 1);
    TORCH_CHECK(cu_seqlens.numel() == N + 1, op, ": cu_seqlens must have numReq+1 entries, got ", cu_seqlens.numel(),
                " for ", N, " requests");
    TORCH_CHECK(page_table.size(0) == N, op, ": page_table must have a row per request, got ", page_table.size(0),
                " for ", N, " requests");
    TORCH_CHECK(N < INT32_MAX && page_table.size(1) <= INT32_MAX && max_query_len >= 0 && max_query_len <= INT32_MAX, op,
                " supports at most 2^31-1 requests, pages and new tokens of a request");
    TORCH_CHECK(window >= 0 && window <= INT32_MAX, op, ": window must be 0 (all keys) or a number of keys, got ", window);
    TORCH_CHECK(logit_cap == 0 || (logit_cap >= 1e-30 && logit_cap <= 1e30), op,
                ": logit_cap must be 0 (none) or within 1e-30 and 1e30, got ", logit_cap);
    check_on_gpu("q", q);
    const c10::DeviceGuard device_guard(q.device());
    at::Tensor out = at::empty(q.sizes(), q.options());
    if (T == 0) {
        return out;
    }
    a.q = q.data_ptr();
    a.out = out.data_ptr();
    a.q_stride_token = q.stride(1);
    a.q_stride_head = q.stride(2);
    a.out_stride_token = out.stride(1);
    a.out_stride_head = out.stride(2);
    a.page_table = page_table.data_ptr();
    a.page_table_stride = page_table.stride(0);
    a.kv_lens = kv_lens.data_ptr();
    a.cu_seqlens = cu_seqlens.data_ptr();
    a.scale = static_cast<float>(scale);
    a.logit_cap = static_cast<float>(logit_cap);
    a.window = static_cast<int32_t>(window);
    a.wide = (page_table.scalar_type() == at::kLong ? KDA_WIDE_PAGE_TABLE : 0) |
             (kv_lens.scalar_type() == at::kLong ? KDA_WIDE_KV_LENS : 0) |
             (cu_seqlens.scalar_type() == at::kLong ? KDA_WIDE_CU_SEQLENS : 0);
    a.num_seqs = static_cast<int32_t>(N);
    a.num_tokens = static_cast<int32_t>(T);
    a.num_heads = static_cast<int32_t>(H);
    a.max_pages = static_cast<int32_t>(page_table.size(1));
    a.max_query_len = static_cast<int32_t>(max_query_len);
    const size_t bytes = kda_paged_attention_workspace_bytes(&a);
    std::optional<at::Tensor> workspace;
    if (bytes > 0) {
        workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    }
    check_ok(kda_paged_attention_launch(&a, workspace.has_value() ? workspace->data_ptr() : nullptr, bytes, stream_of(q)),
             op);
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sgl_glm53_ascend, m) {
    m.def("add_rms_norm(Tensor x, Tensor weight, float eps, *, Tensor(a!)? residual=None) -> Tensor");
    m.def(
        "add_rms_norm_fp8(Tensor x, Tensor weight, float eps, *, Tensor(a!)? residual=None, "
        "int group_size=0) -> (Tensor, Tensor)");
    m.def(
        "paged_kv_store(Tensor k, Tensor v, *, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slot_indices, "
        "Tensor? k_scale=None, Tensor? v_scale=None) -> ()");
    m.def(
        "paged_attention(Tensor q, *, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor kv_lens, "
        "Tensor cu_seqlens, float scale, int max_query_len, int window=0, float logit_cap=0.0, "
        "Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor");
}

#define DECODER_REGISTER_IMPLS(m)                    \
    m.impl("add_rms_norm", &add_rms_norm);           \
    m.impl("add_rms_norm_fp8", &add_rms_norm_fp8);   \
    m.impl("paged_kv_store", &paged_kv_store);       \
    m.impl("paged_attention", &paged_attention)

TORCH_LIBRARY_IMPL(sgl_glm53_ascend, CUDA, m) { DECODER_REGISTER_IMPLS(m); }

// Host tensors reach the same validation and then fail at the device check.
TORCH_LIBRARY_IMPL(sgl_glm53_ascend, CPU, m) { DECODER_REGISTER_IMPLS(m); }
