// paged_store.hip -- new tokens' keys and values into a paged cache, gfx950.
//
// A copy with an address per token: bound by HBM. A thread moves 16 bytes of a
// key head's row and the same 16 of its value, so two loads are in flight before
// either store; a token's threads are neighbours, so its rows are read and
// written in whole cache lines whatever its slot is. 8192 tokens of 8 heads of 128 to
// 8 bits: 11 to 12 us for 50 MB, a third of it written to scattered rows (a plain copy of as much takes 10.2 us);
// 256 tokens: 3 us, the time of an empty launch.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kda_abi.h"
#include "kda_device.h"
#include "paged_cache.h"

namespace kda {
namespace {

constexpr int kThreads = 256;

struct __attribute__((packed, aligned(2))) Bf16x8 {
    uint32_t w[4];
};

// Eight bf16 times inv to e4m3, held within its range; NaN stays NaN.
__device__ __forceinline__ uint2 to_fp8(const Bf16x8 &x, float inv) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(x.w[i] << 16) * inv;
        f[2 * i + 1] = __uint_as_float(x.w[i] & 0xffff0000u) * inv;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] = f[i] > 448.0f ? 448.0f : (f[i] < -448.0f ? -448.0f : f[i]);
    }
    uint2 r;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    r.x = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true));
    w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
    r.y = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], w, true));
    return r;
}

// shift: 2^shift threads a token (its 16-byte chunks, rounded up to a power of
// two, at most a workgroup); the rest of the workgroup takes further tokens.
// first: the launch's first token.
template <bool FP8>
__global__ __launch_bounds__(kThreads) void paged_store_kernel(const KdaPagedStoreArgs a, int shift, int64_t first) {
    const KdaPagedCache &c = a.cache;
    const int64_t t = first + static_cast<int64_t>(blockIdx.x) * (kThreads >> shift) + (threadIdx.x >> shift);
    if (t >= a.num_tokens) {
        return;
    }
    const int64_t slot = a.slots_int64 != 0 ? static_cast<const int64_t *>(a.slots)[t]
                                            : static_cast<const int32_t *>(a.slots)[t];
    if (slot < 0 || slot >= c.num_pages * c.page_size) {
        return;
    }
    const uint32_t page = static_cast<uint32_t>(slot) / static_cast<uint32_t>(c.page_size);
    const uint32_t off = static_cast<uint32_t>(slot) - page * static_cast<uint32_t>(c.page_size);
    const int row_shift = c.head_dim == 128 ? 4 : 3;  // chunks of 8 in a row
    const int chunks = c.kv_heads << row_shift;
    for (int i = threadIdx.x & ((1 << shift) - 1); i < chunks; i += 1 << shift) {
        const int h = i >> row_shift;
        const int d = (i & ((1 << row_shift) - 1)) * 8;
        const Bf16x8 k = *reinterpret_cast<const Bf16x8 *>(static_cast<const uint16_t *>(a.k) + t * a.k_stride_token +
                                                           h * a.k_stride_head + d);
        const Bf16x8 v = *reinterpret_cast<const Bf16x8 *>(static_cast<const uint16_t *>(a.v) + t * a.v_stride_token +
                                                           h * a.v_stride_head + d);
        const int64_t ko = page * c.k_stride_page + off * c.k_stride_token + h * c.k_stride_head + d;
        const int64_t vo = page * c.v_stride_page + off * c.v_stride_token + h * c.v_stride_head + d;
        if constexpr (FP8) {
            // the reciprocal once a row instead of a division an element: at most an fp32
            // rounding away from x / scale, far below the 8-bit step
            const float ik = c.k_scale != nullptr ? 1.0f / c.k_scale[h] : 1.0f;
            const float iv = c.v_scale != nullptr ? 1.0f / c.v_scale[h] : 1.0f;
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(c.k) + ko) = to_fp8(k, ik);
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(c.v) + vo) = to_fp8(v, iv);
        } else {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(c.k) + ko) = make_uint4(k.w[0], k.w[1], k.w[2], k.w[3]);
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(c.v) + vo) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
        }
    }
}

}  // namespace
}  // namespace kda

extern "C" int kda_paged_store_launch(const KdaPagedStoreArgs *args, void *stream) {
    using namespace kda;
    if (args == nullptr || args->num_tokens < 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const KdaPagedStoreArgs &a = *args;
    if (const int rc = check_cache(a.cache); rc != KDA_OK) {
        return rc;
    }
    if (a.num_tokens == 0 || a.cache.num_pages == 0) {
        return KDA_OK;
    }
    if (a.k == nullptr || a.v == nullptr || a.slots == nullptr || reinterpret_cast<uintptr_t>(a.k) % 2 != 0 ||
        reinterpret_cast<uintptr_t>(a.v) % 2 != 0 ||
        reinterpret_cast<uintptr_t>(a.slots) % (a.slots_int64 != 0 ? 8 : 4) != 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const int64_t chunks = static_cast<int64_t>(a.cache.kv_heads) * (a.cache.head_dim / 8);
    int shift = 0;
    while ((1 << shift) < chunks && (1 << shift) < kThreads) {
        ++shift;
    }
    const int tokens = kThreads >> shift;
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    // a grid counts its threads in 32 bits
    constexpr int64_t kMostGroups = (INT64_C(1) << 24) - 1;
    for (int64_t first = 0; first < a.num_tokens; first += kMostGroups * tokens) {
        const unsigned grid = static_cast<unsigned>(std::min((a.num_tokens - first + tokens - 1) / tokens, kMostGroups));
        if (a.cache.dtype == KDA_FP8_E4M3) {
            paged_store_kernel<true><<<grid, kThreads, 0, s>>>(a, shift, first);
        } else {
            paged_store_kernel<false><<<grid, kThreads, 0, s>>>(a, shift, first);
        }
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}
