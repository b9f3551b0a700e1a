// linear_recurrent.hip -- linear attention with a decay for each head, token by token, gfx950.
//
//   S <- exp(g_t) S + k_t v_t^T;   out_t = scale * S^T q_t
//
// Nothing mixes the columns of S, which are the contiguous rows of the pool: a lane holds four of
// the K elements of NP rows, D / 4 lanes a row, and the state stays in its registers from the one load to the one
// store. The only sum over lanes is the readout's. The update is formed as written, in fp32, one of its two
// products and the sum in one rounding: none more than a loop over the tokens in fp32 has.
//
// Bound by HBM: a state is 4 D^2 bytes in and out for 5 D^2 operations a token. States are touched once a
// call, so their loads and stores are marked as streams. One MI355X, heads of 128: one token of 256 requests, 32 heads, in
// 172 us (5.9 TB/s); four tokens of 64 requests, 16 heads, with all checkpoints in 70 us (4.9 TB/s, mostly writes); one of one
// request in 3.7 us, a launch's time.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kda_abi.h"
#include "kda_device.h"
#include "linear_device.h"

namespace kda {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float widened(uint16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ float widened(float x) { return x; }
template <typename T> __device__ __forceinline__ T narrowed(float x) {
    if constexpr (sizeof(T) == 2) {
        return f32_to_bf16(x);
    } else {
        return x;
    }
}

// N elements in one access, or in two of 16 bytes: what the tensors' rows are aligned to.
template <typename T, int N> struct Vector {
    static constexpr int kBytes = sizeof(T) * N < 16 ? sizeof(T) * N : 16;
    typedef T type __attribute__((ext_vector_type(N), aligned(kBytes)));
    static_assert(alignof(type) == kBytes);
};

template <typename T, int D, int NP> struct Token {
    alignas(16) T q[4];
    alignas(16) T k[4];
    alignas(16) T v[NP];
    float g;
    __device__ __forceinline__ void load(const LinearParams &a, int64_t t, int head, int c, int row) {
        const T *qp = static_cast<const T *>(a.q) + t * a.q_stride_token + head * a.q_stride_head + c;
        const T *kp = static_cast<const T *>(a.k) + t * a.k_stride_token + head * a.k_stride_head + c;
        const T *vp = static_cast<const T *>(a.v) + t * a.v_stride_token + head * a.v_stride_head + row;
        typedef typename Vector<T, 4>::type four;
        *reinterpret_cast<four *>(q) = *reinterpret_cast<const four *>(qp);
        *reinterpret_cast<four *>(k) = *reinterpret_cast<const four *>(kp);
        typedef typename Vector<T, NP>::type some;
        *reinterpret_cast<some *>(v) = *reinterpret_cast<const some *>(vp);
        g = a.g[t * a.g_stride_token + head * a.g_stride_head];
    }
};

template <int D, typename T, int NP>
__global__ __launch_bounds__(kThreads) void linear_recurrent_kernel(const LinearParams a) {
    constexpr int kLanes = D / 4;                     // of a row
    constexpr int kRows = kThreads / kLanes * NP;     // rows of a workgroup
    constexpr int kTiles = D / kRows;                 // workgroups of a (request, head)
    static_assert(kTiles * kRows == D);
    linear_zero_uncovered<D, T, kThreads>(a, blockIdx.x, gridDim.x);
    const int tile = blockIdx.x % kTiles;
    const int pair = blockIdx.x / kTiles;
    const int n = pair / a.num_heads;
    const int head = pair - n * a.num_heads;
    const int kc = threadIdx.x % kLanes;
    const int row = tile * kRows + threadIdx.x / kLanes * NP;  // NP rows, one after another
    const int at = row * D + kc * 4;

    const int begin = a.cu(n), end = a.cu(n + 1);
    const int64_t slot = a.slot(n);
    float4 s[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        s[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    Token<T, D, NP> now;
    if (begin < end) {
        now.load(a, begin, head, kc * 4, row);
    }
    if (slot > 0) {
        const float *from = a.pool(slot, head) + at;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            s[p] = load4_stream(from + p * D);
        }
    }
    auto store = [&](float *to) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            store4_stream(to + at + p * D, s[p]);
        }
    };
    const int64_t track_slot = a.track_slot(n);
    const int64_t track_at = track_slot > 0 ? begin + a.track_len(n) : -1;  // stored before this token
    const bool checkpoints = a.intermediate != nullptr;

    for (int t = begin; t < end; ++t) {
        if (t == track_at) {
            store(a.pool(track_slot, head));
        }
        const Token<T, D, NP> x = now;
        if (t + 1 < end) {
            now.load(a, t + 1, head, kc * 4, row);
        }
        const float decay = expf(x.g);
        float k[4], q[4], o[NP];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k[e] = widened(x.k[e]);
            q[e] = widened(x.q[e]);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const float v = widened(x.v[p]);
            s[p].x = s[p].x * decay + k[0] * v;
            s[p].y = s[p].y * decay + k[1] * v;
            s[p].z = s[p].z * decay + k[2] * v;
            s[p].w = s[p].w * decay + k[3] * v;
            o[p] = group_sum<kLanes>(s[p].x * q[0] + s[p].y * q[1] + s[p].z * q[2] + s[p].w * q[3]) * a.scale;
        }
        if (kc == 0) {
            typedef typename Vector<T, NP>::type some;
            some y;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                y[p] = narrowed<T>(o[p]);
            }
            *reinterpret_cast<some *>(static_cast<T *>(a.out) + (static_cast<int64_t>(t) * a.num_heads + head) * D + row) = y;
        }
        if (checkpoints && slot > 0 && n < a.mid_rows && t - begin < a.mid_steps) {
            store(a.intermediate + n * a.mid_stride_req + (t - begin) * a.mid_stride_step + head * a.mid_stride_head);
        }
    }
    if (max(begin, end) == track_at) {
        store(a.pool(track_slot, head));
    }
    if (slot > 0 && !checkpoints && begin < end) {
        store(a.pool(slot, head));
    }
}

template <int D, typename T, int NP> int launch(const LinearParams &a, hipStream_t s) {
    constexpr int kTiles = D / (kThreads / (D / 4) * NP);
    const int64_t blocks = static_cast<int64_t>(a.num_seqs) * a.num_heads * kTiles;
    if (blocks > (INT64_C(1) << 24) - 1) {  // a grid counts its threads in 32 bits
        return KDA_ERR_TOO_LARGE;
    }
    linear_recurrent_kernel<D, T, NP><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

// Rows a lane: two where a call has few states, so that they spread over more CUs; else four, and of heads of 128 eight
// where requests have several tokens, since q and k are read and widened again for every tile of rows. us, heads of 128,
// states not in the caches, with 2, 4 and 8 rows:
//   1 token of 1 request, 32 heads  3.6 3.6 3.9    of 4  6.1 4.9 5.1    of 16  15.4 13.7 14.0    of 256  179 183 191
//   4 tokens of 4 requests          7.2 6.4 6.6                         of 16  20.6 16.7 12.7    of 64    68  51  51
template <int D, typename T> int launch(const LinearParams &a, hipStream_t s) {
    if (static_cast<int64_t>(a.num_seqs) * a.num_heads < 64) {
        return launch<D, T, 2>(a, s);
    }
    if constexpr (D == 128) {
        if (a.num_tokens > a.num_seqs) {
            return launch<D, T, 8>(a, s);
        }
    }
    return launch<D, T, 4>(a, s);
}

}  // namespace
}  // namespace kda

extern "C" int kda_linear_recurrent_launch(const KdaLinearArgs *args, void *stream) {
    using namespace kda;
    if (args == nullptr) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    if (const int rc = check_linear(*args); rc != KDA_OK) {
        return rc;
    }
    const LinearParams a{*args};
    if (a.intermediate != nullptr) {
        if (reinterpret_cast<uintptr_t>(a.intermediate) % 16 != 0 || a.mid_stride_req % 4 != 0 ||
            a.mid_stride_step % 4 != 0 || a.mid_stride_head % 4 != 0 || a.mid_rows < 0 || a.mid_steps < 0) {
            return KDA_ERR_INVALID_ARGUMENT;
        }
    }
    if (a.num_seqs == 0) {
        return a.num_tokens == 0 ? KDA_OK : KDA_ERR_INVALID_ARGUMENT;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (a.head_dim == 128) {
        return a.dtype == KDA_BF16 ? launch<128, uint16_t>(a, s) : launch<128, float>(a, s);
    }
    return a.dtype == KDA_BF16 ? launch<64, uint16_t>(a, s) : launch<64, float>(a, s);
}
