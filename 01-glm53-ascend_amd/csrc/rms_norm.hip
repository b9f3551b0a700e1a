// rms_norm.hip -- residual addition and root-mean-square norm, gfx950.
//
//   h = x + r;  r <- round(h);  y = h w / sqrt(mean(h^2) + eps)
//   out = round(y), or e4m3(y / s) with s = max(max|y| / 448, 1e-12) over a
//   row or over each 128 columns of it
//
// h, the sum of squares and y are fp32; the norm reads h before it is rounded
// into the residual. y is formed as (h w) rsqrt, so the largest |y| is the
// largest |h w| times the same factor, rounded alike: it is known from the
// pass that sums the squares, and a row takes one reduction, not two.
//
// Bound by HBM: a row stays in registers between its one read and its one
// write. A lane holds 8 neighbouring columns at a time (16 or 32 bytes), so 16
// lanes hold a group of 128. Loads and stores are typed as unaligned vectors
// (gfx950 serves them at any element address): rows of odd widths take the same
// path, and only the last, partial chunk of a row goes element by element.
// One row after another of an odd width costs little: 1001 x 5003 fp32 with
// residual, see the table of kernels below.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kda_abi.h"
#include "kda_device.h"

namespace kda {
namespace {

constexpr int kVec = 8;          // columns a lane holds at a time
constexpr int kGroup = 128;      // columns of a scale group
constexpr float kFp8Max = 448.0f;
constexpr float kMinScale = 1e-12f;

struct __attribute__((packed, aligned(2))) Bf16x8 {
    uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) F32x4 {
    float w[4];
};
struct __attribute__((packed, aligned(1))) Fp8x8 {
    uint32_t w[2];
};

__device__ __forceinline__ void load8(const uint16_t *p, float (&f)[kVec]) {
    const Bf16x8 r = *reinterpret_cast<const Bf16x8 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(r.w[i] << 16);
        f[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load8(const float *p, float (&f)[kVec]) {
    const F32x4 a = *reinterpret_cast<const F32x4 *>(p);
    const F32x4 b = *reinterpret_cast<const F32x4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = a.w[i];
        f[4 + i] = b.w[i];
    }
}
__device__ __forceinline__ void store8(uint16_t *p, const float (&f)[kVec]) {
    Bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    }
    *reinterpret_cast<Bf16x8 *>(p) = r;
}
__device__ __forceinline__ void store8(float *p, const float (&f)[kVec]) {
    F32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a.w[i] = f[i];
        b.w[i] = f[4 + i];
    }
    *reinterpret_cast<F32x4 *>(p) = a;
    *reinterpret_cast<F32x4 *>(p + 4) = b;
}

// Four fp32 to four e4m3 bytes, round to nearest even. |y / s| is at most
// 448 (1 + 2^-22), which rounds to 448: nothing saturates. NaN stays NaN.
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
__device__ __forceinline__ void store8(uint8_t *p, const float (&f)[kVec]) {
    Fp8x8 r;
    r.w[0] = pack_fp8x4(f[0], f[1], f[2], f[3]);
    r.w[1] = pack_fp8x4(f[4], f[5], f[6], f[7]);
    *reinterpret_cast<Fp8x8 *>(p) = r;
}
using kda::store1;
__device__ __forceinline__ void store1(uint8_t *p, float x) {
    *p = static_cast<uint8_t>(pack_fp8x4(x, 0.0f, 0.0f, 0.0f));
}

// A chunk of a row: whole, or its first n columns (the others read as 0).
template <class T> __device__ __forceinline__ void load_chunk(const T *p, int n, float (&f)[kVec]) {
    if (n >= kVec) {
        load8(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            f[i] = i < n ? load1(p + i) : 0.0f;
        }
    }
}
template <class T> __device__ __forceinline__ void store_chunk(T *p, int n, const float (&f)[kVec]) {
    if (n >= kVec) {
        store8(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            if (i < n) {
                store1(p + i, f[i]);
            }
        }
    }
}
__device__ __forceinline__ void load_chunk(const void *p, int dtype, int64_t at, int n, float (&f)[kVec]) {
    if (dtype == KDA_F32) {
        load_chunk(static_cast<const float *>(p) + at, n, f);
    } else {
        load_chunk(static_cast<const uint16_t *>(p) + at, n, f);
    }
}

// Largest magnitude, as bits: the order of the bits of |x| is that of |x|, with
// infinity and then NaN above it, so a NaN is kept where fmaxf would drop it.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return larger(x, __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ uint32_t group_max16(uint32_t x) {
    x = dpp_max<kDppQuadXor1>(x);
    x = dpp_max<kDppQuadXor2>(x);
    x = dpp_max<kDppRowHalfMirror>(x);
    return dpp_max<kDppRowMirror>(x);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = group_max16(x);
    x = larger(x, __shfl_xor(x, 16));
    return larger(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float wave_sum(float x) {
    x = group_sum32(x);
    return x + __shfl_xor(x, 32);
}

// Sum of squares and largest magnitude of a row, in all its threads.
template <int WAVES> __device__ __forceinline__ void row_reduce(float &sum, uint32_t &top) {
    sum = wave_sum(sum);
    top = wave_max(top);
    if constexpr (WAVES > 1) {
        __shared__ float sums[WAVES];
        __shared__ uint32_t tops[WAVES];
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) {
            sums[wave] = sum;
            tops[wave] = top;
        }
        __syncthreads();
        sum = 0.0f;
        top = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {  // every thread in the same order
            sum += sums[i];
            top = larger(top, tops[i]);
        }
    }
}

__device__ __forceinline__ float scale_of(uint32_t top, float rsqrt) {
    const float s = __uint_as_float(top) * rsqrt * (1.0f / kFp8Max);
    return s < kMinScale ? kMinScale : s;  // a NaN stays one
}

// y of a chunk from h w, its 8-bit scale's group already reduced in `top` (the
// whole row's) or reduced here over 16 lanes, and the chunk's store.
template <class TO>
__device__ __forceinline__ void finish(const KdaRmsNormArgs &a, int64_t row, int col, float rsqrt, uint32_t top,
                                       float (&hw)[kVec]) {
    TO *out = static_cast<TO *>(a.out) + row * a.out_stride + col;
    const int n = a.width - col;  // may be <= 0: the lane only takes part in the group's maximum
    if constexpr (sizeof(TO) == 1) {
        if (a.group != 0) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                m = larger(m, magnitude(hw[i]));
            }
            top = group_max16(m);
        }
        const float s = scale_of(top, rsqrt);
        const float inv = rsqrt / s;
        // a zero sum of squares with eps = 0 gives an infinite factor: y is NaN there as 0 * inf is
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            hw[i] = hw[i] * inv;
        }
        if (a.group != 0 && threadIdx.x % 16 == 0 && n > 0) {
            a.scale[row * ((a.width + kGroup - 1) / kGroup) + col / kGroup] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            hw[i] *= rsqrt;
        }
    }
    if (n > 0) {
        store_chunk(out, n, hw);
    }
}

// x + r of a chunk.
template <class TX>
__device__ __forceinline__ void load_sum(const KdaRmsNormArgs &a, int64_t row, int col, int n, float (&h)[kVec]) {
    load_chunk(static_cast<const TX *>(a.x) + row * a.x_stride + col, n, h);
    if (a.residual != nullptr) {
        float r[kVec];
        load_chunk(a.residual, a.residual_dtype, row * a.residual_stride + col, n, r);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            h[i] += r[i];
        }
    }
}
__device__ __forceinline__ void store_residual(const KdaRmsNormArgs &a, int64_t row, int col, int n,
                                               const float (&h)[kVec]) {
    if (a.residual != nullptr) {
        const int64_t at = row * a.residual_stride + col;
        if (a.residual_dtype == KDA_F32) {
            store_chunk(static_cast<float *>(a.residual) + at, n, h);
        } else {
            store_chunk(static_cast<uint16_t *>(a.residual) + at, n, h);
        }
    }
}

// THREADS threads a row (64: four rows a workgroup), CHUNKS chunks of 8 columns
// a thread in registers.
template <int THREADS, int CHUNKS, class TX, class TO>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void rms_norm_kernel(const KdaRmsNormArgs a) {
    constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
    const int lane = threadIdx.x % THREADS;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / THREADS;
    if (row >= a.rows) {
        return;  // whole waves: only rows of one wave share a workgroup
    }
    float h[CHUNKS][kVec];
    float sum = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int col = (c * THREADS + lane) * kVec;
        if (col < a.width) {
            load_sum<TX>(a, row, col, a.width - col, h[c]);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                h[c][i] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int col = (c * THREADS + lane) * kVec;
        if (col < a.width) {
            float w[kVec];
            load_chunk(a.weight, a.weight_dtype, col, a.width - col, w);
            store_residual(a, row, col, a.width - col, h[c]);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                sum += h[c][i] * h[c][i];
                h[c][i] *= w[i];
                if constexpr (sizeof(TO) == 1) {
                    top = larger(top, magnitude(h[c][i]));
                }
            }
        }
    }
    row_reduce<THREADS / 64>(sum, top);
    const float rsqrt = 1.0f / sqrtf(sum / static_cast<float>(a.width) + a.eps);
    if (sizeof(TO) == 1 && a.group == 0 && lane == 0) {
        a.scale[row] = scale_of(top, rsqrt);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        // a chunk's 16 lanes leave the row's end together or not at all
        const int col = (c * THREADS + lane) * kVec;
        if (col / kGroup * kGroup < a.width) {
            finish<TO>(a, row, col, rsqrt, top, h[c]);
        }
    }
}

// A row wider than the registers hold: read twice, its second read mostly from
// the L2 cache. The residual is written in the second pass, which still reads
// the old one.
template <class TX, class TO> __global__ __launch_bounds__(1024) void rms_norm_wide_kernel(const KdaRmsNormArgs a) {
    const int64_t row = blockIdx.x;
    float sum = 0.0f;
    uint32_t top = 0;
    for (int col = threadIdx.x * kVec; col < a.width; col += 1024 * kVec) {
        float h[kVec], w[kVec];
        load_sum<TX>(a, row, col, a.width - col, h);
        load_chunk(a.weight, a.weight_dtype, col, a.width - col, w);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            sum += h[i] * h[i];
            if constexpr (sizeof(TO) == 1) {
                top = larger(top, magnitude(h[i] * w[i]));
            }
        }
    }
    row_reduce<16>(sum, top);
    const float rsqrt = 1.0f / sqrtf(sum / static_cast<float>(a.width) + a.eps);
    if (sizeof(TO) == 1 && a.group == 0 && threadIdx.x == 0) {
        a.scale[row] = scale_of(top, rsqrt);
    }
    for (int col = threadIdx.x * kVec; col / kGroup * kGroup < a.width; col += 1024 * kVec) {
        float h[kVec] = {}, w[kVec];
        if (col < a.width) {
            load_sum<TX>(a, row, col, a.width - col, h);
            load_chunk(a.weight, a.weight_dtype, col, a.width - col, w);
            store_residual(a, row, col, a.width - col, h);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                h[i] *= w[i];
            }
        }
        finish<TO>(a, row, col, rsqrt, top, h);
    }
}

template <class TX, class TO> void launch(const KdaRmsNormArgs &a, hipStream_t stream) {
    const unsigned rows = static_cast<unsigned>(a.rows);
    if (a.width <= 512) {
        rms_norm_kernel<64, 1, TX, TO><<<(rows + 3) / 4, 256, 0, stream>>>(a);
    } else if (a.width <= 2048) {
        rms_norm_kernel<256, 1, TX, TO><<<rows, 256, 0, stream>>>(a);
    } else if (a.width <= 4096) {
        rms_norm_kernel<256, 2, TX, TO><<<rows, 256, 0, stream>>>(a);
    } else if (a.width <= 8192) {
        rms_norm_kernel<256, 4, TX, TO><<<rows, 256, 0, stream>>>(a);
    } else if (a.width <= 32768) {
        rms_norm_kernel<1024, 4, TX, TO><<<rows, 1024, 0, stream>>>(a);
    } else {
        rms_norm_wide_kernel<TX, TO><<<rows, 1024, 0, stream>>>(a);
    }
}

bool is_float(int32_t dtype) { return dtype == KDA_BF16 || dtype == KDA_F32; }
bool misplaced(const void *p, int32_t dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == KDA_F32 ? 4 : 2) != 0; }

}  // namespace
}  // namespace kda

extern "C" int kda_rms_norm_launch(const KdaRmsNormArgs *args, void *stream) {
    using namespace kda;
    if (args == nullptr || args->rows < 0 || args->rows > INT32_MAX || args->width <= 0 ||
        args->width > (1 << 30)) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const KdaRmsNormArgs &a = *args;
    const bool fp8 = a.out_dtype == KDA_FP8_E4M3;
    if (!is_float(a.x_dtype) || !is_float(a.weight_dtype) || (a.residual != nullptr && !is_float(a.residual_dtype)) ||
        (!fp8 && (a.out_dtype != a.x_dtype || a.group != 0)) || (a.group != 0 && a.group != kGroup)) {
        return KDA_ERR_UNSUPPORTED;
    }
    if (a.rows == 0) {
        return KDA_OK;
    }
    if (a.x == nullptr || a.weight == nullptr || a.out == nullptr || (fp8 && a.scale == nullptr) ||
        misplaced(a.x, a.x_dtype) || misplaced(a.weight, a.weight_dtype) || misplaced(a.residual, a.residual_dtype) ||
        (!fp8 && misplaced(a.out, a.out_dtype)) || reinterpret_cast<uintptr_t>(a.scale) % 4 != 0 ||
        (a.rows > 1 && (a.out_stride < a.width || (a.residual != nullptr && a.residual_stride < a.width)))) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (a.x_dtype == KDA_F32) {
        fp8 ? launch<float, uint8_t>(a, s) : launch<float, float>(a, s);
    } else {
        fp8 ? launch<uint16_t, uint8_t>(a, s) : launch<uint16_t, uint16_t>(a, s);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}
