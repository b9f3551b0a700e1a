// rms_norm.hip -- residual addition and root-mean-square norm, gfx950.
//
//   h = x + r;  r <- round(h);  y = h w / sqrt(mean(h^2) + eps)
//   out = round(y), or e4m3(y / s) with s = max(max|y| / 448, 1e-12) over a
//   row or over each 128 columns of it
//
// h, the sum of squares and y are fp32; the norm reads h before it is rounded
// into the residual. y is formed as (h w) rsqrt, so the largest |y| is the
// largest |h w| times the same factor, rounded alike: it is known from the
// pass that sums the squares, and a row takes one reduction, not two. An 8-bit output is
// (h w)(rsqrt / s) accordingly, a few fp32 roundings from y / s: a value beside a tie
// may take the neighbouring 8-bit step, with the same error against exact arithmetic.
//
// Bound by HBM: a row stays in registers between its one read and its one
// write. A lane holds 16 bytes of the input at a time (8 or 4 columns), so 16 or 32
// lanes hold a group of 128, and all of a row's loads are issued before the
// first is waited for. x and the residual are streamed (read or written once); the
// weight and the output, which the next kernel reads, stay in the caches. Loads and
// stores are typed as unaligned vectors (gfx950 serves them at any element
// address), so rows of odd widths take the same path; the last, partial chunk of a row is loaded as the
// row's last whole vector and moved down in registers, and stored element by element.
//
// Measured, residual read and written: 8192 x 8192 bf16 to 8 bits with a scale per 128
// columns 75 us = 6.3 TB/s (reading alone reaches 6.1 to 6.4 on this card, a copy 4.9), with one
// per row 75.5;
// 1001 x 5003 fp32 16 us = 5.0 TB/s; one row 3 us.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kda_abi.h"
#include "kda_device.h"

namespace kda {
namespace {

constexpr int kGroup = 128;      // columns of a scale group
constexpr float kFp8Max = 448.0f;
constexpr float kMinScale = 1e-12f;

// Vectors at any element address.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int BYTES> struct Any;
template <> struct Any<16> {
    typedef u32x4 T __attribute__((aligned(1)));
};
template <> struct Any<8> {
    typedef u32x2 T __attribute__((aligned(1)));
};
template <> struct Any<4> {
    typedef uint32_t T __attribute__((aligned(1)));
};
// STREAM: data read or written once. (A template argument: of a choice at run time the compiler
// makes one access, without the hint.)
template <class A, bool STREAM, class T> __device__ __forceinline__ auto load_as(const T *p) {
    const typename A::T *q = reinterpret_cast<const typename A::T *>(p);
    if constexpr (STREAM) {
        return __builtin_nontemporal_load(q);
    } else {
        return *q;
    }
}
template <class A, bool STREAM, class T, class R> __device__ __forceinline__ void store_as(T *p, R r) {
    if constexpr (STREAM) {
        __builtin_nontemporal_store(r, reinterpret_cast<typename A::T *>(p));
    } else {
        *reinterpret_cast<typename A::T *>(p) = r;
    }
}

// A row's first element in x; rows of a launch are counted in 32 bits.
__device__ __forceinline__ int64_t x_at(const KdaRmsNormArgs &a, int64_t row) {
    if (a.x_inner > 1) {
        const uint32_t r = static_cast<uint32_t>(row), outer = r / static_cast<uint32_t>(a.x_inner);
        return outer * a.x_outer_stride + static_cast<int64_t>(r - outer * a.x_inner) * a.x_stride;
    }
    return row * a.x_stride;
}

// Columns a lane holds at a time: 16 bytes of the input, so that the lanes of a load are neighbours.
template <class T> constexpr int kVec = 16 / sizeof(T);

// V (4 or 8) consecutive elements as they stand in memory, and as fp32.
template <class T, int V> struct Raw {
    static constexpr int kBytes = V * sizeof(T);
    uint32_t w[kBytes / 4];
    template <bool STREAM> __device__ __forceinline__ void load(const T *p) {
        if constexpr (kBytes == 8) {
            const u32x2 r = load_as<Any<8>, STREAM>(p);
            w[0] = r[0];
            w[1] = r[1];
        } else {
#pragma unroll
            for (int j = 0; j < kBytes / 16; ++j) {
                const u32x4 r = load_as<Any<16>, STREAM>(reinterpret_cast<const char *>(p) + 16 * j);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[4 * j + i] = r[i];
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (sizeof(T) == 4) {
                f[i] = __uint_as_float(w[i]);
            } else {
                f[i] = __uint_as_float(i % 2 == 0 ? w[i / 2] << 16 : w[i / 2] & 0xffff0000u);
            }
        }
    }
};
template <int V, bool STREAM> __device__ __forceinline__ void store(uint16_t *p, const float (&f)[V]) {
    if constexpr (V == 8) {
        store_as<Any<16>, STREAM>(p, u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])});
    } else {
        store_as<Any<8>, STREAM>(p, u32x2{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])});
    }
}
template <int V, bool STREAM> __device__ __forceinline__ void store(float *p, const float (&f)[V]) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        store_as<Any<16>, STREAM>(p + j, u32x4{__float_as_uint(f[j]), __float_as_uint(f[j + 1]), __float_as_uint(f[j + 2]), __float_as_uint(f[j + 3])});
    }
}

// Four fp32 to four e4m3 bytes, round to nearest even. |y / s| is at most
// 448 (1 + 2^-22), which rounds to 448: nothing saturates. NaN stays NaN.
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
template <int V, bool STREAM> __device__ __forceinline__ void store(uint8_t *p, const float (&f)[V]) {
    if constexpr (V == 8) {
        store_as<Any<8>, STREAM>(p, u32x2{pack_fp8x4(f[0], f[1], f[2], f[3]), pack_fp8x4(f[4], f[5], f[6], f[7])});
    } else {
        store_as<Any<4>, STREAM>(p, pack_fp8x4(f[0], f[1], f[2], f[3]));
    }
}
using kda::store1;
__device__ __forceinline__ void store1(uint8_t *p, float x) {
    *p = static_cast<uint8_t>(pack_fp8x4(x, 0.0f, 0.0f, 0.0f));
}

// Chunk c of a lane: V columns from `col`. Where the row ends inside it or before it, the row's last V
// columns are loaded instead and moved down, zeros after them: loads that no branch holds back, which a
// lane by lane choice of a shorter one would (every load is then waited for before the next is issued).
struct Place {
    int col;    // may lie past the row's end
    int at;     // the load's first column
    bool any;   // the lanes that share the row in a wave have columns of it in this chunk
    bool tail;  // and some lane's end before its chunk does
};
template <int V, int LANES> __device__ __forceinline__ Place place(int index, int wave_first, int width) {
    Place p;
    p.col = index * V;
    p.at = min(p.col, width - V);
    p.any = wave_first * V < width;
    p.tail = (wave_first + LANES) * V > width;
    return p;
}
template <int V> __device__ __forceinline__ void move_down(const Place &p, float (&f)[V]) {
    const int by = p.col - p.at;
#pragma unroll
    for (int s = V / 2; s > 0; s /= 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float from = i + s < V ? f[i + s] : 0.0f;
            f[i] = (by & s) != 0 ? from : f[i];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        f[i] = by >= V ? 0.0f : f[i];
    }
}
template <int V, bool STREAM, class T> __device__ __forceinline__ void store_chunk(T *p, int n, const float (&f)[V]) {
    if (n >= V) {
        store<V, STREAM>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (i < n) {
                store1(p + i, f[i]);
            }
        }
    }
}

// Largest magnitude, as bits: the order of the bits of |x| is that of |x|, with
// infinity and then NaN above it, so a NaN is kept where fmaxf would drop it.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
    return larger(x, __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false));
}
template <int LANES> __device__ __forceinline__ uint32_t group_max(uint32_t x) {  // of 16 or 32 lanes
    x = dpp_max<kDppQuadXor1>(x);
    x = dpp_max<kDppQuadXor2>(x);
    x = dpp_max<kDppRowHalfMirror>(x);
    x = dpp_max<kDppRowMirror>(x);
    return LANES == 16 ? x : larger(x, __shfl_xor(x, 16));
}

// Sum of squares and largest magnitude of a row, in all its threads (16, 32, 64 or more).
template <int THREADS> __device__ __forceinline__ void row_reduce(float &sum, uint32_t &top) {
    constexpr int WAVES = THREADS / 64;
    if constexpr (THREADS == 16) {
        sum = group_sum16(sum);
        top = group_max<16>(top);
    } else {
        sum = group_sum32(sum);
        top = group_max<32>(top);
    }
    if constexpr (THREADS >= 64) {
        sum += __shfl_xor(sum, 32);
        top = larger(top, __shfl_xor(top, 32));
    }
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
// whole row's) or reduced here over the group's lanes, and the chunk's store.
template <class TO, int V>
__device__ __forceinline__ void finish(const KdaRmsNormArgs &a, int64_t row, int col, float rsqrt, uint32_t top,
                                       float (&hw)[V]) {
    TO *out = static_cast<TO *>(a.out) + row * a.out_stride + col;
    const int n = a.width - col;  // may be <= 0: the lane only takes part in the group's maximum
    if constexpr (sizeof(TO) == 1) {
        if (a.group != 0) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                m = larger(m, magnitude(hw[i]));
            }
            top = group_max<kGroup / V>(m);
        }
        const float s = scale_of(top, rsqrt);
        const float inv = rsqrt / s;
        // a zero sum of squares with eps = 0 gives an infinite factor: y is NaN there as 0 * inf is
#pragma unroll
        for (int i = 0; i < V; ++i) {
            hw[i] = hw[i] * inv;
        }
        if (a.group != 0 && threadIdx.x % (kGroup / V) == 0 && n > 0) {
            a.scale[row * ((a.width + kGroup - 1) / kGroup) + col / kGroup] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            hw[i] *= rsqrt;
        }
    }
    if (n > 0) {
        store_chunk<V, false>(out, n, hw);
    }
}

// A row's columns in registers: CHUNKS chunks of V a thread, THREADS threads a row.
template <int V, int THREADS, int CHUNKS> struct Columns {
    __device__ __forceinline__ static Place at(int c, int width) {
        const int lane = threadIdx.x % THREADS;
        constexpr int kTogether = THREADS < 64 ? THREADS : 64;  // lanes of one row in a wave
        const int first = THREADS <= 64 ? 0 : __builtin_amdgcn_readfirstlane(lane & ~63);
        return place<V, kTogether>(c * THREADS + lane, c * THREADS + first, width);
    }
    // f(chunk, place, columns) for every chunk of an array that the wave has columns in; all loads first
    template <bool STREAM, class T, class F> __device__ __forceinline__ static void each(const T *row, int width, F f) {
        Raw<T, V> raw[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const Place p = at(c, width);
            if (p.any) {
                raw[c].template load<STREAM>(row + p.at);
            }
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const Place p = at(c, width);
            if (p.any) {
                float x[V];
                raw[c].get(x);
                if (p.tail) {
                    move_down<V>(p, x);
                }
                f(c, p, x);
            }
        }
    }
    template <bool STREAM, class F> __device__ __forceinline__ static void each(const void *row, int dtype, int64_t at, int width, F f) {
        if (dtype == KDA_F32) {
            each<STREAM>(static_cast<const float *>(row) + at, width, f);
        } else {
            each<STREAM>(static_cast<const uint16_t *>(row) + at, width, f);
        }
    }
};

// THREADS threads a row (fewer than 256: several rows a workgroup); width >= V.
template <int THREADS, int CHUNKS, class TX, class TO>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void rms_norm_kernel(const KdaRmsNormArgs a) {
    constexpr int V = kVec<TX>;
    using Row = Columns<V, THREADS, CHUNKS>;
    constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / THREADS;
    if (row >= a.rows) {
        return;  // all threads of a row, and no barrier follows where rows share a workgroup
    }
    float h[CHUNKS][V];
    float sum = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            h[c][i] = 0.0f;
        }
    }
    const TX *x = static_cast<const TX *>(a.x) + x_at(a, row);
    Raw<TX, V> raw[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const Place p = Row::at(c, a.width);
        if (p.any) {
            raw[c].template load<true>(x + p.at);
        }
    }
    const auto take_x = [&](int c, const Place &p) {
        raw[c].get(h[c]);
        if (p.tail) {
            move_down<V>(p, h[c]);
        }
    };
    if (a.residual != nullptr) {
        const int64_t at = row * a.residual_stride;
        Row::template each<true>(a.residual, a.residual_dtype, at, a.width, [&](int c, const Place &p, const float (&r)[V]) {
            take_x(c, p);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[c][i] += r[i];
            }
            // read again only a layer later
            if (a.residual_dtype == KDA_F32) {
                store_chunk<V, true>(static_cast<float *>(a.residual) + at + p.col, a.width - p.col, h[c]);
            } else {
                store_chunk<V, true>(static_cast<uint16_t *>(a.residual) + at + p.col, a.width - p.col, h[c]);
            }
        });
    } else {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const Place p = Row::at(c, a.width);
            if (p.any) {
                take_x(c, p);
            }
        }
    }
    Row::template each<false>(a.weight, a.weight_dtype, 0, a.width, [&](int c, const Place &, const float (&w)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum += h[c][i] * h[c][i];
            h[c][i] *= w[i];
            if constexpr (sizeof(TO) == 1) {
                top = larger(top, magnitude(h[c][i]));
            }
        }
    });
    row_reduce<THREADS>(sum, top);
    const float rsqrt = 1.0f / sqrtf(sum / static_cast<float>(a.width) + a.eps);
    if (sizeof(TO) == 1 && a.group == 0 && threadIdx.x % THREADS == 0) {
        a.scale[row] = scale_of(top, rsqrt);
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const Place p = Row::at(c, a.width);
        if (p.any) {
            finish<TO, V>(a, row, p.col, rsqrt, top, h[c]);
        }
    }
}

// A row wider than the registers hold: read twice, its second read mostly from the caches. The residual
// is written in the second pass, which still reads the old one. Rows of less than 8 columns come here too:
// no vector fits them.
template <class TX, class TO> __global__ __launch_bounds__(1024) void rms_norm_wide_kernel(const KdaRmsNormArgs a) {
    constexpr int V = kVec<TX>;
    const int64_t row = blockIdx.x;
    const auto columns = [&](const void *p, int dtype, int64_t at, int n, float (&f)[V]) {
        if (n >= V) {
            if (dtype == KDA_F32) {
                Raw<float, V> r;
                r.template load<false>(static_cast<const float *>(p) + at);
                r.get(f);
            } else {
                Raw<uint16_t, V> r;
                r.template load<false>(static_cast<const uint16_t *>(p) + at);
                r.get(f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                f[i] = i >= n ? 0.0f
                              : dtype == KDA_F32 ? load1(static_cast<const float *>(p) + at + i)
                                                 : load1(static_cast<const uint16_t *>(p) + at + i);
            }
        }
    };
    const auto sum_of = [&](int col, int n, float (&h)[V]) {
        columns(a.x, a.x_dtype, x_at(a, row) + col, n, h);
        if (a.residual != nullptr) {
            float r[V];
            columns(a.residual, a.residual_dtype, row * a.residual_stride + col, n, r);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] += r[i];
            }
        }
    };
    float sum = 0.0f;
    uint32_t top = 0;
    for (int col = threadIdx.x * V; col < a.width; col += 1024 * V) {
        float h[V], w[V];
        sum_of(col, a.width - col, h);
        columns(a.weight, a.weight_dtype, col, a.width - col, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum += h[i] * h[i];
            if constexpr (sizeof(TO) == 1) {
                top = larger(top, magnitude(h[i] * w[i]));
            }
        }
    }
    row_reduce<1024>(sum, top);
    const float rsqrt = 1.0f / sqrtf(sum / static_cast<float>(a.width) + a.eps);
    if (sizeof(TO) == 1 && a.group == 0 && threadIdx.x == 0) {
        a.scale[row] = scale_of(top, rsqrt);
    }
    for (int col = threadIdx.x * V; col / kGroup * kGroup < a.width; col += 1024 * V) {
        float h[V] = {}, w[V];
        const int n = a.width - col;
        if (n > 0) {
            sum_of(col, n, h);
            columns(a.weight, a.weight_dtype, col, n, w);
            if (a.residual != nullptr) {
                const int64_t at = row * a.residual_stride + col;
                if (a.residual_dtype == KDA_F32) {
                    store_chunk<V, false>(static_cast<float *>(a.residual) + at, n, h);
                } else {
                    store_chunk<V, false>(static_cast<uint16_t *>(a.residual) + at, n, h);
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] *= w[i];
            }
        }
        finish<TO, V>(a, row, col, rsqrt, top, h);
    }
}

// Threads a row, by its width: few enough that each has columns, more where a row would not fit their
// registers. TB/s of 0.27 GB, bf16 with residual, and with the neighbouring choice:
//   <= 128    16 lanes (fp32: 32)   262144 x 128   6.0   3.7 with 32 lanes
//   <= 256    32 lanes (fp32: 64)   131072 x 256   6.0   3.5 with a wave
//   <= 2048   a wave                32768 x 1024   6.25  4.8 with 256 threads;  16384 x 2048  6.25, 5.7
//   <= 8192   256 threads           8192 x 4096    5.9   5.6 with a wave, 5.2 with 1024 threads
//   <= 32768  1024 threads          2048 x 16384   5.6   4.6 read twice;        1024 x 32768  5.35, 4.1
template <class TX, class TO> void launch_rows(const KdaRmsNormArgs &a, hipStream_t stream) {
    constexpr int C = 8 / kVec<TX>;  // chunks in 8 columns
    const unsigned rows = static_cast<unsigned>(a.rows);
    if (a.width < 8) {
        rms_norm_wide_kernel<TX, TO><<<rows, 1024, 0, stream>>>(a);
    } else if (a.width <= 128) {
        constexpr int kThreads = 128 / kVec<TX>, kRows = 256 / kThreads;
        rms_norm_kernel<kThreads, 1, TX, TO><<<(rows + kRows - 1) / kRows, 256, 0, stream>>>(a);
    } else if (a.width <= 256) {
        constexpr int kThreads = 256 / kVec<TX>, kRows = 256 / kThreads;
        rms_norm_kernel<kThreads, 1, TX, TO><<<(rows + kRows - 1) / kRows, 256, 0, stream>>>(a);
    } else if (a.width <= 512) {
        rms_norm_kernel<64, C, TX, TO><<<(rows + 3) / 4, 256, 0, stream>>>(a);
    } else if (a.width <= 1024) {
        rms_norm_kernel<64, 2 * C, TX, TO><<<(rows + 3) / 4, 256, 0, stream>>>(a);
    } else if (a.width <= 2048) {
        rms_norm_kernel<64, 4 * C, TX, TO><<<(rows + 3) / 4, 256, 0, stream>>>(a);
    } else if (a.width <= 4096) {
        rms_norm_kernel<256, 2 * C, TX, TO><<<rows, 256, 0, stream>>>(a);
    } else if (a.width <= 8192) {
        rms_norm_kernel<256, 4 * C, TX, TO><<<rows, 256, 0, stream>>>(a);
    } else if (a.width <= 32768) {
        rms_norm_kernel<1024, 4 * C, TX, TO><<<rows, 1024, 0, stream>>>(a);
    } else {
        rms_norm_wide_kernel<TX, TO><<<rows, 1024, 0, stream>>>(a);
    }
}

// A grid counts its threads in 32 bits: kMostRows rows of at most 1024 a launch (whole groups of x_inner).
constexpr int64_t kMostRows = (INT64_C(1) << 22) - 1;
template <class TX, class TO> void launch(KdaRmsNormArgs a, hipStream_t stream) {
    const int64_t inner = a.x_inner > 1 ? a.x_inner : 1, most = kMostRows / inner * inner;
    const int64_t scales = a.group == 0 ? 1 : (static_cast<int64_t>(a.width) + kGroup - 1) / kGroup;
    for (int64_t left = a.rows; left > 0; left -= a.rows) {
        a.rows = left < most ? left : most;
        launch_rows<TX, TO>(a, stream);
        a.x = static_cast<const TX *>(a.x) + (inner > 1 ? a.rows / inner * a.x_outer_stride : a.rows * a.x_stride);
        a.out = static_cast<TO *>(a.out) + a.rows * a.out_stride;
        if (a.residual != nullptr) {
            a.residual = static_cast<char *>(a.residual) + a.rows * a.residual_stride * (a.residual_dtype == KDA_F32 ? 4 : 2);
        }
        if (a.scale != nullptr) {
            a.scale += a.rows * scales;
        }
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
    if (a.x_inner > kMostRows) {
        return KDA_ERR_TOO_LARGE;
    }
    if (a.x_inner < 0 || (a.x_inner > 1 && a.rows % a.x_inner != 0)) {
        return KDA_ERR_INVALID_ARGUMENT;
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
