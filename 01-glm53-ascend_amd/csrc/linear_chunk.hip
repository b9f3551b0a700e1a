// linear_chunk.hip -- linear attention with a decay for each head, in chunks of 64 tokens, gfx950.
//
// With G_i the sum of the chunk's log decays up to token i and S the state before it,
//
//   out_i = scale (e^{G_i} S^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j)
//   S    <- e^{G_64} S + sum_j k_j (e^{G_64 - G_j} v_j)^T
//
// A request is cut into segments of L tokens, which go to workgroups at once:
//
//   sums_kernel     every segment but a request's last: its own sum of k_j v_j^T, from zero
//   starts_kernel   from them, elementwise and in order, the state before each segment
//   outputs_kernel  every segment from its state: outputs, tracked prefixes, final state
//
// (a request of one segment needs the last only). L goes by the call's tokens and heads, so that two
// workgroups a CU have work whatever the number of heads is.
//
// A wave owns 16 or 32 of the state's columns (values) and keeps them as accumulators, in fp32, through its segment:
// as they lie there they are, split into bf16 parts, the left operand of S^T q. The values, read transposed from
// LDS, serve both the outputs (left operand) and the update (right operand, times their decays). The
// scores of 16 tokens are formed by each wave for all of them. q, k and v are exact in bf16; what is rounded
// is split: scores and S into two parts (17 bits), the decayed values into three (25 bits, all of fp32: these errors
// would stay in the state). The sums of log decays are formed in 64 bits, so that neighbours' differences are exact
// behind a steep decay.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kda_abi.h"
#include "kda_device.h"
#include "linear_device.h"
#include "matrix_device.h"

namespace kda {
namespace {

#define KDA_INLINE __attribute__((always_inline))

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kChunk = 64;
constexpr double kLog2e = 1.4426950408889634;
constexpr float kSteepest = -1e4f;  // of a log decay: its exponential is 0 long before

struct ChunkParams : LinearParams {
    float *starts;  // [slots][heads][D * D]: a segment's sum, then the state before it
    float *decays;  // [slots][heads]: of a whole segment
    int segment;    // tokens, a multiple of 64
};

// A workgroup's segment of a request.
struct Segment {
    int n, index, count;
    int request_begin, begin, end;
    int64_t slot;  // in the workspace, for requests of several segments
};

// Segment number `tile` of all: request n gets the numbers from floor(cu[n] / L) + n, at least as many as it has
// segments. By a whole workgroup; n < 0: none.
__device__ __forceinline__ Segment segment_of(const ChunkParams &a, int tile) {
    Segment s;
    int below = 0;  // requests that begin at or before this tile
    for (int first = 0; first < a.num_seqs; first += kThreads) {
        const int x = first + static_cast<int>(threadIdx.x);
        below += __syncthreads_count(x < a.num_seqs && a.cu(x) / a.segment + x <= tile);
    }
    s.n = __builtin_amdgcn_readfirstlane(below) - 1;
    if (s.n < 0) {
        return s;
    }
    s.request_begin = a.cu(s.n);
    const int end = max(a.cu(s.n + 1), s.request_begin);
    s.index = tile - s.request_begin / a.segment - s.n;
    s.count = max((end - s.request_begin + a.segment - 1) / a.segment, 1);
    if (s.index < 0 || s.index >= s.count) {
        s.n = -1;
        return s;
    }
    s.begin = s.request_begin + s.index * a.segment;
    s.end = min(end, s.begin + a.segment);
    // len > L: ceil(len / L) <= floor(2 (begin + len) / L) - floor(2 begin / L)
    s.slot = 2 * static_cast<int64_t>(s.request_begin) / a.segment + s.index;
    return s;
}

// Rows of 64 tokens in LDS, without padding: chunks of 16 bytes permuted within 256 bytes by the row, so that
// neither reads of one column over 16 rows nor transposing reads of 32 bytes of 8 rows meet in a bank.
template <int D> __device__ __forceinline__ int place(int row, int chunk) {
    const int f = D == 128 ? (row & 7) << 1 | (row >> 3 & 1) : (row >> 1 & 3) << 1 | (row >> 3 & 1);
    return row * 2 * D + ((chunk ^ f) << 4);
}

// Eight values of one column, tokens 4 g .. and 16 + 4 g .. of the 32 from `row`: transposed.
template <int D> __device__ __forceinline__ u32x4 column(const char *tile, int row, int col16, int lane) {
    const int r = row + 4 * (lane >> 4) + (lane >> 2 & 3), c = lane & 3;
    const u32x2 lo = lds_read_tr(tile + place<D>(r, 2 * col16 + (c >> 1)) + (c & 1) * 8);
    const u32x2 hi = lds_read_tr(tile + place<D>(r + 16, 2 * col16 + (c >> 1)) + (c & 1) * 8);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

__device__ __forceinline__ float low_bf16(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float high_bf16(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// x = hi + lo + rest, hi and lo in bf16
__device__ __forceinline__ uint32_t split(float &x, float &y) {
    const uint32_t hi = pack_bf16x2(x, y);
    x -= low_bf16(hi);
    y -= high_bf16(hi);
    return hi;
}

template <int D, bool OUTPUTS> struct Shared {
    char k[kChunk * D * 2];
    char v[kChunk * D * 2];
    char q[OUTPUTS ? kChunk * D * 2 : 16];
    u32x4 scores[OUTPUTS ? 4 : 1][2][2][64];  // [16 tokens][32 earlier ones][part][lane]
    double sum[kChunk];                       // G in log2 units
    float late[kChunk];                       // e^(G_64 - G_j)
    float early[kChunk];                      // e^G_i
    int odd[kWaves];                          // some value is not finite
};

// Tokens [segment.begin, segment.end) of one head, from the state in s (accumulators: columns 16 (wave VT + vt) + lane % 16,
// rows 16 kt + 4 (lane / 16) + e). Returns the sum of the log decays (log2).
template <int D, bool OUTPUTS>
__device__ __forceinline__ double walk(const ChunkParams &a, Shared<D, OUTPUTS> &sm, const Segment &seg, int head,
                                       f32x4 (&s)[D / 16][D / 64], int64_t track_slot, int64_t track_at) {
    constexpr int VT = D / 64, KT = D / 16, X = D / 32;
    constexpr int kRowChunks = D / 8;
    constexpr int kLoads = D / 32;  // 16-byte loads a thread makes of 64 rows
    constexpr int kStep = kThreads / kRowChunks;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, col = lane & 15;
    const int row = tid / kRowChunks, chunk = tid % kRowChunks;
    const char *qb = static_cast<const char *>(a.q) + 2 * (head * a.q_stride_head) + chunk * 16;
    const char *kb = static_cast<const char *>(a.k) + 2 * (head * a.k_stride_head) + chunk * 16;
    const char *vb = static_cast<const char *>(a.v) + 2 * (head * a.v_stride_head) + chunk * 16;
    u32x4 q[OUTPUTS ? kLoads : 1], k[kLoads], v[kLoads];
    float decay = 0.0f;
    double total = 0.0;

    auto load = [&](int pos, int len) KDA_INLINE {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int64_t t = pos + min(row + i * kStep, len - 1);
            if constexpr (OUTPUTS) {
                q[i] = *reinterpret_cast<const u32x4 *>(qb + 2 * t * a.q_stride_token);
            }
            k[i] = *reinterpret_cast<const u32x4 *>(kb + 2 * t * a.k_stride_token);
            v[i] = *reinterpret_cast<const u32x4 *>(vb + 2 * t * a.v_stride_token);
        }
        decay = a.g[(pos + min(lane, len - 1)) * a.g_stride_token + head * a.g_stride_head];
    };
    int single = 0;  // tokens before this one go one at a time
    auto length = [&](int pos) KDA_INLINE -> int {
        const int len = pos < single ? 1 : min(kChunk, seg.end - pos);
        return track_at > pos && track_at < pos + len ? static_cast<int>(track_at) - pos : len;
    };

    int pos = seg.begin, len = length(pos);
    if (pos < seg.end) {
        load(pos, len);
    }
    while (pos < seg.end) {
        // ---- the chunk into LDS, its sums of decays
        uint32_t odd = 0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = row + i * kStep;
            if (r >= len) {
                k[i] = v[i] = u32x4{0, 0, 0, 0};
            }
            *reinterpret_cast<u32x4 *>(sm.k + place<D>(r, chunk)) = k[i];
            *reinterpret_cast<u32x4 *>(sm.v + place<D>(r, chunk)) = v[i];
            if constexpr (OUTPUTS) {
                if (r >= len) {
                    q[i] = u32x4{0, 0, 0, 0};
                }
                // elements 4 u .. 4 u + 3 of each 32 go to place (u % 4, u / 4): a lane's eight of the
                // contraction, 4 g .. and 16 + 4 g .., are then one read
                const int c = chunk & ~3, u = 2 * (chunk & 3);
                *reinterpret_cast<u32x2 *>(sm.q + place<D>(r, c + (u & 3)) + (u >> 2) * 8) = u32x2{q[i][0], q[i][1]};
                *reinterpret_cast<u32x2 *>(sm.q + place<D>(r, c + (u & 3) + 1) + (u >> 2) * 8) = u32x2{q[i][2], q[i][3]};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    odd |= ((v[i][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                }
            }
        }
        if (wave == 0) {
            double sum = lane < len ? static_cast<double>(decay < kSteepest ? kSteepest : decay) : 0.0;
            sum *= kLog2e;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double up = __shfl_up(sum, d);
                sum += lane >= d ? up : 0.0;
            }
            sm.sum[lane] = sum;
            sm.late[lane] = ex2(static_cast<float>(__shfl(sum, 63) - sum));
            sm.early[lane] = ex2(static_cast<float>(sum));
        }
        if constexpr (OUTPUTS) {
            const unsigned long long some = __ballot(odd != 0);
            if (lane == 0) {
                sm.odd[wave] = some != 0;
            }
        }
        lds_barrier();
        if constexpr (OUTPUTS) {
            // An infinite or NaN value must not reach earlier tokens of its chunk, but in the product their score of 0
            // makes a NaN of it: such a chunk goes token by token.
            if (len > 1 && (sm.odd[0] | sm.odd[1] | sm.odd[2] | sm.odd[3]) != 0) {
                single = pos + len;
                len = 1;
                load(pos, len);
                lds_barrier();
                continue;
            }
        }
        const int next = pos + len, next_len = length(next);
        if (next < seg.end) {
            load(next, next_len);
        }
        total += sm.sum[63];
        const float all = ex2(static_cast<float>(sm.sum[63]));

        f32x4 o[VT][4];
        u32x4 values[VT][2];
        if constexpr (OUTPUTS) {
            // ---- scores of this wave's 16 tokens with those before them: lane: token 16 wave + col, earlier 16 jt + 4 g + e
            f32x4 p[4];
            const double mine = sm.sum[16 * wave + col];
#pragma unroll
            for (int jt = 0; jt < 4; ++jt) {
                p[jt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (jt > wave) {
                    continue;
                }
#pragma unroll
                for (int x = 0; x < X; ++x) {
                    const char *kr = sm.k + (g & 1) * 8;
                    const int r = 16 * jt + col;
                    const u32x2 k0 = *reinterpret_cast<const u32x2 *>(kr + place<D>(r, 4 * x + (g >> 1)));
                    const u32x2 k1 = *reinterpret_cast<const u32x2 *>(kr + place<D>(r, 4 * x + 2 + (g >> 1)));
                    const u32x4 qx = *reinterpret_cast<const u32x4 *>(sm.q + place<D>(16 * wave + col, 4 * x + g));
                    p[jt] = mfma16(u32x4{k0[0], k0[1], k1[0], k1[1]}, qx, p[jt]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = 16 * jt + 4 * g + e;
                    const float w = ex2(static_cast<float>(mine - sm.sum[j]));
                    p[jt][e] = j <= 16 * wave + col ? p[jt][e] * w : 0.0f;
                }
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (2 * y > wave) {
                    continue;
                }
                u32x4 part;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f32x4 &two = p[2 * y + (e >> 1)];
                        float p0 = two[2 * (e & 1)], p1 = two[2 * (e & 1) + 1];
                        part[e] = split(p0, p1);
                        two[2 * (e & 1)] = p0;
                        two[2 * (e & 1) + 1] = p1;
                    }
                    sm.scores[wave][y][z][lane] = part;
                }
            }
            // ---- what the state gives, for all 64 tokens: rows 16 (wave VT + vt) + 4 g + e, token 16 it + col
#pragma unroll
            for (int it = 0; it < 4; ++it) {
#pragma unroll
                for (int vt = 0; vt < VT; ++vt) {
                    o[vt][it] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
#pragma unroll
            for (int x = 0; x < X; ++x) {
                u32x4 hi[VT], lo[VT];
#pragma unroll
                for (int vt = 0; vt < VT; ++vt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float s0 = s[2 * x + (e >> 1)][vt][2 * (e & 1)], s1 = s[2 * x + (e >> 1)][vt][2 * (e & 1) + 1];
                        hi[vt][e] = split(s0, s1);
                        lo[vt][e] = pack_bf16x2(s0, s1);
                    }
                }
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const u32x4 qx = *reinterpret_cast<const u32x4 *>(sm.q + place<D>(16 * it + col, 4 * x + g));
#pragma unroll
                    for (int vt = 0; vt < VT; ++vt) {
                        o[vt][it] = mfma16(hi[vt], qx, o[vt][it]);
                        o[vt][it] = mfma16(lo[vt], qx, o[vt][it]);
                    }
                }
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const float f = sm.early[16 * it + col];
#pragma unroll
                for (int vt = 0; vt < VT; ++vt) {
                    o[vt][it] *= f;
                }
            }
        }
#pragma unroll
        for (int vt = 0; vt < VT; ++vt) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                values[vt][y] = column<D>(sm.v, 32 * y, wave * VT + vt, lane);
            }
        }
        if constexpr (OUTPUTS) {
            lds_barrier();  // all scores are there
#pragma unroll
            for (int it = 0; it < 4; ++it) {
#pragma unroll
                for (int y = 0; y <= it / 2; ++y) {
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const u32x4 part = sm.scores[it][y][z][lane];
#pragma unroll
                        for (int vt = 0; vt < VT; ++vt) {
                            o[vt][it] = mfma16(values[vt][y], part, o[vt][it]);
                        }
                    }
                }
                const int i = 16 * it + col;
                if (i < len) {
                    uint16_t *to = static_cast<uint16_t *>(a.out) +
                                   (static_cast<int64_t>(pos + i) * a.num_heads + head) * D + 16 * wave * VT + 4 * g;
#pragma unroll
                    for (int vt = 0; vt < VT; ++vt) {
                        const f32x4 y = o[vt][it] * a.scale;
                        *reinterpret_cast<u32x2 *>(to + 16 * vt) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
                    }
                }
            }
        }
        // ---- the state
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
            for (int vt = 0; vt < VT; ++vt) {
                s[kt][vt] *= all;
            }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            u32x4 part[VT][3];
            const f32x4 w0 = *reinterpret_cast<const f32x4 *>(sm.late + 32 * y + 4 * g);
            const f32x4 w1 = *reinterpret_cast<const f32x4 *>(sm.late + 32 * y + 16 + 4 * g);
#pragma unroll
            for (int vt = 0; vt < VT; ++vt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t pair = values[vt][y][e];
                    float x0 = low_bf16(pair) * (e < 2 ? w0[2 * e] : w1[2 * e - 4]);
                    float x1 = high_bf16(pair) * (e < 2 ? w0[2 * e + 1] : w1[2 * e - 3]);
                    part[vt][0][e] = split(x0, x1);
                    part[vt][1][e] = split(x0, x1);
                    part[vt][2][e] = pack_bf16x2(x0, x1);
                }
            }
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const u32x4 keys = column<D>(sm.k, 32 * y, kt, lane);
#pragma unroll
                for (int vt = 0; vt < VT; ++vt) {
#pragma unroll
                    for (int z = 2; z >= 0; --z) {
                        s[kt][vt] = mfma16(keys, part[vt][z], s[kt][vt]);
                    }
                }
            }
        }
        if constexpr (OUTPUTS) {
            if (next == track_at) {
                float *to = a.pool(track_slot, head) + (16 * wave * VT + col) * D + 4 * g;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                    for (int vt = 0; vt < VT; ++vt) {
                        *reinterpret_cast<f32x4 *>(to + 16 * vt * D + 16 * kt) = s[kt][vt];
                    }
                }
            }
        }
        pos = next;
        len = next_len;
        lds_barrier();  // before the next chunk is staged over this one
    }
    return total;
}

template <int D> __global__ __launch_bounds__(kThreads, 2) void sums_kernel(const ChunkParams a) {
    __shared__ __attribute__((aligned(16))) Shared<D, false> sm;
    const int head = blockIdx.x % a.num_heads;
    const Segment seg = segment_of(a, blockIdx.x / a.num_heads);
    if (seg.n < 0 || seg.index + 1 >= seg.count) {
        return;
    }
    f32x4 s[D / 16][D / 64];
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
#pragma unroll
        for (int vt = 0; vt < D / 64; ++vt) {
            s[kt][vt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    const double total = walk<D, false>(a, sm, seg, head, s, 0, -1);
    const int64_t at = seg.slot * a.num_heads + head;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *to = a.starts + at * (D * D) + (16 * wave * (D / 64) + (lane & 15)) * D + 4 * (lane >> 4);
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
#pragma unroll
        for (int vt = 0; vt < D / 64; ++vt) {
            *reinterpret_cast<f32x4 *>(to + 16 * vt * D + 16 * kt) = s[kt][vt];
        }
    }
    if (threadIdx.x == 0) {
        a.decays[at] = ex2(static_cast<float>(total));
    }
}

// A thread takes four elements of a state at a time through all of the request's segments.
template <int D> __global__ __launch_bounds__(kThreads) void starts_kernel(const ChunkParams a, int parts) {
    const int part = blockIdx.x % parts;
    const int pair = blockIdx.x / parts;
    const int n = pair / a.num_heads, head = pair - n * a.num_heads;
    const int begin = a.cu(n), end = max(a.cu(n + 1), begin);
    const int count = (end - begin + a.segment - 1) / a.segment;
    if (count < 2) {
        return;
    }
    const int64_t slot = a.slot(n), first = 2 * static_cast<int64_t>(begin) / a.segment;
    for (int e = (part * kThreads + threadIdx.x) * 4; e < D * D; e += parts * kThreads * 4) {
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (slot > 0) {
            s = *reinterpret_cast<const f32x4 *>(a.pool(slot, head) + e);
        }
        constexpr int kAtOnce = 8;
        for (int i = 0; i < count; i += kAtOnce) {
            f32x4 sum[kAtOnce];
            float decay[kAtOnce];
#pragma unroll
            for (int x = 0; x < kAtOnce; ++x) {
                const int64_t at = (first + min(i + x, count - 2)) * a.num_heads + head;
                sum[x] = *reinterpret_cast<const f32x4 *>(a.starts + at * (D * D) + e);
                decay[x] = a.decays[at];
            }
#pragma unroll
            for (int x = 0; x < kAtOnce; ++x) {
                if (i + x < count) {
                    *reinterpret_cast<f32x4 *>(a.starts + ((first + i + x) * a.num_heads + head) * (D * D) + e) = s;
                    s = s * decay[x] + sum[x];
                }
            }
        }
    }
}

template <int D> __global__ __launch_bounds__(kThreads, 2) void outputs_kernel(const ChunkParams a) {
    __shared__ __attribute__((aligned(16))) Shared<D, true> sm;
    linear_zero_uncovered<D, uint16_t>(a, blockIdx.x, gridDim.x);
    const int head = blockIdx.x % a.num_heads;
    const Segment seg = segment_of(a, blockIdx.x / a.num_heads);
    if (seg.n < 0) {
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = (16 * wave * (D / 64) + (lane & 15)) * D + 4 * (lane >> 4);
    const int64_t slot = a.slot(seg.n);
    f32x4 s[D / 16][D / 64];
    const float *from = seg.count > 1 ? a.starts + (seg.slot * a.num_heads + head) * (D * D) : slot > 0 ? a.pool(slot, head) : nullptr;
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
#pragma unroll
        for (int vt = 0; vt < D / 64; ++vt) {
            s[kt][vt] = from == nullptr ? f32x4{0.0f, 0.0f, 0.0f, 0.0f}
                                        : *reinterpret_cast<const f32x4 *>(from + at + 16 * vt * D + 16 * kt);
        }
    }
    auto store = [&](int64_t to_slot) KDA_INLINE {
        float *to = a.pool(to_slot, head) + at;
#pragma unroll
        for (int kt = 0; kt < D / 16; ++kt) {
#pragma unroll
            for (int vt = 0; vt < D / 64; ++vt) {
                *reinterpret_cast<f32x4 *>(to + 16 * vt * D + 16 * kt) = s[kt][vt];
            }
        }
    };
    const int64_t track_slot = a.track_slot(seg.n);
    const int64_t track_len = track_slot > 0 ? a.track_len(seg.n) : -1;
    if (track_len == 0 && seg.index == 0) {
        store(track_slot);
    }
    walk<D, true>(a, sm, seg, head, s, track_slot, track_len > 0 ? seg.request_begin + track_len : -1);
    if (slot > 0 && seg.index + 1 == seg.count && seg.begin < seg.end) {
        store(slot);
    }
}

// Two workgroups a CU where all segments are whole.
int segment_of_call(const KdaLinearArgs &a) {
    const int64_t per = (static_cast<int64_t>(a.num_tokens) * a.num_heads + 511) / 512;
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>((per + kChunk - 1) / kChunk, 2), 1 << 20) * kChunk);
}

struct Plan {
    int segment;
    int64_t slots;
    size_t decays_at, bytes;
};

Plan plan_of(const KdaLinearArgs &a) {
    Plan p{segment_of_call(a), 0, 0, 0};
    if (a.num_tokens > p.segment) {
        p.slots = 2 * static_cast<int64_t>(a.num_tokens) / p.segment + 1;
        const size_t states = static_cast<size_t>(p.slots) * a.num_heads;
        p.decays_at = states * a.head_dim * a.head_dim * 4;
        p.bytes = (p.decays_at + states * 4 + 255) & ~size_t{255};
    }
    return p;
}

template <int D> int launch(const ChunkParams &a, const Plan &p, hipStream_t s) {
    const int64_t blocks = (static_cast<int64_t>(a.num_tokens) / a.segment + a.num_seqs) * a.num_heads;
    if (blocks > (INT64_C(1) << 24) - 1) {  // a grid counts its threads in 32 bits
        return KDA_ERR_TOO_LARGE;
    }
    if (p.slots > 0) {
        sums_kernel<D><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a);
        const int64_t pairs = static_cast<int64_t>(a.num_seqs) * a.num_heads;
        const int parts = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1024 / pairs, 1), D * D / (4 * kThreads)));
        starts_kernel<D><<<static_cast<unsigned>(pairs * parts), kThreads, 0, s>>>(a, parts);
    }
    outputs_kernel<D><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a);
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}

}  // namespace
}  // namespace kda

extern "C" size_t kda_linear_chunk_workspace_bytes(const KdaLinearArgs *args) {
    using namespace kda;
    if (args == nullptr || check_linear_sizes(*args) != KDA_OK || args->num_seqs == 0) {
        return 0;
    }
    return plan_of(*args).bytes;
}

extern "C" int kda_linear_chunk_launch(const KdaLinearArgs *args, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace kda;
    if (args == nullptr) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    if (const int rc = check_linear(*args); rc != KDA_OK) {
        return rc;
    }
    if (args->dtype != KDA_BF16 || args->intermediate != nullptr) {
        return KDA_ERR_UNSUPPORTED;
    }
    if (args->num_seqs == 0) {
        return args->num_tokens == 0 ? KDA_OK : KDA_ERR_INVALID_ARGUMENT;
    }
    const Plan p = plan_of(*args);
    if (p.bytes > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || workspace_bytes < p.bytes)) {
        return KDA_ERR_WORKSPACE;
    }
    char *ws = static_cast<char *>(workspace);
    const ChunkParams a{{*args}, reinterpret_cast<float *>(ws), reinterpret_cast<float *>(ws + p.decays_at), p.segment};
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    return a.head_dim == 128 ? launch<128>(a, p, s) : launch<64>(a, p, s);
}
