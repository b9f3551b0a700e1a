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
// A wave owns 16 of the state's columns (values) and keeps them as accumulators, in fp32, through its segment:
// as they lie there they are, split into bf16 parts, the left operand of S^T q. The values, read transposed from
// LDS, serve both the outputs (left operand) and the update (right operand, times their decays). The
// scores are formed once, by all waves for all, and go through LDS. q, k and v are exact in bf16; what is rounded
// is split: scores and S into two parts (17 bits), the decayed values into three (25 bits, all of fp32: these errors
// would stay in the state; two would do for 121 us instead of 129). The sums of log decays are formed in 64 bits, so that
// neighbours' differences are exact behind a steep decay.
//
// Bound by the issue of instructions, which splitting costs (each one taken out of outputs_kernel was worth its share; vector ones
// take 49% of the SIMDs' cycles, matrix ones 30%, partly at once), and by HBM wherever all workgroups load at once. One MI355X,
// by card: 8192 tokens of 32 heads of 128 in 126 to 138 us; 16001 of 4 heads in 53 us, of which a chunk is 6 us of latency;
// 37 ragged requests of up to 2000, 16 heads of 64, in 141 to 155 us. Kernels traced one by one, which start and end apart and so
// take longer together: sums 37, starts 15, outputs 87 us (4.6, 4.6 and 3.5 TB/s); 15, 11.5, 31; 31, 12, 105.

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

constexpr int kChunk = 64;
template <int D> constexpr int kWaves = D / 16;
template <int D> constexpr int kThreads = 64 * kWaves<D>;
constexpr int kStartThreads = 64;
constexpr int kWaitMemory = 0x0070;  // s_waitcnt vmcnt(0) lgkmcnt(0)
constexpr double kLog2e = 1.4426950408889634;
constexpr float kSteepest = -1e4f;  // of a log decay: its exponential is 0 long before

struct ChunkParams : LinearParams {
    float *starts;  // [slots][heads][D * D]: a segment's sum, then the state before it
    float *decays;  // [slots][heads]: of a whole segment, see kept_decay
    int segment;    // tokens, a multiple of 64
};

__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<int>(x));
    return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32))) << 32 | low;
}

// A workgroup's segment of a request.
struct Segment {
    int n, index, count;
    int request_begin, begin, end;
    int64_t slot;  // in the workspace, for requests of several segments
};

// A workgroup's segment, by all its threads; n < 0: none. The numbers up to tokens / L are those of segments that
// others of their request follow: request n has those from floor(cu[n] / L), at least as many as it needs. Then one
// for each request: its last segment. Long ones so go first.
template <int THREADS> __device__ __forceinline__ Segment segment_of(const ChunkParams &a, int tile) {
    const int whole = a.num_tokens / a.segment;
    Segment s;
    s.n = tile - whole;
    if (tile < whole) {
        int below = 0;  // requests that begin at or before this tile
        for (int first = 0; first < a.num_seqs; first += THREADS) {
            const int x = first + static_cast<int>(threadIdx.x);
            below += __syncthreads_count(x < a.num_seqs && a.cu(x) / a.segment <= tile);
        }
        s.n = __builtin_amdgcn_readfirstlane(below) - 1;
        if (s.n < 0) {
            return s;
        }
    }
    s.request_begin = __builtin_amdgcn_readfirstlane(a.cu(s.n));
    const int end = __builtin_amdgcn_readfirstlane(max(a.cu(s.n + 1), s.request_begin));
    s.count = max((end - s.request_begin + a.segment - 1) / a.segment, 1);
    s.index = tile < whole ? tile - s.request_begin / a.segment : s.count - 1;
    if (tile < whole && (s.index < 0 || s.index + 1 >= s.count)) {
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

// x + the sum of a pair times two constants
__device__ __forceinline__ float dot(uint32_t pair, uint32_t constants, float x) {
    asm("" : "+s"(constants));  // (0x0000bf80 itself would be encoded as the inline -1.0, whose halves are others here)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, constants), x, false);
}
// x = hi + lo + rest, hi and lo in bf16. What is not finite spreads within the pair: two keys' parts or tokens of one
// column, where it spoils the sums of both.
__device__ __forceinline__ uint32_t split(float &x, float &y) {
    const uint32_t hi = pack_bf16x2(x, y);
    x = dot(hi, 0x0000bf80u, x);  // x - hi's lower, exact
    y = dot(hi, 0xbf800000u, y);
    return hi;
}

// Number of the scores of tokens 16 it .. with 32 y ..: those that can see any of them.
__device__ __forceinline__ constexpr int unit(int it, int y) { return it < 2 ? it : 2 * it - 2 + y; }

template <int D, bool OUTPUTS> struct Shared {
    char k[kChunk * D * 2];
    char v[kChunk * D * 2];
    char q[OUTPUTS ? kChunk * D * 2 : 16];
    u32x4 scores[OUTPUTS ? 6 : 1][2][64];  // [16 tokens and 32 up to them: unit()][part][lane]
    double sum[kChunk];                       // G in log2 units
    float late[kChunk];                       // e^(G_64 - G_j)
    float early[kChunk];                      // scale e^G_i
    int odd[kWaves<D>];                       // some value is not finite
};

// The lane, and what follows from it formed anew: kept from chunk to chunk, addresses in LDS do not all fit the registers.
__device__ __forceinline__ int lane_here() {
    int lane = static_cast<int>(__lane_id());
    asm volatile("" : "+v"(lane));
    return lane;
}

// A sum of the values of this lane and those before it, over the wave.
template <int CTRL, int ROWS> __device__ __forceinline__ double add_from(double x) {
    const u32x2 w = __builtin_bit_cast(u32x2, x);
    const u32x2 up = {static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w[0]), CTRL, ROWS, 0xf, false)),
                      static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(w[1]), CTRL, ROWS, 0xf, false))};
    return x + __builtin_bit_cast(double, up);
}
__device__ __forceinline__ double prefix_sum(double x) {
    x = add_from<0x111, 0xf>(x);  // one lane up within 16, then two, four and eight
    x = add_from<0x112, 0xf>(x);
    x = add_from<0x114, 0xf>(x);
    x = add_from<0x118, 0xf>(x);
    x = add_from<0x142, 0xa>(x);  // lane 15 to the second 16, lane 47 to the fourth
    return add_from<0x143, 0xc>(x);  // lane 31 to the upper half
}

// Tokens [segment.begin, segment.end) of one head, from the state in s (accumulators: column 16 wave + lane % 16, rows
// 16 kt + 4 (lane / 16) + e). Returns the sum of the log decays (log2).
//
// Two barriers a chunk: its rows are in LDS, and nobody reads them any more (the scores are there). What
// comes after the second one, the scores' products with the values held in registers, overlaps with other waves'
// staging of the next chunk, whose loads are in flight all the while.
template <int D, bool OUTPUTS>
__device__ __forceinline__ double walk(const ChunkParams &a, Shared<D, OUTPUTS> &sm, const Segment &seg, int head,
                                       f32x4 (&s)[D / 16], int64_t track_slot, int track_at) {
    constexpr int KT = D / 16, X = D / 32;
    constexpr int kRowChunks = D / 8;
    constexpr int kStep = kThreads<D> / kRowChunks;
    constexpr int kLoads = kChunk / kStep;  // 16-byte loads a thread makes of 64 rows
    static_assert(kLoads == 2);
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = tid / kRowChunks, chunk = tid % kRowChunks;
    struct Rows {
        const char *at;  // this thread's 16 bytes of its first row of the next chunk
        int64_t token;   // bytes
    };
    auto rows_of = [&](const void *x, int64_t token, int64_t of_head) KDA_INLINE -> Rows {
        return Rows{static_cast<const char *>(x) + 2 * (head * of_head + (seg.begin + row) * token) + chunk * 16, 2 * token};
    };
    Rows qr = rows_of(a.q, a.q_stride_token, a.q_stride_head);
    Rows kr = rows_of(a.k, a.k_stride_token, a.k_stride_head);
    Rows vr = rows_of(a.v, a.v_stride_token, a.v_stride_head);
    u32x4 q[kLoads], k[kLoads], v[kLoads];
    float decay = 0.0f;
    double total = 0.0;

    // The next chunk's rows: len tokens, from the pointers on, which go on by as many. Their loads are spread over the
    // chunk before: issued at once by all workgroups, they keep the waves waiting for their issue.
    auto load_rows = [&](Rows &r, u32x4 (&x)[kLoads], int len) KDA_INLINE {
        const int row = (64 * wave + lane_here()) / kRowChunks;
        int64_t first = 0, second = kStep * r.token;
        if (len < kChunk) {  // rows past the last stand for it
            first = min(0, len - 1 - row) * r.token;
            second = min(kStep, len - 1 - row) * r.token;
        }
        x[0] = *reinterpret_cast<const u32x4 *>(r.at + first);
        x[1] = *reinterpret_cast<const u32x4 *>(r.at + second);
        r.at += len * r.token;
    };
    auto load_decay = [&](int pos, int len) KDA_INLINE {
        if (wave == 0) {
            decay = a.g[(pos + min(lane_here(), len - 1)) * a.g_stride_token + head * a.g_stride_head];
        }
    };
    auto load = [&](int pos, int len) KDA_INLINE {
        load_decay(pos, len);
        load_rows(kr, k, len);
        load_rows(vr, v, len);
        if constexpr (OUTPUTS) {
            load_rows(qr, q, len);
        }
    };
    int single = 0;  // tokens before this one go one at a time
    auto length = [&](int pos) KDA_INLINE -> int {
        const int len = pos < single ? 1 : min(kChunk, seg.end - pos);
        return track_at > pos && track_at < pos + len ? track_at - pos : len;
    };
    // A chunk's outputs are stored when the next one is in LDS, before the loads of the one after: whoever waits for
    // those then does not wait for stores that have only begun.
    u32x2 done[4];
    int done_len = 0, done_step = 0;
    const int64_t out_token = static_cast<int64_t>(a.num_heads) * D * 2;  // bytes
    char *out = static_cast<char *>(a.out) + (seg.begin + (tid & 15)) * out_token + 2 * (head * D + 16 * wave + 4 * (tid >> 4 & 3));
    auto store_done = [&]() KDA_INLINE {
        if constexpr (OUTPUTS) {
            const int col = lane_here() & 15;
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                if (16 * it + col < done_len) {
                    *reinterpret_cast<u32x2 *>(out + 16 * it * out_token) = done[it];
                }
            }
            out += done_step * out_token;
            done_len = done_step = 0;
        }
    };

    int pos = seg.begin, len = length(pos);
    if (pos < seg.end) {
        load(pos, len);
    }
    while (pos < seg.end) {
        const int lane = lane_here();
        const int g = lane >> 4, col = lane & 15;
        const int row = (64 * wave + lane) / kRowChunks, chunk = lane % kRowChunks;
        // ---- the chunk into LDS, its sums of decays
        float odd = 0.0f;  // 0 times this thread's values: NaN if one is not finite
        if (wave == 0) {
            const double sum = prefix_sum(lane < len ? kLog2e * static_cast<double>(decay < kSteepest ? kSteepest : decay) : 0.0);
            const u32x2 w = __builtin_bit_cast(u32x2, sum);
            const u32x2 last = {static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(w[0]), 63)),
                                static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(w[1]), 63))};
            sm.sum[lane] = sum;
            sm.late[lane] = ex2(static_cast<float>(__builtin_bit_cast(double, last) - sum));
            sm.early[lane] = ex2(static_cast<float>(sum)) * a.scale;
        }
        if (len < kChunk) {
            asm volatile("");  // stays a branch: selects would cost every chunk
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                if (row + i * kStep >= len) {
                    q[i] = k[i] = v[i] = u32x4{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = row + i * kStep;
            *reinterpret_cast<u32x4 *>(sm.k + place<D>(r, chunk)) = k[i];
            *reinterpret_cast<u32x4 *>(sm.v + place<D>(r, chunk)) = v[i];
            if constexpr (OUTPUTS) {
                // elements 4 u .. 4 u + 3 of each 32 go to place (u % 4, u / 4): a lane's eight of the
                // contraction, 4 g .. and 16 + 4 g .., are then one read
                const int c = chunk & ~3, u = 2 * (chunk & 3);
                *reinterpret_cast<u32x2 *>(sm.q + place<D>(r, c + (u & 3)) + (u >> 2) * 8) = u32x2{q[i][0], q[i][1]};
                *reinterpret_cast<u32x2 *>(sm.q + place<D>(r, c + (u & 3) + 1) + (u >> 2) * 8) = u32x2{q[i][2], q[i][3]};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    odd = dot(v[i][e], 0, odd);
                }
            }
        }
        if constexpr (OUTPUTS) {
            const bool some = __any(odd != odd);
            if (lane == 0) {
                sm.odd[wave] = some;
            }
        }
        lds_barrier();
        if constexpr (OUTPUTS) {
            // An infinite or NaN value must not reach earlier tokens of its chunk, but in the product their score of 0
            // makes a NaN of it: such a chunk goes token by token.
            if (len > 1 && __any(sm.odd[lane % kWaves<D>] != 0)) {
                single = pos + len;
                qr.at -= len * qr.token;
                kr.at -= len * kr.token;
                vr.at -= len * vr.token;
                len = 1;
                load(pos, 1);
                __builtin_amdgcn_s_waitcnt(kWaitMemory);  // or the compiler has everybody wait for loads where this path joins
                lds_barrier();
                continue;
            }
        }
        store_done();
        const int next = pos + len, next_len = length(next);
        const bool more = next < seg.end;
        if (more) {
            load_decay(next, next_len);
            load_rows(kr, k, next_len);
        }
        const double last = sm.sum[kChunk - 1];
        total += last;
        const float all = ex2(static_cast<float>(last));

        f32x4 o[4];
        u32x4 values[2];
        if constexpr (OUTPUTS) {
            // ---- scores of 16 tokens with 32 up to them: lane: token 16 it + col, earlier one 16 jt + 4 g + e
#pragma unroll
            for (int u = 0; u < 8 / kWaves<D>; ++u) {
                const int it = (wave * (8 / kWaves<D>) + u) >> 1, y = (wave * (8 / kWaves<D>) + u) & 1;
                if (y > it / 2) {
                    continue;
                }
                f32x4 p[2];
                const double mine = sm.sum[16 * it + col];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    p[z] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int x = 0; x < X; ++x) {
                    const u32x4 right = *reinterpret_cast<const u32x4 *>(sm.q + place<D>(16 * it + col, 4 * x + g));
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const char *at = sm.k + (g & 1) * 8;
                        const int r = 32 * y + 16 * z + col;
                        const u32x2 k0 = *reinterpret_cast<const u32x2 *>(at + place<D>(r, 4 * x + (g >> 1)));
                        const u32x2 k1 = *reinterpret_cast<const u32x2 *>(at + place<D>(r, 4 * x + 2 + (g >> 1)));
                        p[z] = mfma16(u32x4{k0[0], k0[1], k1[0], k1[1]}, right, p[z]);
                    }
                }
                u32x4 hi, lo;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 32 * y + 16 * z + 4 * g + e;
                        w[e] = p[z][e] * (a.scale * ex2(static_cast<float>(mine - sm.sum[j])));
                        asm volatile("" : "+v"(w[e]));  // formed in all lanes: no branch around it
                        w[e] = j <= 16 * it + col ? w[e] : 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        hi[2 * z + e] = split(w[2 * e], w[2 * e + 1]);
                        lo[2 * z + e] = pack_bf16x2(w[2 * e], w[2 * e + 1]);
                    }
                }
                sm.scores[unit(it, y)][0][lane] = hi;
                sm.scores[unit(it, y)][1][lane] = lo;
            }
            if (more) {
                load_rows(vr, v, next_len);
            }
            // ---- what the state gives, for all 64 tokens: rows 16 wave + 4 g + e, token 16 it + col
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                o[it] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int x = 0; x < X; ++x) {
                u32x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float s0 = s[2 * x + (e >> 1)][2 * (e & 1)], s1 = s[2 * x + (e >> 1)][2 * (e & 1) + 1];
                    hi[e] = split(s0, s1);
                    lo[e] = pack_bf16x2(s0, s1);
                }
#pragma unroll
                for (int it = 0; it < 4; it += 2) {
                    const u32x4 r0 = *reinterpret_cast<const u32x4 *>(sm.q + place<D>(16 * it + col, 4 * x + g));
                    const u32x4 r1 = *reinterpret_cast<const u32x4 *>(sm.q + place<D>(16 * it + 16 + col, 4 * x + g));
                    o[it] = mfma16(hi, r0, o[it]);
                    o[it + 1] = mfma16(hi, r1, o[it + 1]);
                    o[it] = mfma16(lo, r0, o[it]);
                    o[it + 1] = mfma16(lo, r1, o[it + 1]);
                }
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                o[it] *= sm.early[16 * it + col];
            }
        }
        if (more) {
            if constexpr (OUTPUTS) {
                load_rows(qr, q, next_len);
            } else {
                load_rows(vr, v, next_len);
            }
        }
        // ---- the state
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            s[kt] *= all;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            values[y] = column<D>(sm.v, 32 * y, wave, lane);
            u32x4 part[3];
            const f32x4 w0 = *reinterpret_cast<const f32x4 *>(sm.late + 32 * y + 4 * g);
            const f32x4 w1 = *reinterpret_cast<const f32x4 *>(sm.late + 32 * y + 16 + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t pair = values[y][e];
                float x0 = low_bf16(pair) * (e < 2 ? w0[2 * e] : w1[2 * e - 4]);
                float x1 = high_bf16(pair) * (e < 2 ? w0[2 * e + 1] : w1[2 * e - 3]);
                part[0][e] = split(x0, x1);
                part[1][e] = split(x0, x1);
                part[2][e] = pack_bf16x2(x0, x1);
            }
#pragma unroll
            for (int kt = 0; kt < KT; kt += 2) {
                u32x4 keys[2];
#pragma unroll
                for (int z = 2; z >= 0; --z) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (z == 2) {
                            keys[i] = column<D>(sm.k, 32 * y, kt + i, lane);
                        }
                        s[kt + i] = mfma16(keys[i], part[z], s[kt + i]);
                    }
                }
            }
        }
        lds_barrier();  // all scores are there, all reads of the chunk's rows are done
        if constexpr (OUTPUTS) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
#pragma unroll
                    for (int it = 2 * y; it < 4; ++it) {
                        o[it] = mfma16(values[y], sm.scores[unit(it, y)][z][lane], o[it]);
                    }
                }
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                done[it] = u32x2{pack_bf16x2(o[it][0], o[it][1]), pack_bf16x2(o[it][2], o[it][3])};
            }
            done_len = done_step = len;
            if (next == track_at) {
                float *to = a.pool(track_slot, head) + (16 * wave + col) * D + 4 * g;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    *reinterpret_cast<f32x4 *>(to + 16 * kt) = s[kt];
                }
            }
        }
        pos = next;
        len = next_len;
    }
    store_done();
    return total;
}

// A segment's decay from its log2, and its product with a state. Positive log decays may leave exp(sum) to fp32 over 64 tokens but
// not over a segment, where a state (one of 0 above all) may still leave a finite product: such a decay is kept as minus its log2.
__device__ __forceinline__ float kept_decay(double log2) {
    const float decay = ex2(static_cast<float>(log2));
    return decay < __builtin_inff() || !(log2 > 0.0) ? decay : -static_cast<float>(fmin(log2, 4096.0));
}
__device__ __forceinline__ f32x4 decayed(f32x4 s, float decay) {
    if (decay < 0.0f) {
        const float power = floorf(-decay);
        s *= ex2(-decay - power);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[e] = ldexpf(s[e], static_cast<int>(power));
        }
        return s;
    }
    return s * decay;
}

template <int D> __global__ __launch_bounds__(kThreads<D>, 4) void sums_kernel(const ChunkParams a) {
    __shared__ __attribute__((aligned(16))) Shared<D, false> sm;
    const int head = blockIdx.x % a.num_heads;
    const Segment seg = segment_of<kThreads<D>>(a, blockIdx.x / a.num_heads);
    if (seg.n < 0) {
        return;
    }
    f32x4 s[D / 16];
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
        s[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const double total = walk<D, false>(a, sm, seg, head, s, 0, -1);
    const int64_t at = seg.slot * a.num_heads + head;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *to = a.starts + at * (D * D) + (16 * wave + (lane & 15)) * D + 4 * (lane >> 4);
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
        *reinterpret_cast<f32x4 *>(to + 16 * kt) = s[kt];
    }
    if (threadIdx.x == 0) {
        a.decays[at] = kept_decay(total);
    }
}

// A thread takes four elements of a state at a time through all of the request's segments.
template <int D> __global__ __launch_bounds__(kStartThreads) void starts_kernel(const ChunkParams a, int parts) {
    const int part = blockIdx.x % parts;
    const int pair = blockIdx.x / parts;
    const int n = pair / a.num_heads, head = pair - n * a.num_heads;
    const int begin = __builtin_amdgcn_readfirstlane(a.cu(n)), end = max(a.cu(n + 1), begin);
    const int count = __builtin_amdgcn_readfirstlane((end - begin + a.segment - 1) / a.segment);
    if (count < 2) {
        return;
    }
    const int64_t slot = a.slot(n), first = 2 * static_cast<int64_t>(begin) / a.segment;
    for (int e = (part * kStartThreads + threadIdx.x) * 4; e < D * D; e += parts * kStartThreads * 4) {
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (slot > 0) {
            s = *reinterpret_cast<const f32x4 *>(a.pool(slot, head) + e);
        }
        constexpr int kAtOnce = 16;
        for (int i = 0; i < count; i += kAtOnce) {
            f32x4 sum[kAtOnce];
            float decay[kAtOnce];  // the last segment has neither
#pragma unroll
            for (int x = 0; x < kAtOnce; ++x) {
                if (i + x + 1 < count) {
                    const int64_t at = (first + i + x) * a.num_heads + head;
                    sum[x] = *reinterpret_cast<const f32x4 *>(a.starts + at * (D * D) + e);
                    decay[x] = a.decays[at];
                }
            }
            float least = 0.0f;
#pragma unroll
            for (int x = 0; x < kAtOnce; ++x) {
                least = i + x + 1 < count ? fminf(least, decay[x]) : least;
            }
            if (least < 0.0f) {  // one that fp32 does not hold: from memory again, one by one
                for (int x = i; x < min(i + kAtOnce, count); ++x) {
                    const int64_t at = (first + x) * a.num_heads + head;
                    float *to = a.starts + at * (D * D) + e;
                    f32x4 next = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (x + 1 < count) {
                        next = decayed(s, a.decays[at]) + *reinterpret_cast<const f32x4 *>(to);
                    }
                    *reinterpret_cast<f32x4 *>(to) = s;
                    s = next;
                }
                continue;
            }
#pragma unroll
            for (int x = 0; x < kAtOnce; ++x) {
                if (i + x < count) {
                    *reinterpret_cast<f32x4 *>(a.starts + ((first + i + x) * a.num_heads + head) * (D * D) + e) = s;
                }
                if (i + x + 1 < count) {
                    s = s * decay[x] + sum[x];
                }
            }
        }
    }
}

template <int D> __global__ __launch_bounds__(kThreads<D>, 4) void outputs_kernel(const ChunkParams a) {
    __shared__ __attribute__((aligned(16))) Shared<D, true> sm;
    linear_zero_uncovered<D, uint16_t, kThreads<D>>(a, blockIdx.x, gridDim.x);
    const int head = blockIdx.x % a.num_heads;
    const Segment seg = segment_of<kThreads<D>>(a, blockIdx.x / a.num_heads);
    if (seg.n < 0) {
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = (16 * wave + (lane & 15)) * D + 4 * (lane >> 4);
    const int64_t slot = uniform(a.slot(seg.n)), track_slot = uniform(a.track_slot(seg.n));
    const int64_t track_len = track_slot > 0 ? a.track_len(seg.n) : -1;
    f32x4 s[D / 16];
    const float *from = seg.count > 1 ? a.starts + (seg.slot * a.num_heads + head) * (D * D) : slot > 0 ? a.pool(slot, head) : nullptr;
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
        s[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (from != nullptr) {
#pragma unroll
        for (int kt = 0; kt < D / 16; ++kt) {
            s[kt] = *reinterpret_cast<const f32x4 *>(from + at + 16 * kt);
        }
    }
    auto store = [&](int64_t to_slot) KDA_INLINE {
        float *to = a.pool(to_slot, head) + at;
#pragma unroll
        for (int kt = 0; kt < D / 16; ++kt) {
            *reinterpret_cast<f32x4 *>(to + 16 * kt) = s[kt];
        }
    };
    if (track_len == 0 && seg.index == 0) {
        store(track_slot);
    }
    const bool here = track_len > seg.begin - seg.request_begin && track_len <= seg.end - seg.request_begin;
    walk<D, true>(a, sm, seg, head, s, track_slot,
                  __builtin_amdgcn_readfirstlane(here ? seg.request_begin + static_cast<int>(track_len) : -1));
    if (slot > 0 && seg.index + 1 == seg.count && seg.begin < seg.end) {
        store(slot);
    }
}

constexpr int kMostChunks = 1 << 20;  // of a segment
constexpr int kMostTokens = INT32_MAX - kMostChunks * kChunk;  // offsets a segment behind the last token stay in 32 bits

// A segment's tokens. As many workgroups as the card holds at once (of heads of 128, two a CU) where segments are then
// long, at least as many as it has CUs elsewhere; not so short that the states between
// them outweigh them, the less so the more requests and heads there are. Up to 320 tokens go as they are: 256 tokens
// on 16 heads 27.6 us so, 30.0 in segments of 128 (320: 32.9 and 29.7). us, heads of 128, with segments of 128, 192 and 256:
//   16001 tokens, 4 heads  62 65 55    5311, 16 heads  65 65 72    4096, 16  70 61 63    32768, 2  84 72 72
// Of heads of 64 a CU holds four (124 registers, 38 KB of LDS), 1024 in all; 1536 leaves the last ones to a second round, which costs
// single long requests, least where ragged ones fill it. us with work / 768, 1024, 1536 and 2048:
//   16001 tokens, 16 heads  69 71 80 89    8192, 32 heads  67 66 74 81    37 of 1 to 2000, 16 heads  161 152 154 155
//   8 of 2000 to 6000, 16 heads  125 119 123 121    100 of 100 to 1000, 8 heads  113 108 108 108
int segment_of_call(const KdaLinearArgs &a) {
    const int64_t work = static_cast<int64_t>(a.num_tokens) * a.num_heads;
    const int64_t pairs = static_cast<int64_t>(a.num_seqs) * a.num_heads;
    int64_t tokens = work / (a.head_dim == 128 ? 512 : 1536);
    if (a.head_dim == 128) {
        tokens = std::max<int64_t>(tokens, std::min<int64_t>(work / 256, 256));
    }
    tokens = std::max<int64_t>(tokens, a.num_tokens <= 320 ? 320 : std::min<int64_t>(std::max<int64_t>(pairs, 128), 512));
    return static_cast<int>(std::min<int64_t>((tokens + kChunk - 1) / kChunk, kMostChunks) * kChunk);
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
    const int64_t whole = static_cast<int64_t>(a.num_tokens) / a.segment * a.num_heads;
    const int64_t blocks = whole + static_cast<int64_t>(a.num_seqs) * a.num_heads;
    if (blocks * kThreads<D> > UINT32_MAX) {  // a grid counts its threads in 32 bits
        return KDA_ERR_TOO_LARGE;
    }
    if (p.slots > 0) {
        sums_kernel<D><<<static_cast<unsigned>(whole), kThreads<D>, 0, s>>>(a);
        const int64_t pairs = static_cast<int64_t>(a.num_seqs) * a.num_heads;
        const int parts = static_cast<int>(std::min<int64_t>(std::max<int64_t>(4096 / pairs, 1), D * D / (4 * kStartThreads)));
        starts_kernel<D><<<static_cast<unsigned>(pairs * parts), kStartThreads, 0, s>>>(a, parts);
    }
    outputs_kernel<D><<<static_cast<unsigned>(blocks), kThreads<D>, 0, s>>>(a);
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
    if (args->num_tokens > kMostTokens) {
        return KDA_ERR_TOO_LARGE;
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
