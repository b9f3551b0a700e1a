// sample.hip -- a token drawn from every row of logits, from given uniform numbers, gfx950.
//
// Weights w_i = e^{(l_i - max) / T}. Kept are the top_k largest (of equal ones those of the lowest index), of those
// the fewest first whose mass reaches top_p of theirs, of those the ones with w_i >= min_p. The token is the first
// in the vocabulary's order at which the kept mass so far exceeds u times the whole.
//
// Which side of such a border a token falls on decides the result, so masses are whole numbers: a weight is
// formed in 64-bit floats (a table of 2^{j / 256} and four terms, 1e-16) and rounded to a multiple of 2^-S, S as
// large as lets a row's sum stay below 2^62 (2^-44 for 150000 tokens). Sums of whole numbers do not depend on their
// order, so results do not depend on which atomic came first.
//
// A workgroup takes a row:
//   the maximum (and for T = 0 its first place, which is the answer);
//   few candidates (top_k up to kFewK): the k-th largest of the threads' maxima is a bound that at least k elements
//     reach, and hardly more do. Those go into LDS, are sorted, cut and drawn from there;
//   bf16: the few values that such logits have are counted, top_k and top_p cut in their table, and one pass looks the
//     weights up for the blocks' masses;
//   else one pass forms the weights, their mass in kBins bins by distance from the maximum, and each
//     block's mass. Where top_k or top_p cuts, the bin in which the border lies is gathered and sorted (bins of more
//     elements than fit are divided again by their keys, equal elements by their index), and blocks' masses
//     formed anew; the token's block is read once more.
//
// A row takes one CU, all of whose threads it has: the first pass is bound by what one CU can read, the later ones, which
// read the caches, by the vector instructions. Those of all passes, an element: 32 in bf16 (150000 with top_p and min_p), 59 in fp32
// with a temperature alone and 129 with top_p (32000, a fixed part included), where weights are formed one by one. One MI355X: a row
// of 131072 in bf16 with top_k 50 17 us, 256 rows of 150000 with top_p and min_p 52 us (257: 88 with top_p, a CU holds one
// workgroup), 37 rows of 32000 in fp32 18.5 us, of which 12 do not depend on the length (barriers, sorting, the launch).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kda_abi.h"
#include "kda_device.h"

namespace kda {
namespace {

#define KDA_INLINE __attribute__((always_inline))

constexpr int kThreads = 1024;
constexpr int kWaves = 16;
constexpr int kBins = 2048;
constexpr int kList = 1024;    // elements that are sorted, one a thread
constexpr int kFew = kList;    // elements that are drawn from in LDS
// top_k up to which candidates are looked for: with more, sorting them costs more than the bins do. us with them and without, top_k
// 64, 200, 320 and 400: one row of 131072 in bf16 20 34, 28 36, 38 37, 49 38 (with top_p too 20 39, 28 41, 38 41, 49 42); 256 rows of
// 32000 in fp32 18 31, 24 33, 35 34, 43 35 (18 49, 24 52, 35 53, 43 53). One number for all rows: short ones in bf16 take less
// without from 200 on (one row of 32000 15 23, 22 23, 31 23), long ones in fp32 with them for longer (131072: 22 53, 29 58, 40 63, 49 65).
constexpr int kFewK = 320;
constexpr int kMaxBlocks = 2048;
constexpr int kUnroll = 4;     // 16-byte loads of a lane in flight together
constexpr float kInf = __builtin_inff();
constexpr double kLog2e = 1.4426950408889634;
constexpr double kLn2 = 0.6931471805599453;

typedef uint64_t u64;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t s16x2 __attribute__((ext_vector_type(2)));

struct SampleParams : KdaSampleArgs {
    int shift;   // S: weights are multiples of 2^-S
    int groups;  // of kUnroll loads of a wave that make a block
};

// kPatterns: of bf16 logits, see Sampler
template <int kPatterns> struct __attribute__((aligned(16))) Shared {
    union {
        u64 bins[kBins + 1];
        uint32_t pattern_numbers[kPatterns + 5];
    };
    union {
        u64 list[kList];
        u64 pattern_weights[kPatterns + 3];
    };
    // Of the patterns' places 0 to kPatterns + 1, with those from 1 on at multiples of 16 bytes.
    __device__ __forceinline__ uint32_t *numbers() { return pattern_numbers + 3; }
    __device__ __forceinline__ u64 *table() { return pattern_weights + 1; }
    u64 blocks[kMaxBlocks];
    u64 weights[kFew];
    double powers[256];  // 2^{S + j / 256}
    u64 waves[kWaves];
    float tops[kWaves];
    int places[kWaves];
    int ranks[256];
    int count;
    uint32_t low, high;  // keys
    u64 before, found;
    uint32_t ties[kMaxBlocks];  // numbers of elements that equal the last one left
    u64 between;  // mass of the logits between the patterns of both signs
    uint32_t between_count;
};

// A larger float has the larger key; both zeros have one.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float((k >> 31) != 0 ? k ^ 0x80000000u : ~k);
}
// Elements in the order of their rank have falling numbers: by logit, then by index.
__device__ __forceinline__ u64 rank_of(uint32_t key, uint32_t index) { return static_cast<u64>(key) << 32 | (0xffffffffu - index); }
__device__ __forceinline__ uint32_t index_of(u64 rank) { return 0xffffffffu - static_cast<uint32_t>(rank); }

template <int CTRL, int ROWS> __device__ __forceinline__ u64 add_from(u64 x) {
    const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(x >> 32), CTRL, ROWS, 0xf, false);
    return x + (static_cast<u64>(high) << 32 | low);
}
// The sum of the values of this lane and those before it in the wave.
__device__ __forceinline__ u64 wave_scan(u64 x) {
    x = add_from<0x111, 0xf>(x);  // one lane up within 16, then two, four and eight
    x = add_from<0x112, 0xf>(x);
    x = add_from<0x114, 0xf>(x);
    x = add_from<0x118, 0xf>(x);
    x = add_from<0x142, 0xa>(x);  // lane 15 to the second 16, lane 47 to the fourth
    return add_from<0x143, 0xc>(x);  // lane 31 to the upper half
}
__device__ __forceinline__ u64 lane_of(u64 x, int lane) {
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(x), lane);
    return static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane))) << 32 | low;
}
__device__ __forceinline__ u64 last_lane(u64 x) { return lane_of(x, 63); }
// ... of this thread and those before it, and the sum of all. By all threads.
template <class S> __device__ __forceinline__ u64 block_scan(S &sm, u64 x, u64 &total) {
    const int lane = static_cast<int>(__lane_id()), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    x = wave_scan(x);
    __syncthreads();  // the last one's sums are read
    if (lane == 63) {
        sm.waves[wave] = x;
    }
    __syncthreads();
    u64 sums = lane < kWaves ? sm.waves[lane] : 0;
    sums = add_from<0x111, 0xf>(sums);
    sums = add_from<0x112, 0xf>(sums);
    sums = add_from<0x114, 0xf>(sums);
    sums = add_from<0x118, 0xf>(sums);
    total = lane_of(sums, kWaves - 1);
    return wave > 0 ? x + lane_of(sums, wave - 1) : x;
}

// The list's first n entries (all different, but for zeros) in falling order. By all threads. Up to 256 by counting what is
// larger, a quarter of the list a thread (60 entries 7000 cycles by steps of a sorting network, 1000 so); more by such a
// network, an element a thread, where steps within a wave go through its lanes.
template <class S> __device__ __forceinline__ void sort(S &sm, int n) {
    __syncthreads();
    const int i = threadIdx.x;
    if (n <= 256) {
        const int at = i & 255;
        const u64 mine = at < n ? sm.list[at] : 0;
        int larger = 0;
        const int per = (n + 3) / 4, first = (i >> 8) * per;
        for (int j = first; j < min(first + per, n); ++j) {
            larger += sm.list[j] > mine ? 1 : 0;
        }
        if (i < 256) {
            sm.ranks[i] = 0;
        }
        __syncthreads();
        atomicAdd(&sm.ranks[at], larger);
        __syncthreads();
        const bool real = i < n && mine != 0;
        const int rank = real ? sm.ranks[i] : 0;
        if (i < 256) {
            sm.list[i] = 0;
        }
        __syncthreads();
        if (real) {
            sm.list[rank] = mine;
        }
        __syncthreads();
        return;
    }
    const int size = 1 << (32 - __clz(n - 1));
    u64 x = i < n ? sm.list[i] : 0;
    for (int span = 2; span <= size; span <<= 1) {
        for (int step = span >> 1; step > 0; step >>= 1) {
            u64 y;
            if (step >= 64) {
                __syncthreads();
                sm.list[i] = x;
                __syncthreads();
                y = sm.list[i ^ step];
            } else if (__builtin_amdgcn_readfirstlane(i) >= size) {
                break;  // a wave behind the list
            } else {
                y = static_cast<u64>(__shfl_xor(static_cast<unsigned long long>(x), step));
            }
            const bool larger = ((i & step) == 0) == ((i & span) == 0);
            x = (x < y) == larger ? y : x;
        }
    }
    __syncthreads();
    sm.list[i] = x;
    __syncthreads();
}
// A row's logits. Comparisons are written such that NaN fails them: it counts as -infinity.
template <typename T> struct Row {
    static constexpr int E = 16 / sizeof(T);
    static constexpr int kGroup = 64 * E * kUnroll;  // elements that a wave loads at a time
    const T *at;
    int size;

    struct __attribute__((packed, aligned(sizeof(T)))) Raw {
        u32x4 w;
    };
    struct Group {
        u32x4 w[kUnroll];
    };
    // E logits from element `first`, beyond the row -infinity
    __device__ __forceinline__ u32x4 guarded(int64_t first) const {
        if (first + E <= size) {
            return reinterpret_cast<const Raw *>(at + first)->w;
        }
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = first + i < size ? __float_as_uint(at[first + i]) : 0xff800000u;
            } else {
                const uint32_t lo = first + 2 * i < size ? at[first + 2 * i] : 0xff80u;
                const uint32_t hi = first + 2 * i + 1 < size ? at[first + 2 * i + 1] : 0xff80u;
                w[i] = lo | hi << 16;
            }
        }
        return w;
    }
    static __device__ __forceinline__ float element(u32x4 w, int i) {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[i]);
        } else {
            return __uint_as_float((i & 1) != 0 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        }
    }
    __device__ __forceinline__ Group load(int64_t group) const {
        const int64_t begin = group * kGroup;
        const int lane = static_cast<int>(__lane_id()) * E;
        Group r;
        if (begin + kGroup <= size) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                r.w[u] = reinterpret_cast<const Raw *>(at + begin + u * 64 * E + lane)->w;
            }
        } else {
#pragma unroll 1
            for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
                for (int i = 0; i + 1 < kUnroll; ++i) {
                    r.w[i] = r.w[i + 1];
                }
                r.w[kUnroll - 1] = guarded(begin + u * 64 * E + lane);
            }
        }
        return r;
    }
    // f(index of the first, E logits) for the lane's loads of a group. A loop, the loads handed down in it: unrolled, the
    // passes' code would not fit the instruction cache.
    template <class F> __device__ __forceinline__ void each(int64_t group, Group r, F f) const {
        const int first = static_cast<int>(group * kGroup) + static_cast<int>(__lane_id()) * E;
#pragma unroll 1
        for (int u = 0; u < kUnroll; ++u) {
            f(first + u * 64 * E, r.w[0]);
#pragma unroll
            for (int i = 0; i + 1 < kUnroll; ++i) {
                r.w[i] = r.w[i + 1];
            }
        }
    }
};

// The least sum that reaches the part p of a whole, 1 at least.
__device__ __forceinline__ u64 reaching(double p, u64 whole) {
    const double x = ceil(p * static_cast<double>(whole));
    return x >= static_cast<double>(whole) ? whole : x > 1.0 ? static_cast<u64>(x) : 1;
}
// The least sum that exceeds the part u of a whole, the whole at most. (The 1 is added to a whole number: a double of this
// size has no room for it.)
__device__ __forceinline__ u64 exceeding(double u, u64 whole) {
    const double x = u * static_cast<double>(whole);
    return x >= static_cast<double>(whole) ? whole : min(static_cast<u64>(x) + 1, whole);
}

enum Mode { kNumbers, kNucleus, kLeft };

template <typename T, int kPatterns> struct Sampler {
    const SampleParams &a;
    Shared<kPatterns> &sm;
    Row<T> row;
    float top;            // the largest logit
    double scale;         // 256 log2(e) / temperature
    float bin_scale;
    float last;           // the last element in the order of the ranks that is not cut
    int last_index;
    double least_weight;  // min_p 2^S
    float floor;          // logits below it do not reach min_p (some others do not either)
    float least;          // logits below it are cut or do not reach min_p

    static constexpr int E = Row<T>::E;
    static constexpr u64 kBias = 0x4330000000000000ull;  // the bits of 2^52

    // 256 log2 of a weight
    __device__ __forceinline__ double exponent(float x) const { return (static_cast<double>(x) - static_cast<double>(top)) * scale; }
    // A weight times 2^S, not rounded; 0 where `in` does not hold.
    __device__ __forceinline__ double scaled_weight(float x, bool in) const {
        const double t = exponent(x);
        constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: a sum's low bits are the nearest whole number
        const double k = t + kMagic;
        const int whole = __double2loint(k);
        const double r = t - (k - kMagic);
        constexpr double c1 = kLn2 / 256.0, c2 = c1 * c1 / 2.0, c3 = c2 * c1 / 3.0, c4 = c3 * c1 / 4.0;
        const double p = sm.powers[whole & 255] * fma(r, fma(r, fma(r, fma(r, c4, c3), c2), c1), 1.0);
        const int high = __double2hiint(p) + static_cast<int>(static_cast<uint32_t>(whole & ~255) << 12);  // times 2^(whole / 256)
        // below 2^-64 (and for NaN) 0; with a high word of 0 the number is far below 1, which is as good
        return __hiloint2double(in && t > -16384.0 ? high : 0, __double2loint(p));
    }
    // Such a number rounded to a whole one, plus kBias.
    static __device__ __forceinline__ u64 biased(double w) {
        return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0));
    }
    __device__ __forceinline__ u64 weight(float x) const { return biased(scaled_weight(x, true)) - kBias; }
    // Larger for smaller logits.
    __device__ __forceinline__ int bin(float x) const {
        return static_cast<int>(fminf((top - x) * bin_scale, static_cast<float>(kBins - 1)));
    }
    __device__ __forceinline__ bool passes(float x, int index) const {
        return x > last || (x == last && index <= last_index);
    }
    // Of an element that is left.
    __device__ __forceinline__ u64 kept(int index, float x) const {
        const double w = scaled_weight(x, passes(x, index));
        return w >= least_weight ? biased(w) - kBias : 0;
    }
    // f(index of the first, E logits) for every load, group by group, the next group's loads in flight; after(block) when a
    // block's are done.
    template <class F, class G> __device__ __forceinline__ void pass(F f, G after) const {
        const int64_t groups = (row.size + Row<T>::kGroup - 1) / Row<T>::kGroup;
        int block = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
        int64_t at = static_cast<int64_t>(block) * a.groups;
        if (at >= groups) {
            return;
        }
        typename Row<T>::Group now = row.load(at);
        for (;;) {
            int64_t next = at + 1;
            const bool done = next >= groups || next == static_cast<int64_t>(block + 1) * a.groups;
            if (done) {
                next = static_cast<int64_t>(block + kWaves) * a.groups;
            }
            typename Row<T>::Group ahead = now;
            if (next < groups) {
                ahead = row.load(next);
            }
            row.each(at, now, f);
            if (done) {
                after(block);
                block += kWaves;
            }
            if (next >= groups) {
                break;
            }
            now = ahead;
            at = next;
        }
    }
    // f(index, x) for the elements for which test(x) holds, few in earnest
    template <class Test, class F> __device__ __forceinline__ void pass_some(Test test, F f) const {
        pass(
            [&](int first, u32x4 w) KDA_INLINE {
                bool some = false;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    some |= test(Row<T>::element(w, e));
                }
                if (__any(some)) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float x = Row<T>::element(w, e);
                        if (test(x)) {
                            f(first + e, x);
                        }
                    }
                }
            },
            [](int) {});
    }
    __device__ __forceinline__ int blocks() const {
        const int64_t per = static_cast<int64_t>(a.groups) * Row<T>::kGroup;
        return static_cast<int>((row.size + per - 1) / per);
    }
    // The sum of the blocks' masses, once they are there. By all threads.
    __device__ __forceinline__ u64 all_blocks() {
        __syncthreads();
        u64 total;
        const int n = blocks(), i = 2 * static_cast<int>(threadIdx.x);
        block_scan(sm, (i < n ? sm.blocks[i] : 0) + (i + 1 < n ? sm.blocks[i + 1] : 0), total);
        return total;
    }
    __device__ __forceinline__ void block_done(int block, u64 &mine) {
        const u64 sum = last_lane(wave_scan(mine));
        if (__lane_id() == 0) {
            sm.blocks[block] = sum;
        }
        mine = 0;
    }
    // The blocks' masses of what is left (kNucleus: and the bins' of all that pass; kNumbers: only the bins' numbers); their sum.
    template <bool CUT> __device__ __forceinline__ u64 masses(Mode mode) {
        u64 mine = 0;
        pass(
            [&](int first, u32x4 w) KDA_INLINE {
                if (mode == kNumbers) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float x = Row<T>::element(w, e);
                        if (x > -kInf) {
                            atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[bin(x)]), 1ull);
                        }
                    }
                    return;
                }
                if (mode == kLeft) {
                    bool some = false;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        some |= Row<T>::element(w, e) >= least;
                    }
                    if (!__any(some)) {
                        return;
                    }
                }
#pragma unroll
                for (int part = 0; part < E; part += 4) {
                    u64 m[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = Row<T>::element(w, part + e);
                        const double v = scaled_weight(x, CUT ? passes(x, first + part + e) : true);
                        m[e] = biased(v);
                        mine += v >= least_weight ? m[e] : kBias;
                    }
                    if (mode == kNucleus) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (!CUT || m[e] != kBias) {  // 0 is added to a bin sooner than looked for
                                atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[bin(Row<T>::element(w, part + e))]),
                                          static_cast<unsigned long long>(m[e] - kBias));
                            }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);  // four at a time: all at once do not fit the registers
                }
                mine -= E * kBias;
            },
            [&](int block) KDA_INLINE { block_done(block, mine); });
        return all_blocks();
    }
    // The blocks' numbers of elements equal to x that pass; their sum.
    __device__ __forceinline__ u64 numbers_of(float x) {
        u64 mine = 0;
        pass(
            [&](int first, u32x4 w) KDA_INLINE {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    mine += Row<T>::element(w, e) == x && passes(x, first + e) ? 1 : 0;
                }
            },
            [&](int block) KDA_INLINE { block_done(block, mine); });
        return all_blocks();
    }
    // The first element in the vocabulary's order where the sum of w(index, value) reaches `target` (1 to the sum of
    // the blocks' masses), in every thread.
    template <class W> __device__ __forceinline__ int locate(u64 target, W w) {
        u64 before;
        return locate_in(block_of(target, before), before, target, w);
    }
    // The block in which the sum of the blocks' masses reaches `target`, and the sum before it, in every thread; one of the
    // row's blocks whatever the sums are.
    __device__ __forceinline__ int block_of(u64 target, u64 &before) {
        const int n = blocks(), i = 2 * static_cast<int>(threadIdx.x);
        const u64 m0 = i < n ? sm.blocks[i] : 0, m1 = i + 1 < n ? sm.blocks[i + 1] : 0;
        u64 total;
        const u64 sum = block_scan(sm, m0 + m1, total);
        if (sum >= target && sum - m0 - m1 < target) {
            const bool second = sum - m1 < target;
            sm.count = second ? i + 1 : i;
            sm.before = second ? sum - m1 : sum - m0 - m1;
        }
        __syncthreads();
        const uint32_t found = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sm.count));
        before = sm.before;
        __syncthreads();
        return static_cast<int>(min(found, static_cast<uint32_t>(n - 1)));
    }
    template <class W> __device__ __forceinline__ int locate_in(int block, u64 before, u64 target, W w) {
        // a wave for each load of a group
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
        const int64_t first_group = static_cast<int64_t>(block) * a.groups;
        for (int64_t g = first_group; g < first_group + a.groups; ++g) {
            u64 m[E], mine = 0;
            const int64_t first = g * Row<T>::kGroup + (wave * 64 + static_cast<int>(__lane_id())) * E;
            if (wave < kUnroll) {
                const u32x4 raw = row.guarded(first);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    m[e] = w(static_cast<int>(first) + e, Row<T>::element(raw, e));
                    mine += m[e];
                    if (e % 4 == 3) {
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            u64 all;
            u64 sum = before + block_scan(sm, mine, all);
            if (sum >= target && sum - mine < target) {
                sum -= mine;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (sum < target && sum + m[e] >= target) {
                        sm.found = static_cast<u64>(first + e);
                    }
                    sum += m[e];
                }
            }
            before += all;
            if (before >= target) {
                break;
            }
        }
        __syncthreads();
        const int found = static_cast<int>(sm.found);
        __syncthreads();
        return found;
    }
    // The bin where the sum of the bins reaches `target`, and the sum before it, in every thread.
    __device__ __forceinline__ int border(u64 target, u64 &before) {
        __syncthreads();
        const int i = 2 * static_cast<int>(threadIdx.x);
        const u64 m0 = sm.bins[i], m1 = sm.bins[i + 1];
        u64 total;
        const u64 sum = block_scan(sm, m0 + m1, total);
        if (sum >= target && sum - m0 - m1 < target) {
            const bool second = sum - m1 < target;
            sm.count = second ? i + 1 : i;
            sm.before = second ? sum - m1 : sum - m0 - m1;
        }
        __syncthreads();
        const int found = __builtin_amdgcn_readfirstlane(sm.count);
        before = sm.before;
        __syncthreads();
        return found;
    }
    __device__ __forceinline__ void clear_bins() {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            sm.bins[i] = 0;
        }
        __syncthreads();
    }
    // Appends to the list what test(x) and in(index, x) hold for, as far as it fits, and returns their number and the
    // least and largest key. By all threads.
    template <class Test, class In> __device__ __forceinline__ int gather(Test test, In in, uint32_t &low, uint32_t &high) {
        __syncthreads();
        if (threadIdx.x == 0) {
            sm.count = 0;
            sm.low = 0xffffffffu;
            sm.high = 0;
        }
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        pass_some(test, [&](int index, float x) KDA_INLINE {
            if (in(index, x)) {
                const uint32_t key = key_of(x);
                lo = min(lo, key);
                hi = max(hi, key);
                const int at = atomicAdd(&sm.count, 1);
                if (at < kList) {
                    sm.list[at] = rank_of(key, static_cast<uint32_t>(index));
                }
            }
        });
        if (hi != 0) {
            atomicMin(&sm.low, lo);
            atomicMax(&sm.high, hi);
        }
        __syncthreads();
        low = sm.low;
        high = sm.high;
        const int n = __builtin_amdgcn_readfirstlane(sm.count);
        __syncthreads();
        return n;
    }
    __device__ __forceinline__ float logprob_of(int index, u64 mass) const {
        const float x = Row<T>::element(row.guarded(index), 0);
        // (the mass in units of the largest weight: a token that is left alone gets exactly 0)
        return static_cast<float>(exponent(x) * (kLn2 / 256.0) - log(ldexp(static_cast<double>(mass), -a.shift)));
    }
    __device__ __forceinline__ void cut_behind(float x, int index) {
        last = x;
        last_index = index;
        least = fmaxf(floor, x);
    }
    __device__ __forceinline__ void uncut() { cut_behind(-kInf, -1); }

    // ---- bf16 logits have few values. Those of a row that have a weight lie within kOctaves powers of two of
    // the largest magnitude among them, kPatterns patterns. Their places are in falling order: positive ones 1 to kSide from the
    // largest on, negative ones kSide + 1 to kPatterns to the largest magnitude; 0 and kPatterns + 1 are for all
    // others, which have no weight, but those between the two sides (zeros too), which are formed one by one.
    static constexpr int kSide = kPatterns / 2, kOctaves = kSide / 128;
    int base;       // the least magnitude's pattern
    u64 tie_limit;  // how many of those equal to `last` are left
    // The places of a word's two patterns, 16 bits each (one at a time: 256 rows of 150000 57 us, 52 so); `magnitude` gets how
    // far they are from the least one, 0x8000 and above for those between the sides.
    __device__ __forceinline__ u16x2 places_of(uint32_t word, u16x2 &magnitude) const {
        magnitude = __builtin_bit_cast(u16x2, word & 0x7fff7fffu) - static_cast<uint16_t>(base);
        const u16x2 inside = __builtin_elementwise_min(magnitude, u16x2{kSide, kSide});
        const uint32_t negative = __builtin_bit_cast(uint32_t, __builtin_bit_cast(s16x2, word) >> static_cast<int16_t>(15));
        return __builtin_bit_cast(u16x2, __builtin_bit_cast(uint32_t, inside) ^ ~negative) + static_cast<uint16_t>(kSide + 1);
    }
    __device__ __forceinline__ float value_at(int place) const {
        const uint32_t m = static_cast<uint32_t>(place <= kSide ? kSide - place : place - kSide - 1) + base;
        return __uint_as_float((m | (place <= kSide ? 0u : 0x8000u)) << 16);
    }
    // A window that fits most rows, of magnitudes below 2^7: patterns may be counted in it before the largest logit is
    // known.
    static constexpr int kUsualBase = (134 - kOctaves) << 7;
    static constexpr uint32_t kAside = kMaxBlocks;  // logits between the sides that are kept (in place of the blocks) until then
    __device__ __forceinline__ void clear_patterns() {
        __syncthreads();
        for (int i = threadIdx.x; i < kPatterns; i += kThreads) {
            sm.numbers()[i + 1] = 0;
        }
        if (threadIdx.x == 0) {
            sm.between = 0;
            sm.between_count = 0;
        }
        __syncthreads();
    }
    // Whether the row's logits are taken so; their weights into the table, and their numbers if `cuts`. `counted`: these are
    // there, in the usual window, which may not do.
    __device__ __forceinline__ bool tabulate(bool counted, bool cuts) {
        const float range = static_cast<float>(256.0 * (a.shift + 2.1) / scale);  // below it weights are 0
        const float most = fmaxf(fabsf(top), fabsf(top - range));
        const int exponent_of_most = __float_as_int(most) >> 23, exponent_of_top = __float_as_int(fabsf(top)) >> 23;
        // (a very high temperature would put most logits between the sides)
        if (sizeof(T) != 2 || exponent_of_most <= kOctaves || exponent_of_most > max(exponent_of_top, 130) + kOctaves - 12 || exponent_of_most > 254) {
            return false;
        }
        counted = counted && exponent_of_most < 134 && sm.between_count <= kAside;
        base = counted ? kUsualBase : (exponent_of_most - (kOctaves - 1)) << 7;
        if (!counted) {
            clear_patterns();
            if (cuts) {
                count_patterns();
            }
        }
        for (int i = threadIdx.x; i < kPatterns + 2; i += kThreads) {
            sm.table()[i] = i > 0 && i <= kPatterns ? weight(fminf(value_at(i), top)) : 0;
        }
        if (counted) {
            u64 mine = 0;
            const uint32_t *aside = reinterpret_cast<const uint32_t *>(sm.blocks);
            for (uint32_t i = threadIdx.x; i < sm.between_count; i += kThreads) {
                mine += weight(__uint_as_float(aside[i]));
            }
            u64 all;
            block_scan(sm, mine, all);
            if (threadIdx.x == 0) {
                sm.between = all;
            }
        }
        __syncthreads();
        return true;
    }
    // Counts eight logits; the high bits of the result's halves tell whether some are between the sides.
    __device__ __forceinline__ uint32_t count(u32x4 w) const {
        uint32_t some = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u16x2 magnitude;
            const u16x2 place = places_of(w[i], magnitude);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (magnitude[e] < kSide) {
                    atomicAdd(&sm.numbers()[place[e]], 1u);
                }
            }
            some |= __builtin_bit_cast(uint32_t, magnitude);
        }
        return some;
    }
    // The patterns' numbers in the usual window, and the largest logit.
    __device__ __forceinline__ void count_first(float &largest) {
        base = kUsualBase;
        clear_patterns();
        pass(
            [&](int, u32x4 w) KDA_INLINE {
                const uint32_t some = count(w);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    largest = fmaxf(largest, Row<T>::element(w, e));
                }
                if (__any((some & 0x80008000u) != 0)) {
                    each_between(w, [&](float x) KDA_INLINE {
                        const uint32_t at = atomicAdd(&sm.between_count, 1u);
                        if (at < kAside) {
                            reinterpret_cast<uint32_t *>(sm.blocks)[at] = __float_as_uint(x);
                        }
                    });
                }
            },
            [](int) {});
    }
    // f(x) for the logits between the sides among a lane's
    template <class F> __device__ __forceinline__ void each_between(u32x4 w, F f) const {
#pragma unroll 1
        for (int e = 0; e < E; ++e) {
            if (static_cast<int>(w[0] & 0x7fffu) < base) {
                f(Row<T>::element(w, 0));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = w[i] >> 16 | (i < 3 ? w[(i + 1) & 3] << 16 : 0u);
            }
        }
    }
    // Each pattern's number, and number and mass of what lies between.
    __device__ __forceinline__ void count_patterns() {
        pass(
            [&](int, u32x4 w) KDA_INLINE {
                if (__any((count(w) & 0x80008000u) != 0)) {
                    each_between(w, [&](float x) KDA_INLINE {
                        const u64 m = weight(x);
                        atomicAdd(&sm.between_count, m != 0 ? 1u : 0u);
                        atomicAdd(reinterpret_cast<unsigned long long *>(&sm.between), static_cast<unsigned long long>(m));
                    });
                }
            },
            [](int) {});
        __syncthreads();
    }
    // Cuts behind the k-th (0: does not) and behind the nucleus of what is left; false where a border lies between the sides.
    // `left`: about how many are left.
    __device__ __forceinline__ bool cut_patterns(u64 k, bool nucleus, double top_p, u64 &left) {
        constexpr int kEach = kPatterns / kThreads;
        const int first = kEach * static_cast<int>(threadIdx.x) + 1;
        u64 n[kEach], all, total;
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {  // 16 bytes at a time, or the lanes meet in few banks
            const u32x4 four = *reinterpret_cast<const u32x4 *>(sm.numbers() + first + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                n[i + e] = four[e];
            }
        }
        u64 between = sm.between;
        const auto sum_of = [](const u64 (&m)[kEach]) KDA_INLINE -> u64 {
            u64 sum = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                sum += m[i];
            }
            return sum;
        };
        // the place at which the sum of m reaches the target, and the sum before it, into sm; false if that is between the sides
        const auto border_at = [&](const u64 (&m)[kEach], u64 middle, u64 target) KDA_INLINE -> bool {
            u64 sum = sum_of(m);
            sum = block_scan(sm, sum, all) - sum + (first > kSide ? middle : 0);
            if (threadIdx.x == 0) {
                sm.count = -1;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                if (sum < target && sum + m[i] >= target) {
                    sm.count = first + i;
                    sm.before = sum;
                }
                sum += m[i];
            }
            __syncthreads();
            return sm.count >= 0;
        };
        block_scan(sm, sum_of(n), total);
        left = total;
        if (k > 0 && k < total + sm.between_count) {
            left = k;
            if (!border_at(n, sm.between_count, k)) {
                return false;
            }
            const int at = sm.count;
            tie_limit = k - sm.before;
            cut_behind(value_at(at), 0x7fffffff);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                n[i] = first + i < at ? n[i] : first + i == at ? tie_limit : 0;
            }
            between = at <= kSide ? 0 : between;
        }
        if (nucleus) {
            u64 m[kEach];
#pragma unroll
            for (int i = 0; i < kEach; i += 2) {
                const u32x4 two = *reinterpret_cast<const u32x4 *>(sm.table() + first + i);
                m[i] = n[i] * (static_cast<u64>(two[1]) << 32 | two[0]);
                m[i + 1] = n[i + 1] * (static_cast<u64>(two[3]) << 32 | two[2]);
            }
            block_scan(sm, sum_of(m), total);
            const u64 target = reaching(top_p, total + between);
            if (!border_at(m, between, target)) {
                return false;
            }
            const int at = sm.count;
            const u64 each = sm.table()[at];
            tie_limit = (target - sm.before + each - 1) / each;
            cut_behind(value_at(at), 0x7fffffff);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                n[i] = first + i <= at ? n[i] : 0;
            }
            block_scan(sm, sum_of(n), left);
        }
        return true;
    }
    // Takes out of the table what is cut or does not reach min_p; what equals `last` gets kTie: a lane's weights of a block
    // stay below it, and their number above.
    __device__ __forceinline__ void cut_table() {
        __syncthreads();
        const u64 at_least = biased(least_weight) - kBias;
        for (int i = threadIdx.x + 1; i <= kPatterns; i += kThreads) {
            const float x = value_at(i);
            const u64 m = sm.table()[i];
            // rounded weights decide where they differ from min_p's
            if (!(x > last) || m < at_least || (m == at_least && !(scaled_weight(fminf(x, top), true) >= least_weight))) {
                sm.table()[i] = x == last ? kTie : 0;
            }
        }
        __syncthreads();
    }
    static constexpr int kTieShift = 57;  // 32 elements of at most 2^51
    static constexpr u64 kTie = u64{1} << kTieShift;
    // The blocks' masses of what is left, as masses(); equal ones at the cut are counted by block, and those of the
    // lowest indices added. `tie_block` gets the last block that holds any of those, `tie_count` their number in it.
    // `few`: most groups of loads hold nothing that is left.
    __device__ __forceinline__ u64 pattern_masses(bool few, int &tie_block, u64 &tie_count) {
        u64 mine = 0;
        const bool cut = last > -kInf;
        pass(
            [&](int, u32x4 w) KDA_INLINE {
                if (few) {
                    bool some = false;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        some |= Row<T>::element(w, e) >= least;
                    }
                    if (!__any(some)) {
                        return;
                    }
                }
                uint32_t between = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u16x2 magnitude;
                    const u16x2 place = places_of(w[i], magnitude);
                    mine += sm.table()[place[0]];
                    mine += sm.table()[place[1]];
                    between |= __builtin_bit_cast(uint32_t, magnitude);
                }
                if (__any((between & 0x80008000u) != 0)) {
                    each_between(w, [&](float x) KDA_INLINE {
                        const double v = scaled_weight(x, x > last);
                        mine += v >= least_weight ? biased(v) - kBias : 0;
                    });
                }
            },
            [&](int block) KDA_INLINE {
                if (cut) {
                    const u64 number = last_lane(wave_scan(mine >> kTieShift));
                    if (__lane_id() == 0) {
                        sm.ties[block] = static_cast<uint32_t>(number);
                    }
                    mine &= kTie - 1;
                }
                block_done(block, mine);
            });
        tie_block = 0x7fffffff;
        tie_count = 0;
        if (cut) {
            __syncthreads();
            const int n = blocks(), first = 2 * static_cast<int>(threadIdx.x);
            const double v = scaled_weight(last, true);
            const u64 each = v >= least_weight ? biased(v) - kBias : 0;
            u64 t[2] = {first < n ? sm.ties[first] : 0u, first + 1 < n ? sm.ties[first + 1] : 0u}, all;
            u64 before = block_scan(sm, t[0] + t[1], all) - t[0] - t[1];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const u64 left = before >= tie_limit ? 0 : min(t[i], tie_limit - before);
                if (left > 0) {
                    sm.blocks[first + i] += left * each;
                }
                if (before < tie_limit && before + t[i] >= tie_limit) {
                    sm.count = first + i;
                    sm.before = left;
                }
                before += t[i];
            }
            __syncthreads();
            tie_block = sm.count;
            tie_count = sm.before;
        }
        return all_blocks();
    }

    // Cuts behind the element at which the number (or mass) of the elements that pass, in the order of their ranks,
    // reaches `target`, which that of all does. The bins hold those of their elements.
    __device__ __forceinline__ void cut(u64 target, bool number) {
        u64 before, more;
        uint32_t at = static_cast<uint32_t>(border(target, before));
        uint32_t first = 0, last_key = 0, low, high;  // keys
        int shift = -1;                               // of the keys' bins, -1: bins by distance
        // logits that bin `at` may hold, and some more
        float from = -kInf, to = kInf;
        if (bin_scale > 0.0f && bin_scale < 1e30f) {
            const float slack = 1e-5f * fabsf(top);
            from = at + 1 < kBins ? top - (static_cast<float>(at) + 2.0f) / bin_scale - slack : -kInf;
            to = top - (static_cast<float>(at) - 1.0f) / bin_scale + slack;
        }
        int n;
        for (;;) {
            n = gather([&](float x) KDA_INLINE { return x >= from && x <= to; },
                       [&](int index, float x) KDA_INLINE {
                           return x > -kInf && passes(x, index) && (shift < 0 ? static_cast<uint32_t>(bin(x)) == at
                                                                              : (last_key - key_of(x)) >> shift == at);
                       },
                       low, high);
            if (n <= kList || low == high) {
                break;
            }
            // more than fit: bins of their keys, the largest first
            first = low;
            last_key = high;
            from = of_key(first);
            to = of_key(last_key);
            shift = max(21 - __clz(high - low), 0);
            clear_bins();
            pass_some([&](float x) KDA_INLINE { return x >= from && x <= to; },
                      [&](int index, float x) KDA_INLINE {
                          if (passes(x, index)) {
                              const u64 w = number ? 1 : weight(x);
                              atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[(last_key - key_of(x)) >> shift]),
                                        static_cast<unsigned long long>(w));
                          }
                      });
            at = static_cast<uint32_t>(border(target - before, more));
            before += more;
        }
        if (n > kList) {
            // all equal: so many of them in the vocabulary's order
            const float x = of_key(low);
            const u64 each = number ? 1 : weight(x);
            const u64 count = (target - before + each - 1) / each;
            numbers_of(x);
            cut_behind(x, locate(count, [&](int index, float y) KDA_INLINE -> u64 { return y == x && passes(x, index) ? 1 : 0; }));
            return;
        }
        sort(sm, n);
        const int i = threadIdx.x;
        const u64 mass = i < n ? (number ? 1 : weight(of_key(static_cast<uint32_t>(sm.list[i] >> 32)))) : 0;
        u64 total;
        const u64 sum = before + block_scan(sm, mass, total);
        if (sum >= target && sum - mass < target) {
            sm.found = sm.list[i];
        }
        __syncthreads();
        const u64 rank = sm.found;
        __syncthreads();
        cut_behind(of_key(static_cast<uint32_t>(rank >> 32)), static_cast<int>(index_of(rank)));
    }
};

template <typename T, int kPatterns> __global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams a) {
    __shared__ Shared<kPatterns> sm;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t n = blockIdx.x;
    const float temperature = a.temperature != nullptr ? a.temperature[n] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    // (all of a row's numbers at once, before its logits)
    const float min_p = a.min_p != nullptr ? a.min_p[n] : 0.0f;
    const float top_p = a.top_p != nullptr ? a.top_p[n] : 1.0f;
    const bool nucleus = top_p < 1.0f;
    const int64_t k = a.top_k == nullptr          ? 0
                      : (a.top_k_int64 != 0) ? static_cast<const int64_t *>(a.top_k)[n]
                                             : static_cast<const int32_t *>(a.top_k)[n];
    const bool few_k = k > 0 && k < a.vocab;
    const float given = a.uniforms[n];
    const double u = given > 0.0f ? static_cast<double>(given) : 0.0;
    Row<T> row{static_cast<const T *>(a.logits) + n * a.logits_stride, a.vocab};
    Sampler<T, kPatterns> s{a, sm, row, 0.0f, 0.0, 0.0f, -kInf, -1, 0.0, -kInf, -kInf};

    // ---- the largest logit, and where it is first
    float top = -kInf;
    int place = 0;
    bool counted = false;  // bf16 patterns
    if (greedy) {
        s.pass(
            [&](int first, u32x4 w) KDA_INLINE {
#pragma unroll
                for (int e = 0; e < s.E; ++e) {
                    const float x = Row<T>::element(w, e);
                    place = x > top ? first + e : place;
                    top = fmaxf(top, x);
                }
            },
            [](int) {});
    } else {
        if constexpr (sizeof(T) == 2) {
            counted = a.groups == 1 && (few_k ? k > kFewK : nucleus);
        }
        if (counted) {
            s.count_first(top);
        } else {
            s.pass(
                [&](int, u32x4 w) KDA_INLINE {
#pragma unroll
                    for (int e = 0; e < s.E; ++e) {
                        top = fmaxf(top, Row<T>::element(w, e));
                    }
                },
                [](int) {});
        }
        if (tid < 256) {
            sm.powers[tid] = ldexp(exp2(tid * (1.0 / 256.0)), a.shift);
        }
    }
    const float mine = top;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const float x = __shfl_xor(top, d);
        const int at = __shfl_xor(place, d);
        place = x > top ? at : x == top ? min(place, at) : place;
        top = fmaxf(top, x);
    }
    if (lane == 0) {
        sm.tops[wave] = top;
        sm.places[wave] = place;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float x = sm.tops[w];
        place = x > top ? sm.places[w] : x == top ? min(place, sm.places[w]) : place;
        top = fmaxf(top, x);
    }
    int64_t *token = a.tokens + n;
    float *logprob = a.logprobs + n;
    if (top == -kInf || greedy) {
        if (tid == 0) {
            *token = top == -kInf ? -1 : place;
            *logprob = top == -kInf ? -kInf : 0.0f;
        }
        return;
    }
    if (top == kInf) {  // the infinite ones share the mass
        u64 share = s.numbers_of(kInf);
        share = few_k ? min(share, static_cast<u64>(k)) : share;
        share = nucleus ? reaching(static_cast<double>(top_p), share) : share;
        const int found = s.locate(exceeding(u, share), [](int, float x) KDA_INLINE -> u64 { return x == kInf ? 1 : 0; });
        if (tid == 0) {
            *token = found;
            *logprob = static_cast<float>(-log(static_cast<double>(share)));
        }
        return;
    }
    s.top = top;
    s.scale = 256.0 * kLog2e / static_cast<double>(temperature);
    s.bin_scale = static_cast<float>(static_cast<double>(kBins - 1) / (static_cast<double>(temperature) * kLn2 * (a.shift + 2)));
    if (min_p > 0.0f) {
        const double p = static_cast<double>(fminf(min_p, 1.0f));
        s.least_weight = ldexp(p, a.shift);
        // (of p = 1 the logarithm is 0, which an infinite temperature would make NaN)
        const double x = static_cast<double>(top) + (p < 1.0 ? log(p) * static_cast<double>(temperature) : 0.0);
        s.floor = s.least = static_cast<float>(x - 1e-6 * (fabs(x) + fabs(static_cast<double>(top)) + static_cast<double>(temperature)));
    }

    if (few_k && k <= kFewK && s.bin_scale > 1e-30f && s.bin_scale < 1e30f) {
        // ---- candidates: what is in the bins up to that of the k-th largest of the threads' maxima. (The last bin's
        // weights are 0.)
        s.clear_bins();
        const int own = mine > -kInf ? s.bin(mine) : kBins;
        atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[own]), 1ull);
        __syncthreads();
        u64 all;
        const u64 m0 = sm.bins[2 * tid], m1 = sm.bins[2 * tid + 1];
        const u64 below = block_scan(sm, m0 + m1, all) - m0 - m1;
        if (tid == 0) {
            sm.count = kBins - 1;
        }
        __syncthreads();
        if (below < static_cast<u64>(k) && below + m0 + m1 >= static_cast<u64>(k)) {
            sm.count = below + m0 >= static_cast<u64>(k) ? 2 * tid : 2 * tid + 1;
        }
        __syncthreads();
        const int bins = min(__builtin_amdgcn_readfirstlane(sm.count) + 1, kBins - 1);
        uint32_t low, high;
        const float reached = top - (static_cast<float>(bins) + 1.0f) / s.bin_scale - 1e-5f * fabsf(top);
        const int count = s.gather([&](float x) KDA_INLINE { return x >= reached; },
                                   [&](int, float x) KDA_INLINE { return s.bin(x) < bins; }, low, high);
        if (count <= kFew) {
            sort(sm, count);
            const u64 rank = tid < count ? sm.list[tid] : 0;
            bool in = tid < count && (!few_k || tid < k);
            u64 w = in ? s.weight(of_key(static_cast<uint32_t>(rank >> 32))) : 0;
            const bool high_enough = in && s.scaled_weight(of_key(static_cast<uint32_t>(rank >> 32)), true) >= s.least_weight;
            u64 total;
            u64 sum = block_scan(sm, w, total);
            if (nucleus) {
                in = in && sum - w < reaching(static_cast<double>(top_p), total);
            }
            w = in && high_enough ? w : 0;
            sm.weights[tid] = w;
            __syncthreads();  // everybody has their rank
            // in the vocabulary's order
            sm.list[tid] = w > 0 ? static_cast<u64>(index_of(rank) ^ 0xffffffffu) << 32 | static_cast<uint32_t>(tid) : 0;
            sort(sm, count);
            const u64 entry = sm.list[tid];
            w = tid < count && entry != 0 ? sm.weights[static_cast<uint32_t>(entry)] : 0;
            sum = block_scan(sm, w, total);
            const u64 target = exceeding(u, total);
            if (sum >= target && sum - w < target) {
                const int index = static_cast<int>(static_cast<uint32_t>(entry >> 32) ^ 0xffffffffu);
                *token = index;
                *logprob = s.logprob_of(index, total);
            }
            return;
        }
    }
    const auto finish = [&](int found, u64 mass) KDA_INLINE {
        found = min(static_cast<uint32_t>(found), static_cast<uint32_t>(a.vocab - 1));  // also if logits change between the passes
        if (tid == 0) {
            *token = found;
            *logprob = s.logprob_of(found, mass);
        }
    };
    // ---- bf16: the patterns' numbers cut, then one pass for the blocks' masses
    if constexpr (sizeof(T) == 2) {
        if (a.groups == 1 && s.tabulate(counted, few_k || nucleus)) {
            bool cut = true;
            u64 left = 0;
            if (few_k || nucleus) {
                cut = s.cut_patterns(few_k ? static_cast<u64>(k) : 0, nucleus, static_cast<double>(top_p), left);
            }
            if (cut) {
                if (s.least > -kInf) {
                    s.cut_table();
                }
                int tie_block;
                u64 tie_count, before;
                const u64 mass = s.pattern_masses(s.floor > -kInf || (s.last > -kInf && left < static_cast<u64>(a.vocab >> 8)), tie_block, tie_count);
                const u64 target = exceeding(u, mass);
                const int block = s.block_of(target, before);
                // of equal elements at the cut: in blocks before the last that holds some all are left, behind it none
                if (block == tie_block) {
                    s.last_index = 0x7fffffff;
                    const float x = s.last;
                    s.last_index = s.locate_in(block, 0, tie_count, [&](int, float y) KDA_INLINE -> u64 { return y == x ? 1 : 0; });
                } else {
                    s.last_index = block < tie_block ? 0x7fffffff : -1;
                }
                finish(s.locate_in(block, before, target, [&](int index, float x) KDA_INLINE -> u64 { return s.kept(index, x); }), mass);
                return;
            }
            s.uncut();
        }
    }
    // ---- top_k's cut (numbers in bins), the nucleus' (masses in bins), the blocks' masses of what is left
    Mode mode = few_k ? kNumbers : nucleus ? kNucleus : kLeft;
    if (mode != kLeft) {
        s.clear_bins();
    }
    u64 mass = s.template masses<false>(mode);
    while (mode != kLeft) {
        u64 all;
        block_scan(sm, sm.bins[2 * tid] + sm.bins[2 * tid + 1], all);
        const u64 target = mode == kNumbers ? static_cast<u64>(k) : reaching(static_cast<double>(top_p), all);
        if (mode == kNumbers ? target < all : target < mass) {
            s.cut(target, mode == kNumbers);
        } else if (mode == kNucleus) {
            break;  // min_p cuts what the nucleus would
        }
        mode = mode == kNumbers && nucleus ? kNucleus : kLeft;
        if (mode == kNucleus) {
            s.clear_bins();
        }
        mass = s.template masses<true>(mode);
    }
    finish(s.locate(exceeding(u, mass), [&](int index, float x) KDA_INLINE -> u64 { return s.kept(index, x); }), mass);
}

}  // namespace
}  // namespace kda

extern "C" int kda_sample_launch(const KdaSampleArgs *args, void *stream) {
    using namespace kda;
    if (args == nullptr) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const auto off = [](const void *p, uintptr_t m) { return reinterpret_cast<uintptr_t>(p) % m != 0; };
    if (args->dtype != KDA_BF16 && args->dtype != KDA_F32) {
        return KDA_ERR_UNSUPPORTED;
    }
    if (args->rows < 0 || args->vocab <= 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    // indices of the last load's elements stay in 32 bits; a grid counts its threads in 32 bits
    if (args->vocab > INT32_MAX - (1 << 16) || args->rows > UINT32_MAX / kThreads) {
        return KDA_ERR_TOO_LARGE;
    }
    if (args->rows == 0) {
        return KDA_OK;
    }
    if (args->logits == nullptr || off(args->logits, args->dtype == KDA_BF16 ? 2 : 4) || args->uniforms == nullptr ||
        off(args->uniforms, 4) || off(args->temperature, 4) || off(args->top_p, 4) || off(args->min_p, 4) ||
        off(args->top_k, args->top_k_int64 != 0 ? 8 : 4) || args->tokens == nullptr || off(args->tokens, 8) ||
        args->logprobs == nullptr || off(args->logprobs, 4)) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    SampleParams a{*args, 0, 0};
    int bits = 0;
    while ((INT64_C(1) << bits) < a.vocab) {
        ++bits;
    }
    a.shift = std::min(62 - bits, 51);
    const int64_t group = a.dtype == KDA_BF16 ? Row<uint16_t>::kGroup : Row<float>::kGroup;
    a.groups = static_cast<int>((a.vocab + group * kMaxBlocks - 1) / (group * kMaxBlocks));
    hipStream_t s = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const unsigned rows = static_cast<unsigned>(a.rows);
    // Logits below the patterns (of 16 powers of two with 4096, 32 with 8192) are formed one by one, a few in 512, which costs long
    // rows more than the larger table does. us with 4096 and 8192 (long rows take 7% less since places come two at a time): 256 rows of 150000 with top_p and min_p 62.6 56.6, a row of 131072
    // with top_k 2000 45 40; of 32000 23.4 24.0 (top_p 25.5 27.4), of 1000 13.8 15.1
    if (a.dtype == KDA_F32) {
        sample_kernel<float, 4096><<<rows, kThreads, 0, s>>>(a);
    } else if (a.vocab <= 65536) {
        sample_kernel<uint16_t, 4096><<<rows, kThreads, 0, s>>>(a);
    } else {
        sample_kernel<uint16_t, 8192><<<rows, kThreads, 0, s>>>(a);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}
