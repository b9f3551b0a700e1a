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
//   else one pass forms the weights, their mass in kBins bins by distance from the maximum, and each
//     block's mass. Where top_k or top_p cuts, the bin in which the border lies is gathered and sorted (bins of more
//     elements than fit are divided again by their keys, equal elements by their index), and blocks' masses
//     formed anew; the token's block is read once more.
//
// Bound by HBM for the first pass; later ones read the caches and are bound by the vector instructions, about 20
// an element where the weight is formed.

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
constexpr int kList = 4096;    // elements that are sorted
constexpr int kFew = 1024;     // elements that are drawn from in LDS, one a thread
constexpr int kFewK = 512;
constexpr int kMaxBlocks = 2048;
constexpr int kUnroll = 4;     // 16-byte loads of a lane in flight together
constexpr float kInf = __builtin_inff();
constexpr double kLog2e = 1.4426950408889634;
constexpr double kLn2 = 0.6931471805599453;

typedef uint64_t u64;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct SampleParams : KdaSampleArgs {
    int shift;   // S: weights are multiples of 2^-S
    int groups;  // of kUnroll loads of a wave that make a block
};

struct Shared {
    u64 bins[kBins];
    u64 list[kList];
    u64 blocks[kMaxBlocks];
    u64 weights[kFew];
    double powers[256];  // 2^{j / 256}
    u64 waves[kWaves];
    float tops[kWaves];
    int places[kWaves];
    int count;
    uint32_t low, high;  // keys
    u64 before, found;
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

__device__ __forceinline__ u64 up64(u64 x, int d) {
    return static_cast<u64>(__shfl_up(static_cast<unsigned long long>(x), d));
}

// The sum of the values of this lane and those before it in the wave.
__device__ __forceinline__ u64 wave_scan(u64 x) {
    const int lane = static_cast<int>(__lane_id());
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 up = up64(x, d);
        x += lane >= d ? up : 0;
    }
    return x;
}
// ... of this thread and those before it, and the sum of all. By all threads.
__device__ __forceinline__ u64 block_scan(Shared &sm, u64 x, u64 &total) {
    const int lane = static_cast<int>(__lane_id()), wave = threadIdx.x >> 6;
    x = wave_scan(x);
    __syncthreads();  // the last one's sums are read
    if (lane == 63) {
        sm.waves[wave] = x;
    }
    __syncthreads();
    u64 before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? sm.waves[w] : 0;
        total += sm.waves[w];
    }
    return x + before;
}

// The list's first `size` (a power of two) entries in falling order. By all threads.
__device__ __forceinline__ void sort(Shared &sm, int size) {
    for (int span = 2; span <= size; span <<= 1) {
        for (int step = span >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const u64 x = sm.list[a], y = sm.list[b];
                if ((x < y) == ((a & span) == 0)) {
                    sm.list[a] = y;
                    sm.list[b] = x;
                }
            }
        }
    }
    __syncthreads();
}
__device__ __forceinline__ int power_above(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// A row's logits; NaN counts as -infinity, and where the maximum is infinite all but it do.
template <typename T> struct Row {
    static constexpr int E = 16 / sizeof(T);
    static constexpr int kGroup = 64 * E * kUnroll;  // elements that a wave loads at a time
    const T *at;
    int size;
    float least, most;

    struct __attribute__((packed, aligned(sizeof(T)))) Raw {
        u32x4 w;
    };
    __device__ __forceinline__ float value(float x) const {
        x = x >= least ? x : -kInf;  // false for NaN
        return fminf(x, most);
    }
    // E logits from element `first`, beyond the row -infinity
    __device__ __forceinline__ u32x4 raw(int first) const {
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
    // f(first index, E values) for the lane's loads of group `group`
    template <class F> __device__ __forceinline__ void each(int group, F f) const {
        const int64_t first = static_cast<int64_t>(group) * kGroup + static_cast<int>(__lane_id()) * E;
        u32x4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t x = first + u * 64 * E;
            w[u] = raw(static_cast<int>(x < size ? x : size));
        }
        // a loop, the loads handed down in it: unrolled, the passes' code would not fit the instruction cache
#pragma unroll 1
        for (int u = 0; u < kUnroll; ++u) {
            f(static_cast<int>(first + u * 64 * E), w[0]);
#pragma unroll
            for (int i = 0; i + 1 < kUnroll; ++i) {
                w[i] = w[i + 1];
            }
        }
    }
};

template <typename T> struct Sampler {
    const SampleParams &a;
    Shared &sm;
    Row<T> row;
    float top;       // the largest logit
    double scale;    // log2(e) / temperature
    float bin_scale;
    float last;      // the last element in the order of the ranks that is not cut
    int last_index;
    double least_weight;  // 0: none

    static constexpr int E = Row<T>::E;

    // log2 of a weight
    __device__ __forceinline__ double exponent(float x) const { return (static_cast<double>(x) - static_cast<double>(top)) * scale; }
    // Of an element; `kept`: it reaches min_p.
    __device__ __forceinline__ u64 weight(float x, bool &kept) const {
        const double t = exponent(x) * 256.0;
        constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: a sum's low bits are the nearest whole number
        const double k = fmax(t, -16384.0) + kMagic;   // 2^-64 at least
        const int whole = static_cast<int>(static_cast<uint32_t>(__double_as_longlong(k)));
        const double r = t - (k - kMagic);
        constexpr double c1 = kLn2 / 256.0, c2 = c1 * c1 / 2.0, c3 = c2 * c1 / 3.0, c4 = c3 * c1 / 4.0;
        const double p = sm.powers[whole & 255] * fma(r, fma(r, fma(r, fma(r, c4, c3), c2), c1), 1.0);
        kept = __builtin_amdgcn_ldexp(p, whole >> 8) >= least_weight;
        constexpr double kTwo52 = 4503599627370496.0;
        const double w = __builtin_amdgcn_ldexp(p, (whole >> 8) + a.shift) + kTwo52;
        return t > -16384.0 ? static_cast<u64>(__double_as_longlong(w)) & 0xfffffffffffffull : 0;
    }
    // Larger for smaller logits.
    __device__ __forceinline__ int bin(float x) const {
        return static_cast<int>(fminf((top - x) * bin_scale, static_cast<float>(kBins - 1)));
    }
    __device__ __forceinline__ bool passes(float x, int index) const {
        return x > last || (x == last && index <= last_index);
    }
    // f(index, value) for every element, group by group; after(block) when a block's are done
    template <class F, class G> __device__ __forceinline__ void pass(F f, G after) const {
        const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
        const int64_t per = static_cast<int64_t>(a.groups) * Row<T>::kGroup;
        for (int block = wave; block * per < row.size; block += kWaves) {
            for (int i = 0; i < a.groups && (static_cast<int64_t>(block) * a.groups + i) * Row<T>::kGroup < row.size; ++i) {
                row.each(block * a.groups + i, [&](int first, u32x4 w) KDA_INLINE {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        f(first + e, row.value(Row<T>::element(w, e)));
                        if (e % 4 == 3) {
                            __builtin_amdgcn_sched_barrier(0);  // four at a time: all at once do not fit the registers
                        }
                    }
                });
            }
            after(block);
        }
    }
    __device__ __forceinline__ int blocks() const {
        const int64_t per = static_cast<int64_t>(a.groups) * Row<T>::kGroup;
        return static_cast<int>((row.size + per - 1) / per);
    }
    // The blocks' masses of w(index, value); their sum. By all threads.
    template <class W> __device__ __forceinline__ u64 block_masses(W w) {
        u64 mine = 0;
        pass([&](int index, float x) KDA_INLINE { mine += w(index, x); },
             [&](int block) KDA_INLINE {
                 const u64 sum = wave_scan(mine);
                 if (__lane_id() == 63) {
                     sm.blocks[block] = sum;
                 }
                 mine = 0;
             });
        return all_blocks();
    }
    __device__ __forceinline__ u64 all_blocks() {
        __syncthreads();
        u64 total;
        const int n = blocks(), i = 2 * static_cast<int>(threadIdx.x);
        block_scan(sm, (i < n ? sm.blocks[i] : 0) + (i + 1 < n ? sm.blocks[i + 1] : 0), total);
        return total;
    }
    // The first element in the vocabulary's order where the sum of w(index, value) reaches `target` (1 to the sum of
    // the blocks' masses), in every thread.
    template <class W> __device__ __forceinline__ int locate(u64 target, W w) {
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
        if (threadIdx.x < 64) {
            const int block = __builtin_amdgcn_readfirstlane(sm.count);
            u64 before = sm.before;
            bool done = false;
            for (int g = 0; g < a.groups && !done && (static_cast<int64_t>(block) * a.groups + g) * Row<T>::kGroup < row.size; ++g) {
                row.each(block * a.groups + g, [&](int first, u32x4 raw) KDA_INLINE {
                    u64 m[E], mine = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        m[e] = w(first + e, row.value(Row<T>::element(raw, e)));
                        mine += m[e];
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    u64 sum = before + wave_scan(mine);
                    if (!done && __any(sum >= target)) {
                        done = true;
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
                    }
                    before = static_cast<u64>(__shfl(static_cast<unsigned long long>(sum), 63));
                });
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
    // Appends to the list what `in` holds for, as far as it fits, and returns their number and the
    // least and largest key. By all threads.
    template <class In> __device__ __forceinline__ int gather(In in, uint32_t &low, uint32_t &high) {
        __syncthreads();
        if (threadIdx.x == 0) {
            sm.count = 0;
            sm.low = 0xffffffffu;
            sm.high = 0;
        }
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        pass(
            [&](int index, float x) KDA_INLINE {
                if (in(index, x)) {
                    const uint32_t key = key_of(x);
                    lo = min(lo, key);
                    hi = max(hi, key);
                    const int at = atomicAdd(&sm.count, 1);
                    if (at < kList) {
                        sm.list[at] = rank_of(key, static_cast<uint32_t>(index));
                    }
                }
            },
            [](int) {});
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
    // Sorted, behind the entries zeros.
    __device__ __forceinline__ int sort_list(int n) {
        const int size = power_above(n);
        for (int i = n + static_cast<int>(threadIdx.x); i < size; i += kThreads) {
            sm.list[i] = 0;
        }
        sort(sm, size);
        return size;
    }

    __device__ __forceinline__ void cut_behind(float x, int index) {
        last = x;
        last_index = index;
    }
    __device__ __forceinline__ u64 weight(float x) const {
        bool reaches;
        return weight(x, reaches);
    }
    // Cuts behind the element at which the number (or mass) of the elements that pass, in the order of their ranks,
    // reaches `target`, which that of all does. The bins hold those of their elements.
    __device__ __forceinline__ void cut(u64 target, bool number) {
        u64 before, more;
        uint32_t at = static_cast<uint32_t>(border(target, before));
        uint32_t first = 0, last_key = 0, low, high;  // keys
        int shift = -1;                               // of the keys' bins, -1: bins by distance
        int n;
        for (;;) {
            n = gather(
                [&](int index, float x) KDA_INLINE {
                    const uint32_t key = key_of(x);
                    return passes(x, index) && (shift < 0 ? static_cast<uint32_t>(bin(x)) == at
                                                          : key >= first && key <= last_key && (last_key - key) >> shift == at);
                },
                low, high);
            if (n <= kList || low == high) {
                break;
            }
            // more than fit: bins of their keys, the largest first
            first = low;
            last_key = high;
            shift = max(21 - __clz(high - low), 0);
            clear_bins();
            pass(
                [&](int index, float x) KDA_INLINE {
                    const uint32_t key = key_of(x);
                    if (passes(x, index) && key >= first && key <= last_key) {
                        const u64 w = number ? 1 : weight(x);
                        atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[(last_key - key) >> shift]), static_cast<unsigned long long>(w));
                    }
                },
                [](int) {});
            at = static_cast<uint32_t>(border(target - before, more));
            before += more;
        }
        if (n > kList) {
            // all equal: so many of them in the vocabulary's order
            const u64 each = number ? 1 : weight(of_key(low));
            const u64 count = (target - before + each - 1) / each;
            const auto one = [&](int index, float x) KDA_INLINE -> u64 { return passes(x, index) && key_of(x) == low ? 1 : 0; };
            block_masses(one);
            cut_behind(of_key(low), locate(count, one));
            return;
        }
        sort_list(n);
        constexpr int kPer = kList / kThreads;
        u64 mass[kPer], mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int x = static_cast<int>(threadIdx.x) * kPer + i;
            mass[i] = x < n ? (number ? 1 : weight(of_key(static_cast<uint32_t>(sm.list[x] >> 32)))) : 0;
            mine += mass[i];
        }
        u64 total;
        u64 sum = before + block_scan(sm, mine, total) - mine;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (sum < target && sum + mass[i] >= target) {
                sm.found = sm.list[threadIdx.x * kPer + i];
            }
            sum += mass[i];
        }
        __syncthreads();
        const u64 rank = sm.found;
        __syncthreads();
        cut_behind(of_key(static_cast<uint32_t>(rank >> 32)), static_cast<int>(index_of(rank)));
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

template <typename T> __global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams a) {
    __shared__ Shared sm;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t n = blockIdx.x;
    const float temperature = a.temperature != nullptr ? a.temperature[n] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    Row<T> row{static_cast<const T *>(a.logits) + n * a.logits_stride, a.vocab, -kInf, kInf};
    Sampler<T> s{a, sm, row, 0.0f, 0.0, 0.0f, -kInf, -1, 0.0};

    // ---- the largest logit, and where it is first
    float top = -kInf;
    int place = 0;
    if (greedy) {
        s.pass(
            [&](int index, float x) KDA_INLINE {
                place = x > top ? index : place;
                top = fmaxf(top, x);
            },
            [](int) {});
    } else {
        s.pass([&](int, float x) KDA_INLINE { top = fmaxf(top, x); }, [](int) {});
        if (tid < 256) {
            sm.powers[tid] = exp2(tid * (1.0 / 256.0));
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
        s.row.least = kInf;
        s.row.most = 0.0f;
        top = 0.0f;
    }
    s.top = top;
    s.scale = kLog2e / static_cast<double>(temperature);
    s.bin_scale = static_cast<float>(static_cast<double>(kBins - 1) / (static_cast<double>(temperature) * kLn2 * (a.shift + 2)));
    const float min_p = a.min_p != nullptr ? a.min_p[n] : 0.0f;
    s.least_weight = min_p > 0.0f ? static_cast<double>(fminf(min_p, 1.0f)) : 0.0;
    const float top_p = a.top_p != nullptr ? a.top_p[n] : 1.0f;
    const bool nucleus = top_p < 1.0f;
    const int64_t k = a.top_k == nullptr          ? 0
                      : (a.top_k_int64 != 0) ? static_cast<const int64_t *>(a.top_k)[n]
                                             : static_cast<const int32_t *>(a.top_k)[n];
    const bool few_k = k > 0 && k < a.vocab;
    const float given = a.uniforms[n];
    const double u = given > 0.0f ? static_cast<double>(given) : 0.0;

    if (a.vocab <= kFew || (few_k && k <= kFewK)) {
        // ---- candidates: what reaches the k-th largest of the threads' maxima
        uint32_t bound = 0;
        if (a.vocab > kFew) {
            const uint32_t own = s.row.value(mine) > -kInf ? key_of(s.row.value(mine)) : 0;
            for (uint32_t bit = 0x80000000u; bit >= (sizeof(T) == 4 ? 1u : 0x10000u); bit >>= 1) {
                bound |= __syncthreads_count(own >= (bound | bit)) >= k ? bit : 0;
            }
        }
        uint32_t low, high;
        const int count = s.gather([&](int, float x) KDA_INLINE { return x > -kInf && key_of(x) >= bound; }, low, high);
        if (count <= kFew) {
            s.sort_list(count);
            const u64 rank = tid < count ? sm.list[tid] : 0;
            bool in = tid < count && (!few_k || tid < k), high_enough = false;
            u64 w = in ? s.weight(of_key(static_cast<uint32_t>(rank >> 32)), high_enough) : 0;
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
            sort(sm, power_above(count));
            const u64 entry = sm.list[tid];
            w = tid < count && entry != 0 ? sm.weights[static_cast<uint32_t>(entry)] : 0;
            sum = block_scan(sm, w, total);
            const u64 target = exceeding(u, total);
            if (sum >= target && sum - w < target) {
                const int index = static_cast<int>(static_cast<uint32_t>(entry >> 32) ^ 0xffffffffu);
                const float x = s.row.value(Row<T>::element(row.raw(index), 0));
                *token = index;
                *logprob = static_cast<float>((s.exponent(x) + a.shift) * kLn2 - log(static_cast<double>(total)));
            }
            return;
        }
    }
    // ---- top_k's cut (numbers in bins), the nucleus' (masses in bins), the blocks' masses of what is left
    const auto kept = [&](int index, float x) KDA_INLINE -> u64 {
        bool reaches;
        const u64 w = s.weight(x, reaches);
        return reaches && s.passes(x, index) ? w : 0;
    };
    enum { kNumbers, kNucleus, kLeft };
    u64 mass;
    for (int mode = few_k ? kNumbers : nucleus ? kNucleus : kLeft;;) {
        if (mode != kLeft) {
            s.clear_bins();
        }
        mass = s.block_masses([&](int index, float x) KDA_INLINE -> u64 {
            if (mode == kNumbers) {
                if (x > -kInf) {
                    atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[s.bin(x)]), 1ull);
                }
                return 0;
            }
            bool reaches;
            const u64 w = s.weight(x, reaches);
            if (w == 0 || !s.passes(x, index)) {
                return 0;
            }
            if (mode == kNucleus) {
                atomicAdd(reinterpret_cast<unsigned long long *>(&sm.bins[s.bin(x)]), static_cast<unsigned long long>(w));
            }
            return reaches ? w : 0;
        });
        if (mode == kLeft) {
            break;
        }
        u64 all;
        block_scan(sm, sm.bins[2 * tid] + sm.bins[2 * tid + 1], all);
        const u64 target = mode == kNumbers ? static_cast<u64>(k) : reaching(static_cast<double>(top_p), all);
        const bool cuts = mode == kNumbers ? target < all : target < mass;  // else min_p cuts what the nucleus would
        if (cuts) {
            s.cut(target, mode == kNumbers);
        } else if (mode == kNucleus) {
            break;
        }
        mode = mode == kNumbers && nucleus ? kNucleus : kLeft;
    }
    const int found = s.locate(exceeding(u, mass), kept);
    if (tid == 0) {
        const float x = s.row.value(Row<T>::element(row.raw(found), 0));
        *token = found;
        *logprob = static_cast<float>((s.exponent(x) + a.shift) * kLn2 - log(static_cast<double>(mass)));
    }
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
    if (a.dtype == KDA_BF16) {
        sample_kernel<uint16_t><<<rows, kThreads, 0, s>>>(a);
    } else {
        sample_kernel<float><<<rows, kThreads, 0, s>>>(a);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}
