// paged_attention.hip -- attention of new tokens over a paged key/value cache, gfx950.
//
// The query heads of a key head share its keys, so a request's new tokens and
// their G = heads / kv_heads query heads of one key head are the rows of one
// matrix: row r is token r / G, head r % G. Both kernels form S^T = K Q^T and
// O^T = V^T P^T, so that a lane owns a row of the softmax (a column of the
// tiles): the running maximum and sum need no LDS, and the scores that a lane
// holds after the first product are, in their order, the operand it must supply
// to the second. V^T comes from the row-major V tile in LDS through the
// transposing read (ds_read_b64_tr_b16).
//
//   decode_kernel   few rows a request (at most 32): HBM-bound on the keys and
//                   values, split over the keys
//   prefill_kernel  many rows: bound by the matrix cores and the softmax's
//                   vector instructions
//   *_combine       join the parts of rows whose keys were split
//
// Softmax in powers of two: c = |scale| log2(e) k_scale is one factor of the
// score (its sign goes into q), the weights are 2^(c s - m). m is raised only when
// a score of its own row passes it by 2^8: the weights then stay below 2^8, far inside fp32 and
// bf16, and the accumulators are rescaled a few times a row instead of every
// tile. (A row that another one's raise took along would round its weights by keys that it does not
// see. The choice per row costs nothing: six chunks over up to 30 K keys 844 us either way.)
// Scores, m, the sums and O are fp32. The weights are rounded to bf16 for the
// second product, and the sum takes them rounded too: numerator and denominator
// then err alike, and a dot product sums two at a time.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kda_abi.h"
#include "kda_device.h"
#include "paged_cache.h"

namespace kda {
namespace {

// The kernels' lambdas belong into them: called, the arrays they work on would go through memory.
#define KDA_INLINE __attribute__((always_inline))

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kCus = 256;  // of an MI355X: only the number of workgroups goes by it
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kRaise = 8.0f;  // log2 of the largest weight before m is raised
// m of a row that sees keys, all with a score of -inf: below every other score's, so that parts of the row are
// joined as ever, and told from -inf, m of a row that sees none. The first row's result is 0 / 0 = NaN as the
// softmax's is, the second one's 0.
constexpr float kLowest = -3e38f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const __attribute__((address_space(1))) u32x4 global_u32x4;
typedef const __attribute__((address_space(1))) int global_int;

struct __attribute__((packed, aligned(2))) Bf16x8Any {
    u32x4 w;
};

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
// A 16-byte load that is known to be from global memory: through a selected or shuffled
// pointer the compiler would issue a flat load, which also counts as an LDS access and is waited for as one.
__device__ __forceinline__ u32x4 load16(const char *p) { return *(global_u32x4 *)p; }
// of data read once: 64 ragged decode requests 620 -> 565 us with their values read so
__device__ __forceinline__ u32x4 load16_stream(const char *p) { return __builtin_nontemporal_load((global_u32x4 *)p); }

// 64 x 16 bytes from memory into 1 KiB of LDS in lane order (`to` is the wave's), without
// registers. Written as assembly because the compiler makes every later LDS read wait for the builtin's loads,
// of whichever buffer; here whoever reads them waits for vmcnt and the barrier first.
// Several KiB: a base the wave shares, each lane's offsets, and for the i-th KiB i * 1024 on both addresses.
template <int N> __device__ __forceinline__ void load16_to_lds(const char *from, const uint32_t (&at)[N], char *to) {
    static_assert(N == 2 || N == 4);
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)to));
    if constexpr (N == 4) {
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024\n\t"
            "global_load_lds_dwordx4 %3, %5 offset:2048\n\tglobal_load_lds_dwordx4 %4, %5 offset:3072"
            :
            : "s"(lds), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "s"(from)
            : "m0", "memory");
    } else {
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024"
            :
            : "s"(lds), "v"(at[0]), "v"(at[1]), "s"(from)
            : "m0", "memory");
    }
}
__device__ __forceinline__ void load16_to_lds(const char *from, char *to) {
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(from) : "m0", "memory");
}

// sum + both bf16 of a pair, in fp32
__device__ __forceinline__ float add_pair(uint32_t pair, float sum) {
    constexpr uint32_t kOnes = 0x3f803f80u;
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, kOnes), sum, false);
}

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// Infinite or NaN values that some rows of a tile do not see must not reach those, but in the matrix
// product their weight of 0 makes a NaN. The steps do not look for them. A tile whose O is not finite at its end,
// and whose rows do not all see the same keys, is formed again from values with 0 in those places, and
// then they are added to the rows that see them.
__device__ __forceinline__ u32x4 finite_only(u32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // the sign bit's place of each bf16 whose exponent is all ones
        const uint32_t t = ((v[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        v[i] &= ~((t - (t >> 15)) | t);
    }
    return v;
}
template <bool FP8> __device__ __forceinline__ bool any_not_finite(u32x4 v) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t |= FP8 ? ((v[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((v[i] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    }
    return t != 0;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < __builtin_inff(); }
// Column c of a row of values where it is infinite or NaN, else 0.
template <bool FP8> __device__ __forceinline__ float not_finite(const char *row, int c) {
    float x;
    if constexpr (FP8) {
        x = (reinterpret_cast<const uint8_t *>(row)[c] & 0x7f) == 0x7f ? __builtin_nanf("") : 0.0f;
    } else {
        x = __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(row)[c]) << 16);
    }
    return is_finite(x) ? 0.0f : x;
}

// Sixteen e4m3 (16 bytes) as bf16, exactly (three mantissa bits): two operands of 8.
__device__ __forceinline__ void fp8_to_bf16(u32x4 x, u32x4 &lo, u32x4 &hi) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        lo[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.0f, false));
        lo[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.0f, true));
        hi[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 + i], 1.0f, false));
        hi[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 + i], 1.0f, true));
    }
}

// Maxima and sums over lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The same over the four groups of 16 lanes.
__device__ __forceinline__ float max_groups(float x) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_groups(float x) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// cap tanh(s / cap) in log2 units; x = 2 log2(e) s / cap, cap2 = cap log2(e). tanh = 1 - 2 / (e^(2s/cap) + 1):
// infinities give +-1, NaN stays. Its error is an ulp of the cap, too much where the cap is far above the
// scores: below a tenth of it the series t - t^3/3 + 2t^5/15, whose next term is under 6e-8 of it. (3% of a
// capped verify step's time; a branch for large caps only would cost every prefill 3%.)
__device__ __forceinline__ float capped(float x, float cap2) {
    const float t = x * (0.5f / kLog2e), t2 = t * t;
    const float low = cap2 * t * (1.0f - t2 * (1.0f / 3.0f - t2 * (2.0f / 15.0f)));
    return t2 < 0.01f ? low : cap2 - 2.0f * cap2 * __builtin_amdgcn_rcpf(ex2(x) + 1.0f);
}

constexpr int kDppQuadEven = 0xA0, kDppQuadOdd = 0xF5;  // quad_perm [0,0,2,2] and [1,1,3,3]

// Rows of zeros that stand for keys outside a request or pages outside the pool.
__device__ const u32x4 g_zero_row[16] = {};

struct Request {
    int begin;   // first token in q
    int tokens;  // new tokens
    int keys;    // keys in the cache, the new tokens' among them
};

struct PageWords {
    const char *row;
    uint32_t step;  // bytes
    __device__ __forceinline__ int of(int at) const {
        return *(global_int *)(row + static_cast<uint64_t>(static_cast<uint32_t>(at)) * step);
    }
};
// The page of an entry of these words: any number, which callers compare with the pool. -1 for one beyond 32 bits.
__device__ __forceinline__ int page_of(int first, int last) { return last != 0 ? -1 : first; }

struct Params : KdaPagedAttentionArgs {
    int group;  // query heads a key head

    // Token ranges and lengths cut to the tensors, whatever the metadata says: int64 entries as they are, not
    // their low words.
    __device__ __forceinline__ int cut(const void *p, int64_t i, int bit, int most) const {
        if ((wide & bit) == 0) {
            return min(max(static_cast<const int32_t *>(p)[i], 0), most);
        }
        return static_cast<int>(min(max(static_cast<const int64_t *>(p)[i], INT64_C(0)), static_cast<int64_t>(most)));
    }
    __device__ __forceinline__ int cu(int n) const { return cut(cu_seqlens, n, KDA_WIDE_CU_SEQLENS, num_tokens); }
    __device__ __forceinline__ Request request(int n) const {
        const int keys = max_pages * cache.page_size;
        if ((wide & (KDA_WIDE_CU_SEQLENS | KDA_WIDE_KV_LENS)) == 0) {  // one branch for three loads in flight together
            const int32_t *c = static_cast<const int32_t *>(cu_seqlens) + n;
            const int begin = min(max(c[0], 0), num_tokens), end = min(max(c[1], 0), num_tokens);
            return Request{begin, max(end - begin, 0), min(max(static_cast<const int32_t *>(kv_lens)[n], 0), keys)};
        }
        const int begin = cu(n);
        return Request{begin, max(cu(n + 1) - begin, 0), cut(kv_lens, n, KDA_WIDE_KV_LENS, keys)};
    }
    // Keys visible to the i-th new token: [x, y)
    __device__ __forceinline__ int2 visible(const Request &r, int i) const {
        const int end = max(r.keys - r.tokens + i + 1, 0);
        return make_int2(window > 0 ? max(end - window, 0) : 0, end);
    }
    // Request n's page table as a lane reads it: the entries' first words, or (`last`) the second ones of int64
    // entries, 0 for int32 ones. Looked up ahead by lanes that share an entry, one word each: one register a
    // lane, nothing waits for the load, and page_of puts them together.
    __device__ __forceinline__ PageWords page_words(int n, bool last) const {
        const bool both = (wide & KDA_WIDE_PAGE_TABLE) != 0;
        const char *row = static_cast<const char *>(page_table) + ((n * page_table_stride) << (both ? 3 : 2));
        return PageWords{last && !both ? reinterpret_cast<const char *>(g_zero_row) : row + (last ? 4 : 0),
                         both ? 8u : last ? 0u : 4u};
    }
    // The row of values of one of request n's keys, null on a page outside the pool.
    template <bool FP8> __device__ __forceinline__ const char *value_row(int n, int head, int key) const {
        const int at = key / cache.page_size;
        const int page = page_of(page_words(n, false).of(at), page_words(n, true).of(at));
        const int64_t offset = page * cache.v_stride_page + key % cache.page_size * cache.v_stride_token + head * cache.v_stride_head;
        return static_cast<uint32_t>(page) < static_cast<uint32_t>(cache.num_pages)
                   ? static_cast<const char *>(cache.v) + (FP8 ? offset : 2 * offset)
                   : nullptr;
    }
};

// A kernel's only argument, read again: what is needed only after a long loop would otherwise be kept in
// scalar registers through it, of which the loop has none to spare.
template <class T> __device__ __forceinline__ const T &arguments_again(const T &) {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const T *)p;
}

// Factor of the scores in log2 units, and what the capped form needs. The sign
// of scale * k_scale goes into q, so the largest score is the largest product.
struct Scores {
    float c;     // of the products, not capped
    float cap;   // cap log2(e), 0: none
    float in;    // 2 log2(e) / cap times the score's factor
    uint32_t flip;
};
__device__ __forceinline__ Scores scores_of(const Params &a, int head) {
    const float ks = a.cache.k_scale != nullptr ? a.cache.k_scale[head] : 1.0f;
    const float f = a.scale * ks;
    Scores s;
    s.flip = f < 0.0f ? 0x80008000u : 0u;
    // never 0: a masked score is -inf and stays it
    const float mag = fabsf(f) < 1e-30f ? 1e-30f : fabsf(f);
    s.c = mag * kLog2e;
    s.cap = a.logit_cap * kLog2e;
    const float in = 2.0f * kLog2e * mag / a.logit_cap;
    s.in = a.logit_cap > 0.0f ? (in > 3e38f ? 3e38f : in) : 0.0f;  // finite: a score of 0 stays 0; but a NaN stays one
    return s;
}

// A row of the cache: D elements, 16-byte chunks.
template <int D, bool FP8> struct Row {
    static constexpr int kBytes = FP8 ? D : 2 * D;
    static constexpr int kLanes = kBytes / 16;   // lanes that load a row
    static constexpr int kRows = 64 / kLanes;    // rows a wave loads at a time
    static constexpr int kShift = FP8 ? 0 : 1;   // bytes of an element, log2
};

// LDS tiles of bf16 rows of D, without padding. Chunks of 16 bytes are permuted
// within 256 bytes (one row of 128 or two of 64) by the row, so that the reads of
// one column over 16 rows touch all banks alike.
// K: chunk reads. V: transposing reads of 32-byte pairs of chunks, which stay together.
// k_chunk, v_chunk: the slot of a chunk, and the chunk at a slot.
template <int D> __device__ __forceinline__ int k_chunk(int row, int slot) {
    return slot ^ (D == 128 ? row & 15 : (row >> 1) & 7);
}
template <int D> __device__ __forceinline__ int v_chunk(int row, int slot) {
    // 32 lanes of a transposing read take 4 neighbouring rows and two neighbouring pairs, or 8 rows and one
    // pair: eight different 32-byte places of the 256 bytes either way
    return slot ^ (D == 128 ? (row & 3) << 2 | (row & 4) >> 1 : (row & 2) << 1 | (row & 4) >> 1);
}
template <int D> __device__ __forceinline__ int k_at(int row, int chunk) {
    return row * 2 * D + (k_chunk<D>(row, chunk) << 4);
}
template <int D> __device__ __forceinline__ int v_at(int row, int chunk) {
    return row * 2 * D + (v_chunk<D>(row, chunk) << 4);
}
// Transposing read of rows row .. row + 3 (16 lanes: lane 4m + c takes row m), columns
// 16 pair .. 16 pair + 15: lane i of the 16 gets column i of the four rows.
template <int D> __device__ __forceinline__ u32x2 read_tr(const char *tile, int row, int pair, int lane) {
    const int r = row + ((lane >> 2) & 3);
    const int c = lane & 3;
    const char *p = tile + v_at<D>(r, 2 * pair + (c >> 1)) + (c & 1) * 8;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
}

// A 16-byte chunk of a loaded row into a tile, 8-bit ones widened to two chunks.
template <int D, bool FP8, class At>
__device__ __forceinline__ void stage(char *tile, int row, int chunk, u32x4 x, At at) {
    if constexpr (FP8) {
        u32x4 lo, hi;
        fp8_to_bf16(x, lo, hi);
        *reinterpret_cast<u32x4 *>(tile + at(row, 2 * chunk)) = lo;
        *reinterpret_cast<u32x4 *>(tile + at(row, 2 * chunk + 1)) = hi;
    } else {
        *reinterpret_cast<u32x4 *>(tile + at(row, chunk)) = x;
    }
}

__device__ __forceinline__ u32x4 load_q(const Params &a, int64_t token, int head, int d, uint32_t flip) {
    const uint16_t *p =
        static_cast<const uint16_t *>(a.q) + token * a.q_stride_token + head * a.q_stride_head + d;
    return reinterpret_cast<const Bf16x8Any *>(p)->w ^ flip;
}

// The first request after n that has new tokens, or num_seqs: 64 at a time, in every lane of a wave.
__device__ __forceinline__ int next_request(const Params &a, int n) {
    for (int first = n + 1; first < a.num_seqs; first += 64) {
        const int x = min(first + static_cast<int>(__lane_id()), a.num_seqs - 1);
        const unsigned long long some = __ballot(a.cu(x + 1) > a.cu(x));
        if (some != 0) {
            return __builtin_amdgcn_readfirstlane(first + __ffsll(some) - 1);
        }
    }
    return a.num_seqs;
}

// f(key, row of values) for the keys in [lo, hi) of a request whose values are not all finite; by a whole wave.
template <int D, bool FP8, class F>
__device__ __forceinline__ void each_not_finite(const Params &a, int n, int head, int lo, int hi, F f) {
    for (int key0 = lo; key0 < hi; key0 += 64) {
        const int key = key0 + static_cast<int>(__lane_id());
        const char *row = key < hi ? a.value_row<FP8>(n, head, key) : nullptr;
        bool some = false;
        if (row != nullptr) {
            for (int c = 0; c < Row<D, FP8>::kBytes; c += 16) {
                some |= any_not_finite<FP8>(load16(row + c));
            }
        }
        for (unsigned long long left = __ballot(some); left != 0; left &= left - 1) {
            const int found = key0 + __ffsll(left) - 1;
            f(found, a.value_row<FP8>(n, head, found));
        }
    }
}

// Tokens that no request covers: zeros, spread over the grid.
template <int D> __device__ __forceinline__ void zero_uncovered(const Params &a, int64_t block, int64_t blocks) {
    const int64_t begin = a.cu(0), end = max(a.cu(a.num_seqs), a.cu(0));
    const int64_t count = begin + (a.num_tokens - end);
    for (int64_t i = block; i < count; i += blocks) {
        const int64_t t = i < begin ? i : end + (i - begin);
        for (int e = threadIdx.x; e < a.num_heads * D; e += kThreads) {
            static_cast<uint16_t *>(a.out)[t * a.out_stride_token + (e / D) * a.out_stride_head + e % D] = 0;
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows: decode and verify steps.
//
// An item is a (request, key head, tile of 16 NB rows); its keys are cut at
// multiples of 128 (a unit: 32 keys a wave). The units of all items in order are
// dealt out evenly to the workgroups, whatever the lengths are: each takes
// one contiguous range, which may begin and end inside an item. Every
// workgroup finds its range itself from the lengths (a prefix sum over the
// requests), so the call needs no host knowledge of them. An item inside one
// range is finished there; the parts of the others are joined by
// decode_combine_kernel, always in the same order.
//
// The waves are independent within an item: each streams its own 32-key blocks
// through registers into 32 rows of keys and 32 of values in LDS, whole rows at a time and
// past the caches (they are read once). The next block's loads (16 KiB a wave in
// bf16 at D = 128) are in flight while one is computed, the page numbers one block
// further ahead. Keys loaded straight into the operands' registers would skip LDS, but
// a lane's 16 bytes of 16 different rows waste the memory's bursts: 64 ragged
// requests of up to 32 K keys took 565 us so, 552 now.
//
// Bound by HBM: those 64 requests (64 heads on 8 key heads, D = 128) read 3.4 GB in
// 552 us = 6.1 TB/s, what a kernel that only reads reaches (other cards: up to 577 us).
// D = 64: 311 us for half of it, 5.4 TB/s. 256 requests in 8 bits:
// 169 us = 5.6 TB/s, 5 us of it for joining parts. A single short request is bound by its
// latencies: 9 to 10 us for the kernel (lengths, page numbers, keys, the waves' join one after another) and
// 4 us for the second one.
// ---------------------------------------------------------------------------

constexpr int kUnit = 128;
constexpr int kBlock = 32;
constexpr int kDecodeGroups = 2 * kCus;

struct DecodeWs {
    float *o;     // [2 groups][rows][D]: a workgroup's part that continues an item, its part that begins one
    float2 *ml;   // [2 groups][rows]
    int4 *desc;   // [groups]: the item that begins in a workgroup and does not end there: its request's first
                  // token, its first row of the request, rows (0: no such item) + 256 key head, last workgroup
};

template <int D, int NB> struct DecodeShared {
    char k[kWaves][kBlock * D * 2];  // keys of a wave's block
    char v[kWaves][kBlock * D * 2];  // values; 16 rows of O when waves join
    float2 ml[kWaves][16 * NB];
    int scan[kWaves];
    int first, before;  // the request of the range's first unit, and the first unit of that request
    Request request;
};

// Units of a tile of `rows` rows of a request: the most that any of its tiles has.
__device__ __forceinline__ int tile_units(const Params &a, const Request &r, int rows) {
    int units = (r.keys + kUnit - 1) / kUnit;
    if (a.window > 0) {
        const int64_t tokens = (rows + a.group - 2) / a.group + 1;  // that a tile may touch
        const int64_t span = a.window + tokens - 1;                 // keys that they see
        const int64_t most = (span + kUnit - 2) / kUnit + 1;
        units = static_cast<int>(min(static_cast<int64_t>(units), most));
    }
    return max(units, 1);  // an item without keys still writes its zeros
}

template <int D, bool FP8, int NB>
__global__ __launch_bounds__(kThreads, 2) void decode_kernel(const Params a, const DecodeWs ws) {
    constexpr int kRows = 16 * NB;
    using R = Row<D, FP8>;
    constexpr int kLoads = kBlock / R::kRows;  // 16-byte loads of a block's keys or values a lane makes
    __shared__ __attribute__((aligned(16))) DecodeShared<D, NB> sm;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4;
    const int col = lane & 15;
    const int heads = a.cache.kv_heads;

    zero_uncovered<D>(a, blockIdx.x, gridDim.x);

    // ---- this workgroup's range of units
    const int per = (a.num_seqs + kThreads - 1) / kThreads;
    const int n0 = min(tid * per, a.num_seqs), n1 = min(n0 + per, a.num_seqs);
    auto units_of = [&](const Request &r) { return (r.tokens * a.group + kRows - 1) / kRows * heads * tile_units(a, r, kRows); };
    int mine = 0;
    bool bad = false;  // token offsets that decrease: requests overlap, and their units may not fit 32 bits
    for (int n = n0; n < n1; ++n) {
        mine += units_of(a.request(n));
        bad |= a.cu(n) > a.cu(n + 1);
    }
    int scan = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(scan, d);
        scan += lane >= d ? up : 0;
    }
    if (lane == 63) {
        sm.scan[wave] = scan;
    }
    if (__any(bad)) {
        sm.scan[wave] = -1;
    }
    __syncthreads();
    int total = 0, base = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        base += w < wave ? sm.scan[w] : 0;
        total += sm.scan[w];
        bad |= sm.scan[w] < 0;
    }
    total = __builtin_amdgcn_readfirstlane(bad ? 0 : total);
    const int w = blockIdx.x;
    const int groups = min(static_cast<int>(gridDim.x), total);
    if (w >= groups) {
        if (tid == 0) {
            ws.desc[w] = make_int4(0, 0, 0, 0);
        }
        return;
    }
    const int share = total / groups, more = total - share * groups;  // the first `more` workgroups take one unit more
    const int u0 = w * share + min(w, more), u1 = u0 + share + (w < more ? 1 : 0);
    int at = base + scan - mine;
    if (u0 >= at && u0 < at + mine) {  // one thread's requests hold the first unit
        int n = n0;
        Request r = a.request(n);
        for (int u = units_of(r); u0 >= at + u; u = units_of(r)) {
            at += u;
            r = a.request(++n);
        }
        sm.first = n;
        sm.before = at;
        sm.request = r;
    }
    __syncthreads();
    int n = __builtin_amdgcn_readfirstlane(sm.first);
    int start = __builtin_amdgcn_readfirstlane(sm.before);  // the first unit of request n
    Request req = {__builtin_amdgcn_readfirstlane(sm.request.begin), __builtin_amdgcn_readfirstlane(sm.request.tokens),
                   __builtin_amdgcn_readfirstlane(sm.request.keys)};
    int4 desc = make_int4(0, 0, 0, 0);

    for (int u = u0; u < u1;) {
        const int rows_all = req.tokens * a.group;
        const int tiles = (rows_all + kRows - 1) / kRows;
        const int count = tile_units(a, req, kRows);
        if (u >= start + tiles * heads * count) {
            start += tiles * heads * count;
            n = next_request(a, n);
            req = a.request(n);
            continue;
        }
        // ---- the item and the part of it that is in this range
        const int item = (u - start) / count;
        const int part0 = u - start - item * count;
        const int part1 = min(count, part0 + (u1 - u));
        const int head = item / tiles;
        const int tile = item - head * tiles;
        const int row0 = tile * kRows;
        const int rows = min(kRows, rows_all - row0);
        const int2 first = a.visible(req, row0 / a.group);
        const int2 last = a.visible(req, (row0 + rows - 1) / a.group);
        const int unit0 = first.x / kUnit;
        const int lo = max(first.x, (unit0 + part0) * kUnit);  // keys of this part: [lo, hi)
        const int hi = min(last.y, (unit0 + part1) * kUnit);
        const Scores sc = scores_of(a, head);

        // ---- queries: 16 rows a block as the right operand
        u32x4 q[NB][D / 32];
        int2 see[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int r = min(b * 16 + col, rows - 1);
            const int t = (row0 + r) / a.group;
            const int h = head * a.group + (row0 + r) - t * a.group;
            see[b] = a.visible(req, t);
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                q[b][s] = load_q(a, req.begin + t, h, s * 32 + g * 8, sc.flip);
            }
        }
        f32x4 o[NB][D / 16];
        float m[NB], l[NB];

        // ---- this wave's blocks of 32 keys: key0 + 128 i
        const int key0 = (unit0 + part0) * kUnit + wave * kBlock;
        const int blocks = hi > key0 ? (hi - key0 + kUnit - 1) / kUnit : 0;
        const char *kbase = static_cast<const char *>(a.cache.k) + ((head * a.cache.k_stride_head) << R::kShift);
        const char *vbase = static_cast<const char *>(a.cache.v) + ((head * a.cache.v_stride_head) << R::kShift);
        auto lookup = [&](int i) KDA_INLINE -> int {  // page of key lane % 32 of block i; any entry where it has none
            int lane = static_cast<int>(__lane_id());
            if constexpr (NB > 1) {  // as in compute: the entry's word in no register of its own
                asm volatile("" : "+v"(lane));
            }
            const int key = key0 + i * kUnit + (lane & 31);
            return a.page_words(n, lane >= 32).of(min(max(key, 0) / a.cache.page_size, a.max_pages - 1));
        };
        // keys of a block that every row of the tile sees: [seen0, seen1)
        const int seen0 = max(lo, last.x), seen1 = min(hi, first.y);
        struct Rows {
            unsigned long long k, v;  // the rows of key lane % 32 of a block
        };
        auto rows_of = [&](int i, int word) KDA_INLINE -> Rows {
            const u32x2 words = __builtin_amdgcn_permlane32_swap(word, word, false, false);
            const int page = page_of(words[0], words[1]);
            const int key = key0 + i * kUnit + (lane & 31);
            const int off = key - key / a.cache.page_size * a.cache.page_size;
            const bool real = key >= lo && key < hi && static_cast<uint32_t>(page) < static_cast<uint32_t>(a.cache.num_pages);
            const char *kp = kbase + ((page * a.cache.k_stride_page + off * a.cache.k_stride_token) << R::kShift);
            const char *vp = vbase + ((page * a.cache.v_stride_page + off * a.cache.v_stride_token) << R::kShift);
            const char *zero = reinterpret_cast<const char *>(g_zero_row);
            return Rows{reinterpret_cast<unsigned long long>(real ? kp : zero), reinterpret_cast<unsigned long long>(real ? vp : zero)};
        };
        u32x4 k[kLoads], v[kLoads];
        auto load = [&](const Rows &rows) KDA_INLINE {
#pragma unroll
            for (int s = 0; s < kLoads; ++s) {
                const int from = s * R::kRows + lane / R::kLanes;
                k[s] = load16_stream(reinterpret_cast<const char *>(__shfl(rows.k, from)) + lane % R::kLanes * 16);
                v[s] = load16_stream(reinterpret_cast<const char *>(__shfl(rows.v, from)) + lane % R::kLanes * 16);
            }
        };
        bool again = false;
        // block i, whose rows are in k and v; the next one's are asked for as soon as these are in LDS
        auto compute = [&](int i, const Rows &next) KDA_INLINE {
            char *kt_ = sm.k[wave], *vt = sm.v[wave];
            int lane = static_cast<int>(__lane_id());
            if constexpr (NB > 1) {  // addresses in LDS formed anew for each block: kept, they do not all fit the registers
                asm volatile("" : "+v"(lane));
            }
            const int col = lane & 15, g = lane >> 4;
#pragma unroll
            for (int x = 0; x < kLoads; ++x) {
                const int r = x * R::kRows + lane / R::kLanes;
                stage<D, FP8>(kt_, r, lane % R::kLanes, k[x], [](int r, int c) { return k_at<D>(r, c); });
                stage<D, FP8>(vt, r, lane % R::kLanes, v[x], [](int r, int c) { return v_at<D>(r, c); });
            }
            if (again) {
#pragma unroll
                for (int x = 0; x < kBlock * 2 * D / 1024; ++x) {
                    u32x4 *p = reinterpret_cast<u32x4 *>(vt + x * 1024 + lane * 16);
                    *p = finite_only(*p);
                }
            }
            load(next);
            __builtin_amdgcn_sched_barrier(0);
            f32x4 s[NB][2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    s[b][kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    const u32x4 op = *reinterpret_cast<const u32x4 *>(kt_ + k_at<D>(kt * 16 + col, 4 * x + g));
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        s[b][kt] = mfma16(op, q[b][x], s[b][kt]);
                    }
                }
            }
            // a lane's scores: row `col`, keys 16 kt + 4 g + e
            const int first_key = key0 + i * kUnit;
            const float c = sc.cap > 0.0f ? 1.0f : sc.c;
            if (sc.cap > 0.0f) {
#pragma unroll
                for (int e = 0; e < NB * 8; ++e) {
                    s[e >> 3][e >> 2 & 1][e & 3] = capped(s[e >> 3][e >> 2 & 1][e & 3] * sc.in, sc.cap);
                }
            }
            if (first_key < seen0 || first_key + kBlock > seen1) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int from = max(see[b].x, lo) - first_key - 4 * g, to = min(see[b].y, hi) - first_key - 4 * g;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = 16 * (e >> 2) + (e & 3);
                        s[b][e >> 2][e & 3] = key >= from && key < to ? s[b][e >> 2][e & 3] : kNegInf;
                    }
                }
            }
            u32x4 p[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float top = kNegInf;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    top = fmaxf(top, s[b][e >> 2][e & 3]);
                }
                top = max_groups(top) * c;
                const bool raise = top > m[b] + kRaise;
                if (__any(raise)) {
                    const float up = raise ? top : m[b];
                    const float f = up == m[b] ? 1.0f : ex2(m[b] - up);
                    m[b] = up;
                    l[b] *= f;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        o[b][d] *= f;
                    }
                }
                const float base = m[b] == kNegInf ? 0.0f : m[b];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int kt = e >> 1;
                    p[b][e] = pack_bf16x2(ex2(s[b][kt][2 * (e & 1)] * c - base), ex2(s[b][kt][2 * (e & 1) + 1] * c - base));
                    l[b] = add_pair(p[b][e], l[b]);
                }
            }
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                const u32x2 v0 = read_tr<D>(vt, 4 * g, d, lane);
                const u32x2 v1 = read_tr<D>(vt, 16 + 4 * g, d, lane);
                const u32x4 op = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    o[b][d] = mfma16(op, p[b], o[b][d]);
                }
            }
        };
        for (;; again = true) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                m[b] = kNegInf;
                l[b] = 0.0f;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    o[b][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
            if (blocks > 0) {
                // past the last block rows of zeros are loaded
                Rows rows = rows_of(0, lookup(0));
                int word = lookup(1);
                load(rows);
                for (int i = 0; i < blocks; ++i) {
                    rows = rows_of(i + 1, word);
                    word = lookup(i + 2);
                    compute(i, rows);
                }
            }
            if (again || (first.x == last.x && first.y == last.y)) {
                break;
            }
            bool fine = true;  // where a score is NaN the whole row is
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        fine &= is_finite(o[b][d][e]) || l[b] != l[b];
                    }
                }
            }
            if (__all(fine)) {
                break;
            }
        }
        if (again) {
            each_not_finite<D, FP8>(a, n, head, lo, hi, [&](int key, const char *row) KDA_INLINE {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (key % kUnit / kBlock == wave && key >= see[b].x && key < see[b].y) {
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                o[b][d][e] += not_finite<FP8>(row, 16 * d + 4 * g + e);
                            }
                        }
                    }
                }
            });
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = see[b].x < see[b].y ? fmaxf(m[b], kLowest) : m[b];
        }
        // ---- join the waves: their maxima, sums and 16 rows of O at a time through LDS
        const bool begins = part0 == 0, ends = part1 == count;
        const int64_t slot = 2 * static_cast<int64_t>(w) + (begins ? 1 : 0);
        if (begins && !ends) {
            const int end = start + item * count + count - 1;  // its last unit, and that unit's workgroup
            const int wide = more * (share + 1);
            desc = make_int4(req.begin, row0, rows + 256 * head, end < wide ? end / (share + 1) : more + (end - wide) / share);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float sum = sum_groups(l[b]);
            if (g == 0) {
                sm.ml[wave][b * 16 + col] = make_float2(m[b], sum);
            }
        }
        const float vs = a.cache.v_scale != nullptr ? a.cache.v_scale[head] : 1.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            // 16 rows of D floats take a wave's 32 rows of D bf16
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {  // 16-byte chunks, permuted by the row against bank conflicts
                const int chunk = (4 * d + g) ^ (D == 128 ? col : col & 7);
                *reinterpret_cast<f32x4 *>(sm.v[wave] + col * D * 4 + chunk * 16) = o[b][d];
            }
            __syncthreads();
            const int r = tid >> 4;  // 16 threads a row
            float2 ml[kWaves];
            float top = kNegInf;
#pragma unroll
            for (int x = 0; x < kWaves; ++x) {
                ml[x] = sm.ml[x][b * 16 + r];
                top = fmaxf(top, ml[x].x);
            }
            float sum = 0.0f, f[kWaves];
#pragma unroll
            for (int x = 0; x < kWaves; ++x) {
                f[x] = ml[x].x == top ? 1.0f : ex2(ml[x].x - top);
                sum += ml[x].y * f[x];
            }
            const float norm = begins && ends ? (top == kNegInf ? 0.0f : vs / sum) : 1.0f;
            const int t = (row0 + b * 16 + r) / a.group;
            const int h = head * a.group + (row0 + b * 16 + r) - t * a.group;
#pragma unroll
            for (int x = 0; x < D / 64; ++x) {
                const int c = (tid & 15) + 16 * x;
                const int chunk = c ^ (D == 128 ? r : r & 7);
                f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < kWaves; ++k) {
                    y += *reinterpret_cast<const f32x4 *>(sm.v[k] + r * D * 4 + chunk * 16) * f[k];
                }
                y *= norm;
                if (b * 16 + r < rows) {
                    if (begins && ends) {
                        uint16_t *out = static_cast<uint16_t *>(a.out) + (req.begin + t) * a.out_stride_token +
                                        h * a.out_stride_head + c * 4;
                        struct __attribute__((packed, aligned(2))) Out {
                            uint32_t w[2];
                        };
                        *reinterpret_cast<Out *>(out) = {{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])}};
                    } else {
                        *reinterpret_cast<f32x4 *>(ws.o + (slot * kRows + b * 16 + r) * D + c * 4) = y;
                    }
                }
            }
            if (!(begins && ends) && (tid & 15) == 0) {
                ws.ml[slot * kRows + b * 16 + r] = make_float2(top, sum);
            }
            __syncthreads();
        }
        u += part1 - part0;
    }
    if (tid == 0) {
        ws.desc[w] = desc;
    }
}

// Joins the items that began in a workgroup of decode_kernel and did not end there:
// gridDim.y workgroups each take every gridDim.y-th row. A workgroup's threads take 4 columns each, and
// the rows and the parts are spread over what is left of them, so that a
// thread's loads are few and in flight together (32 parts of 4 rows: 20.8 us with
// a thread to all parts of a row, one after another).

template <int D, int NB> __global__ __launch_bounds__(kThreads) void decode_combine_kernel(const Params a, const DecodeWs ws) {
    constexpr int kRows = 16 * NB;
    constexpr int kCols = D / 4;
    constexpr int kSlots = kThreads / kCols;
    __shared__ f32x4 sum_o[kThreads];
    __shared__ float2 sum_ml[kThreads];
    const int w = blockIdx.x;
    const int4 desc = ws.desc[w];
    const int step = gridDim.y;
    const int rows = ((desc.z & 255) - static_cast<int>(blockIdx.y) + step - 1) / step;  // of this workgroup
    if (rows <= 0) {
        return;
    }
    const int head = desc.z >> 8;
    const int parts = desc.w - w + 1;  // the second slot of w, then the first ones of w + 1 .. last
    // threads of a row: a power of two, at most the parts, such that all rows are taken at once
    int lanes = 1;
    while (2 * lanes <= parts && 2 * lanes * rows <= kSlots) {
        lanes *= 2;
    }
    const int c = threadIdx.x % kCols;
    const int slot = threadIdx.x / kCols;
    const int lane = slot & (lanes - 1);
    const float vs = a.cache.v_scale != nullptr ? a.cache.v_scale[head] : 1.0f;
    for (int first = 0; first < rows; first += kSlots / lanes) {
        const int i = first + slot / lanes;
        const int r = min(i, rows - 1) * step + blockIdx.y;
        float top = kNegInf, sum = 0.0f;
        f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int x = lane; x < parts; x += 4 * lanes) {
            float2 ml[4];
            f32x4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int part = min(x + k * lanes, parts - 1);
                const int64_t at = (2 * static_cast<int64_t>(w + part) + (part == 0 ? 1 : 0)) * kRows + r;
                ml[k] = ws.ml[at];
                o[k] = *reinterpret_cast<const f32x4 *>(ws.o + at * D + c * 4);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (x + k * lanes < parts) {
                    const float next = fmaxf(top, ml[k].x);
                    const float f0 = top == next ? 1.0f : ex2(top - next), f1 = ml[k].x == next ? 1.0f : ex2(ml[k].x - next);
                    top = next;
                    sum = sum * f0 + ml[k].y * f1;
                    y = y * f0 + o[k] * f1;
                }
            }
        }
        if (lanes > 1) {
            __syncthreads();  // the last round's values are read
            sum_o[threadIdx.x] = y;
            sum_ml[threadIdx.x] = make_float2(top, sum);
            __syncthreads();
            if (lane == 0) {
                for (int k = 1; k < lanes; ++k) {
                    const float2 ml = sum_ml[threadIdx.x + k * kCols];
                    const float next = fmaxf(top, ml.x);
                    const float f0 = top == next ? 1.0f : ex2(top - next), f1 = ml.x == next ? 1.0f : ex2(ml.x - next);
                    top = next;
                    sum = sum * f0 + ml.y * f1;
                    y = y * f0 + sum_o[threadIdx.x + k * kCols] * f1;
                }
            }
        }
        if (lane == 0 && i < rows) {
            y *= top == kNegInf ? 0.0f : vs / sum;
            const int row = desc.y + r;
            const int t = row / a.group;
            const int h = head * a.group + row - t * a.group;
            uint16_t *out = static_cast<uint16_t *>(a.out) + static_cast<int64_t>(desc.x + t) * a.out_stride_token +
                            h * a.out_stride_head + c * 4;
            struct __attribute__((packed, aligned(2))) Out {
                uint32_t w[2];
            };
            *reinterpret_cast<Out *>(out) = {{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])}};
        }
    }
}

// ---------------------------------------------------------------------------
// Many rows: prefill chunks and long verify steps.
//
// A workgroup takes a tile of 128 rows of one (request, key head), 32 a
// wave, and walks the visible keys in tiles of 64. The four waves share a key and
// a value tile in LDS, two of each, so one barrier a tile is enough. While one is
// computed the next one's rows go from memory straight into the other (8-bit ones through
// registers, and widened once for all four waves).
//
// A wave's matrix instructions and its softmax take turns on the same SIMD, so the
// loop is a chain of two stages: the scores of the next 32 keys are formed
// between the instructions that turn this step's scores into weights. K's
// buffer therefore runs 32 keys ahead of V's. Two workgroups a CU (64 KiB of LDS each at D = 128)
// fill each other's waits.
//
// Bound by the matrix cores together with the softmax's vector instructions: 8192
// tokens, 32 heads on 8, D = 128, causal: 550 to 565 us by the card = 1.0 PFLOP/s (the skipped half
// not counted); with 8-bit keys and values 580. D = 64: 338 us = 810 TFLOP/s, as many
// exponentials, maxima and conversions beside half the products. The library's bf16 product reaches 1.1 (4096 cubed) to 1.29 (8192); this
// loop without its softmax and LDS reads 1.27, at the clock the card holds under such
// load. Six chunks against up to 30 K keys: 865 us = 910 TFLOP/s.
//
// Every workgroup finds its tile itself, from the lengths on the device. The longest
// request's tiles go first, its last ones (the longest, under the causal mask) before the
// others, so that the short ones fill the end: 6 chunks over up to 30 K keys 955 us in the requests'
// order, 892 so; 128 chunks of 10 to 40 tokens 135 and 116. A thread a request counts
// the tiles that go before, which costs more than it gives where requests are many
// (250 chunks: 34 us, 52 so): beyond kOrdered request n gets the numbers from floor(cu[n] G / rows) + n,
// at least as many as it needs, the last number first, and its request is a count.
// The key head is the fastest index, so that the workgroups of a head meet in one
// chiplet's L2.
// ---------------------------------------------------------------------------

constexpr int kTile = 64;
constexpr int kTileRows = 128;
constexpr int kMinPart = 256;  // keys of a split, at least: the host knows the table's width only
constexpr int kOrdered = 128;  // requests whose tiles go by length
constexpr int kWaitMemory = 0x0070;  // s_waitcnt vmcnt(0) lgkmcnt(0)

struct PrefillWs {
    float *o;    // [splits][key heads][tokens * group][D], not normalized
    float2 *ml;  // [splits][key heads][tokens * group]
};

struct PrefillArgs {
    Params params;
    PrefillWs ws;
    int tiles, splits;
};

template <int D, bool FP8, bool UNIFORM>
__global__ __launch_bounds__(kThreads, 2) void prefill_kernel(const PrefillArgs args) {
    const Params &a = args.params;
    const int splits = args.splits;
    constexpr int kRows = kTileRows;
    using R = Row<D, FP8>;
    constexpr int kLoads = 16 / R::kRows;  // 16-byte loads a thread, of 16 rows a wave
    constexpr int kBytes = kTile * D * 2;
    __shared__ struct __attribute__((aligned(16))) {
        char kv[2][2][kBytes];  // [parity][K, V]
        int2 keys_tiles[kThreads];  // of each request
        int2 found;  // this workgroup's request, and its first row of it
    } sm;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5;
    const int col = lane & 31;

    if (blockIdx.x < 64) {
        zero_uncovered<D>(a, blockIdx.x, min(gridDim.x, 64u));
    }

    // ---- the tile: key head, split, request, rows
    uint32_t id = blockIdx.x;
    const int head = id % a.cache.kv_heads;
    id /= a.cache.kv_heads;
    const int split = id % splits;
    const int place = static_cast<int>(id / splits);
    int n, row0;
    if (a.num_seqs <= kOrdered) {
        const Request r = a.request(min(tid, a.num_seqs - 1));
        const int mine = tid < a.num_seqs ? (r.tokens * a.group + kRows - 1) / kRows : 0;
        sm.keys_tiles[tid] = make_int2(r.keys, mine);
        if (tid == 0) {
            sm.found = make_int2(-1, 0);
        }
        __syncthreads();
        int before = 0;
        for (int x = 0; x < a.num_seqs; x += 16) {  // past the last one none has tiles
            int2 other[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                other[k] = sm.keys_tiles[x + k];
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                before += other[k].x > r.keys || (other[k].x == r.keys && x + k < tid) ? other[k].y : 0;
            }
        }
        if (place >= before && place < before + mine) {
            sm.found = make_int2(tid, (before + mine - 1 - place) * kRows);
        }
        __syncthreads();
        n = __builtin_amdgcn_readfirstlane(sm.found.x);
        row0 = __builtin_amdgcn_readfirstlane(sm.found.y);
        if (n < 0) {
            return;
        }
    } else {
        const int tile = args.tiles - 1 - place;
        int below = 0;  // requests that begin at or before this tile
        for (int first_n = 0; first_n < a.num_seqs; first_n += kThreads) {
            const int x = first_n + tid;
            const int first = x < a.num_seqs ? static_cast<int>(static_cast<int64_t>(a.cu(x)) * a.group / kRows) + x : INT32_MAX;
            below += __syncthreads_count(first <= tile);
        }
        n = __builtin_amdgcn_readfirstlane(below) - 1;
        if (n < 0) {
            return;
        }
        const int begin = a.cu(n);
        const int64_t row = (tile - static_cast<int64_t>(begin) * a.group / kRows - n) * kRows;
        if (row < 0 || row >= static_cast<int64_t>(a.cu(n + 1) - begin) * a.group) {
            return;
        }
        row0 = static_cast<int>(row);
    }
    const Request req = a.request(n);
    const int rows_all = req.tokens * a.group;
    const int rows = min(kRows, rows_all - row0);

    // ---- visible keys: of the tile in tiles of 64, of the wave, of each lane's rows
    const int2 see0 = a.visible(req, row0 / a.group);
    const int2 see1 = a.visible(req, (row0 + rows - 1) / a.group);
    const int all0 = see0.x / kTile, all1 = (see1.y + kTile - 1) / kTile;
    const int share = max((all1 - all0 + splits - 1) / splits, kMinPart / kTile);
    const int t0 = all0 + split * share, t1 = min(all1, t0 + share);
    const int wrow0 = min(row0 + wave * 32, row0 + rows - 1);
    const int wrow1 = min(wrow0 + 32, row0 + rows) - 1;
    const int2 wsee0 = a.visible(req, wrow0 / a.group);
    const int2 wsee1 = a.visible(req, wrow1 / a.group);
    const bool active = wave * 32 < rows;  // the wave has rows
    const Scores sc = scores_of(a, head);

    u32x4 q[D / 16];
    int2 see;
    {
        const int r = min(row0 + wave * 32 + col, row0 + rows - 1);
        const int t = r / a.group;
        const int h = head * a.group + r - t * a.group;
        see = a.visible(req, t);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            q[s] = load_q(a, req.begin + t, h, s * 16 + half * 8, sc.flip);
        }
    }
    f32x16 o[D / 32];
    float m, l;

    // ---- staging. Of every 64 keys a wave loads 16, a group: keys 64 j + 16 wave, j = t0, t0 + 1, ...
    const char *kbase = static_cast<const char *>(a.cache.k) + ((head * a.cache.k_stride_head) << R::kShift);
    const char *vbase = static_cast<const char *>(a.cache.v) + ((head * a.cache.v_stride_head) << R::kShift);
    const int64_t kpage = a.cache.k_stride_page << R::kShift, vpage = a.cache.v_stride_page << R::kShift;
    const int64_t ktoken = a.cache.k_stride_token << R::kShift, vtoken = a.cache.v_stride_token << R::kShift;
    const char *zero = reinterpret_cast<const char *>(g_zero_row);
    const int srow = lane / R::kLanes, schunk = lane % R::kLanes;  // of a load; kRows of Row further for each next
    const int pool = static_cast<int>(a.cache.num_pages);
    // A group's page entries: of the lane's own rows, or, where pages hold a multiple of 16 tokens
    // (UNIFORM), of all 16 rows. Those are walked without divisions.
    struct Group {
        int key;                       // its first
        int page[UNIFORM ? 1 : kLoads];  // as looked up: the entry's first word in even lanes, its last in odd ones
        int64_t koff, voff;  // UNIFORM: bytes of its first row on the page
    };
    const PageWords words = a.page_words(n, (lane & 1) != 0);
    Group ahead;  // the walk's next
    int at = 0, off = 0;
    const int step_at = kTile / a.cache.page_size, step_off = kTile - step_at * a.cache.page_size;
    auto begin_walk = [&]() KDA_INLINE {
        ahead.key = t0 * kTile + wave * 16;
        if constexpr (UNIFORM) {
            at = ahead.key / a.cache.page_size;
            off = ahead.key - at * a.cache.page_size;
            ahead.koff = off * ktoken;
            ahead.voff = off * vtoken;
        }
    };
    auto walk = [&]() KDA_INLINE -> Group {
        Group r = ahead;
        if constexpr (UNIFORM) {
            r.page[0] = words.of(min(at, a.max_pages - 1));
            at += step_at;
            off += step_off;
            int wrap = 0;
            if (off >= a.cache.page_size) {
                off -= a.cache.page_size;
                ++at;
                wrap = a.cache.page_size;
            }
            ahead.koff += (step_off - wrap) * ktoken;
            ahead.voff += (step_off - wrap) * vtoken;
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                r.page[i] = words.of(min((r.key + srow + i * R::kRows) / a.cache.page_size, a.max_pages - 1));
            }
        }
        ahead.key += kTile;
        return r;
    };
    // The entries have come: their pages, in every lane or (UNIFORM) in a scalar register. Done once, a turn before
    // the group's keys and values are loaded (8192 tokens 563 us; for each of the two loads 567).
    auto looked_up = [&](Group r) KDA_INLINE -> Group {
        if constexpr (!UNIFORM) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                r.page[i] = page_of(__builtin_amdgcn_update_dpp(0, r.page[i], kDppQuadEven, 0xf, 0xf, false),
                                    __builtin_amdgcn_update_dpp(0, r.page[i], kDppQuadOdd, 0xf, 0xf, false));
            }
        } else {
            r.page[0] = page_of(__builtin_amdgcn_readlane(r.page[0], 0), __builtin_amdgcn_readlane(r.page[0], 1));
        }
        return r;
    };
    // A lane's bytes of a group. bf16 rows go from memory into LDS directly, where a wave's 64 x 16
    // bytes land in order: a lane fetches the chunk that belongs at its place. 8-bit ones go through
    // registers, where they are widened. The loads' immediate offsets (1 KiB each) move both addresses.
    constexpr int kKib = FP8 ? 0 : 1024;
    uint32_t krow[kLoads], vrow[kLoads];
    auto kcol = [&](int i) KDA_INLINE { return (FP8 ? schunk : k_chunk<D>(srow + i * R::kRows, schunk)) * 16; };
    auto vcol = [&](int i) KDA_INLINE { return (FP8 ? schunk : v_chunk<D>(srow + i * R::kRows, schunk)) * 16; };
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const uint32_t r = srow + i * R::kRows;
        krow[i] = r * static_cast<uint32_t>(ktoken) + kcol(i) + (kLoads - 1 - i) * kKib;
        vrow[i] = r * static_cast<uint32_t>(vtoken) + vcol(i) + (kLoads - 1 - i) * kKib;
    }
    u32x4 kreg[FP8 ? kLoads : 1], vreg[FP8 ? kLoads : 1];
    auto load = [&](const Group &group, const char *base, int64_t page_bytes, int64_t in_page, int64_t token_bytes,
                    const uint32_t (&row)[kLoads], auto column, auto &reg, char *rows_at) KDA_INLINE {
        if constexpr (UNIFORM) {
            const int page = group.page[0];
            const int key = group.key;
            const bool any = static_cast<uint32_t>(page) < static_cast<uint32_t>(pool) && key < see1.y && key + 16 > see0.x;
            uint32_t lane_at[kLoads];
            const char *first = zero;
            if (any && key >= see0.x && key + 16 <= see1.y) {
                first = base + page * page_bytes + in_page;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    lane_at[i] = row[i];
                }
            } else {
                // some rows have no key that the tile sees: the nearest that has stands in (its
                // scores are masked), so nothing is read that no request wrote
                uint32_t token = 0;
                if (any) {
                    first = base + page * page_bytes + in_page;
                    token = static_cast<uint32_t>(token_bytes);
                }
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = max(min(srow + i * R::kRows, see1.y - 1 - key), see0.x - key);
                    lane_at[i] = static_cast<uint32_t>(r) * token + column(i) + (kLoads - 1 - i) * kKib;
                }
            }
            if constexpr (FP8) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    reg[i] = load16(first + lane_at[i]);
                }
            } else {
                load16_to_lds(first - (kLoads - 1) * kKib, lane_at, rows_at);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int key = group.key + srow + i * R::kRows;
                const int page = group.page[i];
                const int in = key - key / a.cache.page_size * a.cache.page_size;
                const bool real = key >= see0.x && key < see1.y && static_cast<uint32_t>(page) < static_cast<uint32_t>(pool);
                const char *first = (real ? base + page * page_bytes + in * token_bytes : zero) + column(i);
                if constexpr (FP8) {
                    reg[i] = load16(first);
                } else {
                    load16_to_lds(first, rows_at + i * 1024);
                }
            }
        }
    };
    // K's buffer is filled 32 keys ahead of V's: its rows are the groups' of waves 2, 3, then 0, 1
    const int kslot = 16 * ((wave + 2) & 3), vslot = 16 * wave;
    auto load_k = [&](const Group &group, int parity) KDA_INLINE {
        load(group, kbase, kpage, group.koff, ktoken, krow, kcol, kreg, sm.kv[parity][0] + kslot * 2 * D);
    };
    auto load_v = [&](const Group &group, int parity) KDA_INLINE {
        load(group, vbase, vpage, group.voff, vtoken, vrow, vcol, vreg, sm.kv[parity][1] + vslot * 2 * D);
    };
    auto write_k = [&](int parity) KDA_INLINE {
        if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                stage<D, FP8>(sm.kv[parity][0], kslot + srow + i * R::kRows, schunk, kreg[i], [](int r, int c) { return k_at<D>(r, c); });
            }
        }
    };
    auto write_v = [&](int parity) KDA_INLINE {
        if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                stage<D, FP8>(sm.kv[parity][1], vslot + srow + i * R::kRows, schunk, vreg[i], [](int r, int c) { return v_at<D>(r, c); });
            }
        }
    };
    // In the second pass: the wave's rows of values without what is not finite.
    auto finite_v = [&](auto again, int parity) KDA_INLINE {
        if constexpr (again) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(kWaitMemory);  // the wave's own rows have landed
            asm volatile("" ::: "memory");
#pragma unroll
            for (int x = 0; x < 16 * 2 * D / 1024; ++x) {
                u32x4 *p = reinterpret_cast<u32x4 *>(sm.kv[parity][1] + vslot * 2 * D + x * 1024 + lane * 16);
                *p = finite_only(*p);
            }
        }
    };
    // All rows of the buffers are there, and the reads of the others have ended, for every wave.
    auto staged = [&]() KDA_INLINE {
        if constexpr (FP8) {
            lds_barrier();
        } else {
            // as a builtin, so that the compiler counts its own loads as done too
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(kWaitMemory);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
    };

    // ---- the chain, 32 keys a step: a lane's scores are of row `col`, keys 8 (e / 4) + 4 half + e % 4
    auto products = [&](int parity, int kt, f32x16 &s) KDA_INLINE {
        const char *tile = sm.kv[parity][0];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = 0.0f;
        }
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            s = mfma32(*reinterpret_cast<const u32x4 *>(tile + k_at<D>(kt * 32 + col, 2 * x + half)), q[x], s);
        }
    };
    const float c = sc.cap > 0.0f ? 1.0f : sc.c;
    float top;  // largest of the scores that are next, in log2 units
    // cap, mask and largest score of the keys from key0
    auto finish = [&](int key0, f32x16 &s) KDA_INLINE {
        if (sc.cap > 0.0f) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = capped(s[e] * sc.in, sc.cap);
            }
        }
        if (!(key0 >= wsee1.x && key0 + 32 <= wsee0.y)) {  // some row of the wave does not see some key
            const int from = see.x - key0 - 4 * half, to = see.y - key0 - 4 * half;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int k = 8 * (e >> 2) + (e & 3);
                s[e] = k >= from && k < to ? s[e] : kNegInf;
            }
        }
        float x = kNegInf;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x = fmaxf(x, s[e]);
        }
        top = max_halves(x) * c;
    };
    // weights of the scores s and their products with rows 32 kt .. of the values in buffer `parity`; the
    // next 32 keys' scores are formed meanwhile
    auto step = [&](int parity, int kt, const f32x16 &s, f32x16 &next) KDA_INLINE {
        const bool raise = top > m + kRaise;
        if (__any(raise)) {
            const float up = raise ? top : m;
            const float f = up == m ? 1.0f : ex2(m - up);
            m = up;
            l *= f;
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                o[d] *= f;
            }
        }
        products(parity, kt, next);
        const float base = m == kNegInf ? 0.0f : m;
        u32x4 p[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // 16 keys: 8 of this half of the wave
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = ex2(s[8 * x + e] * c - base);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[x][e] = pack_bf16x2(w[2 * e], w[2 * e + 1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                l = add_pair(p[x][e], l);
            }
        }
        const char *vt = sm.kv[parity][1];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const int pair = 2 * d + ((lane >> 4) & 1);
                const int row = 32 * kt + 16 * x + 4 * half;
                const u32x2 v0 = read_tr<D>(vt, row, pair, lane);
                const u32x2 v1 = read_tr<D>(vt, row + 8, pair, lane);
                o[d] = mfma32(u32x4{v0[0], v0[1], v1[0], v1[1]}, p[x], o[d]);
            }
        }
    };

    auto pass = [&](auto again) KDA_INLINE {
        m = kNegInf;
        l = 0.0f;
        top = kNegInf;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[d][e] = 0.0f;
            }
        }
        if (t0 < t1) {
            // tiles that the wave sees: [w0, w1)
            const int w0 = active ? max(t0, wsee0.x / kTile) : t1, w1 = active ? min(t1, (wsee1.y + kTile - 1) / kTile) : t1;
            // In turn t V's buffer holds the keys 64 t .., K's the keys 64 t + 32 ..: the first 32 keys'
            // scores are formed before, from the second half of the other buffer.
            begin_walk();
            Group now = walk(), next = walk(), after = walk();
            now = looked_up(now);
            next = looked_up(next);
            const bool early = wave < 2;  // K's next rows are of the group after V's next rows
            if (early) {
                load_k(now, 1);
            }
            load_v(now, 0);
            write_k(1);
            load_k(early ? next : now, 0);
            write_k(0);
            write_v(0);
            finite_v(again, 0);
            now = next;
            next = looked_up(after);
            after = walk();
            staged();
            f32x16 even, odd;
            if (t0 == w0) {
                products(1, 1, even);
                finish(t0 * kTile, even);
            }
            lds_barrier();  // before the first turn stages over these keys
            auto turn = [&](int t, int parity) KDA_INLINE {
                // past the last tile rows of zeros are loaded and staged, whose scores nobody uses
                load_k(early ? next : now, parity ^ 1);
                load_v(now, parity ^ 1);
                now = next;
                next = looked_up(after);
                after = walk();
                if (t >= w0 && t < w1) {
                    step(parity, 0, even, odd);
                    finish(t * kTile + 32, odd);
                    step(parity, 1, odd, even);
                    finish(t * kTile + kTile, even);
                } else if (t + 1 == w0) {
                    products(parity, 1, even);
                    finish(t * kTile + kTile, even);
                }
                write_k(parity ^ 1);
                write_v(parity ^ 1);
                finite_v(again, parity ^ 1);
                staged();
            };
            for (int t = t0; t < t1; t += 2) {
                turn(t, 0);
                if (t + 1 < t1) {
                    turn(t + 1, 1);
                }
            }
        }
    };
    pass(std::false_type{});
    bool fine = true;  // where a score is NaN the whole row is
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            fine &= is_finite(o[d][e]) || l != l;
        }
    }
    if (!__syncthreads_and(fine)) {
        pass(std::true_type{});
        each_not_finite<D, FP8>(arguments_again(args).params, n, head, max(t0 * kTile, wsee0.x), min(t1 * kTile, wsee1.y), [&](int key, const char *row) KDA_INLINE {
            if (key >= see.x && key < see.y) {
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        o[d][e] += not_finite<FP8>(row, d * 32 + 8 * (e >> 2) + 4 * half + (e & 3));
                    }
                }
            }
        });
    }

    // ---- out, or this split's part: lane: row `col` of 32, columns 32 d + 8 (e / 4) + 4 half + e % 4
    const PrefillArgs &last = arguments_again(args);
    const float vs = last.params.cache.v_scale != nullptr ? last.params.cache.v_scale[head] : 1.0f;
    const int r = wave * 32 + col;
    const float sum = sum_halves(l);
    m = see.x < see.y ? fmaxf(m, kLowest) : m;
    if (r >= rows) {
        return;
    }
    if (last.splits == 1) {
        const float f = m == kNegInf ? 0.0f : vs / sum;
        const int t = (row0 + r) / last.params.group;
        const int h = head * last.params.group + (row0 + r) - t * last.params.group;
        uint16_t *out = static_cast<uint16_t *>(last.params.out) + static_cast<int64_t>(req.begin + t) * last.params.out_stride_token +
                        h * last.params.out_stride_head + half * 4;
        struct __attribute__((packed, aligned(2))) Out {
            uint32_t w[2];
        };
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                *reinterpret_cast<Out *>(out + d * 32 + e * 8) = {
                    {pack_bf16x2(o[d][4 * e] * f, o[d][4 * e + 1] * f),
                     pack_bf16x2(o[d][4 * e + 2] * f, o[d][4 * e + 3] * f)}};
            }
        }
    } else {
        const int64_t all = static_cast<int64_t>(last.params.num_tokens) * last.params.group;
        const int64_t at = (static_cast<int64_t>(split) * last.params.cache.kv_heads + head) * all +
                           static_cast<int64_t>(req.begin) * last.params.group + row0 + r;
        if (half == 0) {
            last.ws.ml[at] = make_float2(m, sum);
        }
        if (sum != 0.0f) {  // the join reads no others
            float *po = last.ws.o + at * D + half * 4;
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    *reinterpret_cast<f32x4 *>(po + d * 32 + e * 8) =
                        f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
                }
            }
        }
    }
}

// Joins the splits of every (token, head): 16 or 32 threads a row, 4 columns each. kAtOnce parts' loads
// are in flight together: as many as there are, up to 8 (16 tokens over 30 K keys 77 us with one after
// another, 58 with 4, 49 so; two splits of 1000 tokens 37 us, 43 with room for 8).
template <int D, int kAtOnce>
__global__ __launch_bounds__(kThreads) void prefill_combine_kernel(const Params a, const PrefillWs ws, int splits) {
    constexpr int kPer = D / 4;
    const int64_t all = static_cast<int64_t>(a.num_tokens) * a.group;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (kThreads / kPer) + threadIdx.x / kPer;
    if (i >= all * a.cache.kv_heads) {
        return;
    }
    const int64_t row = i / a.cache.kv_heads;
    const int head = static_cast<int>(i % a.cache.kv_heads);
    const int64_t t = row / a.group;
    if (t < a.cu(0) || t >= a.cu(a.num_seqs)) {
        return;  // no request's token: zero already
    }
    const int c = threadIdx.x % kPer * 4;
    const int64_t step = a.cache.kv_heads * all, at = head * all + row;
    // parts that saw no key (the table's width, not the request's keys, sets the number) have a sum of 0 and no O
    float top = kNegInf;
    for (int s = 0; s < splits; s += kAtOnce) {
        float2 ml[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            ml[k] = ws.ml[at + min(s + k, splits - 1) * step];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            top = fmaxf(top, ml[k].x);
        }
    }
    float sum = 0.0f;
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < splits; s += kAtOnce) {
        float2 ml[kAtOnce];
        f32x4 o[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            ml[k] = ws.ml[at + min(s + k, splits - 1) * step];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            o[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (s + k < splits && ml[k].y != 0.0f) {
                o[k] = *reinterpret_cast<const f32x4 *>(ws.o + (at + (s + k) * step) * D + c);
            }
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (s + k < splits && ml[k].y != 0.0f) {
                const float f = ml[k].x == top ? 1.0f : ex2(ml[k].x - top);
                sum += ml[k].y * f;
                y += o[k] * f;
            }
        }
    }
    const float vs = a.cache.v_scale != nullptr ? a.cache.v_scale[head] : 1.0f;
    y *= top == kNegInf ? 0.0f : vs / sum;
    uint16_t *out = static_cast<uint16_t *>(a.out) + t * a.out_stride_token +
                    (head * a.group + row - t * a.group) * a.out_stride_head + c;
    struct __attribute__((packed, aligned(2))) Out {
        uint32_t w[2];
    };
    *reinterpret_cast<Out *>(out) = {{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])}};
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct Plan {
    bool decode;
    int blocks;     // decode: NB
    bool join;      // decode: items may be split
    int64_t tiles;  // prefill
    int splits;
    size_t ml_at, desc_at, bytes;
};

size_t up256(size_t x) { return (x + 255) & ~size_t{255}; }

int64_t most_rows(const KdaPagedAttentionArgs &a) {
    return std::max<int64_t>(a.max_query_len, 1) * (a.num_heads / a.cache.kv_heads);
}

// At most 32 rows a request (without requests, the decode kernel only writes the zeros). The largest request
// decides for the whole call. us, in tiles of 16 rows (NB = 1), of 32 rows (NB = 2), by the prefill kernel:
//   rows of each request                    8          16            32            40            64
//   32 x 4096 keys, 32 heads on 4, D 128  56 58 63   57 60 64    98  64  67   142 103  68   176 106  69
//   64 x 4096 keys, 32 heads on 4, D 64   53 55 74   53 55 75    92  56  76   135  96  78   175  95  78
//   64 x 4096 keys, 8 on 1, D 128, 8 bit  26 29 33   28 33 33    36  38  35    48  43  40    58  43  44
//   1 x 8192 keys, 32 heads on 4, D 128   18 20 25   23 24 25    31  30  26    31  36  27    34  41  27
bool decodes(const KdaPagedAttentionArgs &a) { return most_rows(a) <= 32 || a.num_seqs == 0; }

Plan plan_of(const KdaPagedAttentionArgs &a) {
    Plan p{};
    const int64_t group = a.num_heads / a.cache.kv_heads;
    const int64_t rows = most_rows(a);
    const int64_t keys = static_cast<int64_t>(a.max_pages) * a.cache.page_size;
    const size_t d = a.cache.head_dim;
    p.decode = decodes(a);
    if (p.decode) {
        p.blocks = rows <= 16 ? 1 : 2;
        p.join = keys > kUnit;
        const size_t parts = size_t{2} * kDecodeGroups * 16 * p.blocks;
        p.ml_at = up256(p.join ? parts * d * 4 : 0);
        p.desc_at = up256(p.ml_at + (p.join ? parts * 8 : 0));
        p.bytes = p.desc_at + size_t{kDecodeGroups} * 16;
        return p;
    }
    p.tiles = static_cast<int64_t>(a.num_tokens) * group / kTileRows + a.num_seqs;
    // few tiles over many keys: cut the keys until two workgroups a CU have work (512 tokens over 32 K keys:
    // 325 us; 665 with one a CU, 339 with four), in parts of 256 keys at least (64 tokens over 1008 keys 22 us,
    // with 512 30 us). The join's time grows with the parts and the loop's falls with them, so the best number
    // goes with the keys' root. 16 tokens over 30 K keys, us: 53 with at most 16 parts, 41 with 32, 50 with 64, 42 so;
    // 64 tokens over 8 K: 31, 31, 35 and 31.
    const int64_t units = p.tiles * a.cache.kv_heads;
    const int64_t best = static_cast<int64_t>(std::sqrt(static_cast<double>(keys) / 32.0));
    p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({2 * kCus / units, keys / 256, best})));
    if (p.splits > 1) {
        const size_t parts = static_cast<size_t>(p.splits) * a.num_tokens * a.num_heads;
        p.ml_at = up256(parts * d * 4);
        p.bytes = up256(p.ml_at + parts * 8);
    }
    return p;
}

// What the plan and the workspace follow from; no pointer, stride or option of the softmax.
int check_sizes(const KdaPagedAttentionArgs *args) {
    if (args == nullptr) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const KdaPagedAttentionArgs &a = *args;
    if (const int rc = check_cache_sizes(a.cache); rc != KDA_OK) {
        return rc;
    }
    if (a.num_seqs < 0 || a.num_tokens < 0 || a.num_heads <= 0 || a.max_pages < 0 || a.num_heads > INT32_MAX / 128 ||
        a.num_heads % a.cache.kv_heads != 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const int64_t group = a.num_heads / a.cache.kv_heads;
    // row and key numbers, the roundings up of both and the decode kernel's units stay in 32 bits
    const int64_t rows = a.num_tokens * group, keys = static_cast<int64_t>(a.max_pages) * a.cache.page_size;
    if (rows + 128 * static_cast<int64_t>(a.num_seqs) > INT32_MAX - 1024 || keys > INT32_MAX - 1024) {
        return KDA_ERR_TOO_LARGE;
    }
    if (decodes(a) && (rows / 16 + a.num_seqs) * a.cache.kv_heads > INT32_MAX / (keys / kUnit + 1)) {
        return KDA_ERR_TOO_LARGE;
    }
    return KDA_OK;
}

int check(const KdaPagedAttentionArgs *args) {
    if (const int rc = check_sizes(args); rc != KDA_OK) {
        return rc;
    }
    const KdaPagedAttentionArgs &a = *args;
    if (const int rc = check_cache(a.cache); rc != KDA_OK) {
        return rc;
    }
    constexpr int32_t kWide = KDA_WIDE_PAGE_TABLE | KDA_WIDE_KV_LENS | KDA_WIDE_CU_SEQLENS;
    if (a.window < 0 || !(a.logit_cap == 0.0f || (a.logit_cap >= 0.9e-30f && a.logit_cap <= 1.1e30f)) ||
        (a.wide & ~kWide) != 0) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    return KDA_OK;
}

bool misaligned(const void *p, uintptr_t m) { return reinterpret_cast<uintptr_t>(p) % m != 0; }

template <int D, bool FP8, int NB> void launch_decode(const Params &a, const Plan &p, char *ws, hipStream_t s) {
    const DecodeWs w{reinterpret_cast<float *>(ws), reinterpret_cast<float2 *>(ws + p.ml_at),
                     reinterpret_cast<int4 *>(ws + p.desc_at)};
    decode_kernel<D, FP8, NB><<<kDecodeGroups, kThreads, 0, s>>>(a, w);
    if (p.join) {
        // Few items are cut into many parts: more workgroups an item then (one request of 32 K keys and one
        // key head: 26 us for 16 rows, 52 with 4 workgroups; 34 us for 32 rows, 95 with 4). Of many items most
        // are whole, and the workgroups without one cost more than they give (256 requests in 8 bits: 172 us,
        // 177 with 16).
        const int64_t items = static_cast<int64_t>(a.num_seqs) * a.cache.kv_heads;
        const unsigned joins = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(64 / std::max<int64_t>(items, 1), 4), 16 * NB));
        decode_combine_kernel<D, NB><<<dim3(kDecodeGroups, joins), kThreads, 0, s>>>(a, w);
    }
}

template <int D, bool FP8> void launch_attention(const Params &a, const Plan &p, char *ws, hipStream_t s) {
    if (p.decode) {
        p.blocks == 1 ? launch_decode<D, FP8, 1>(a, p, ws, s) : launch_decode<D, FP8, 2>(a, p, ws, s);
        return;
    }
    const PrefillWs w{reinterpret_cast<float *>(ws), reinterpret_cast<float2 *>(ws + p.ml_at)};
    const unsigned grid = static_cast<unsigned>(p.tiles * a.cache.kv_heads * p.splits);
    const PrefillArgs args{a, w, static_cast<int>(p.tiles), p.splits};
    // 16 rows of a page at offsets that fit 32 bits: one page number and one address for the wave's 16
    // rows (8192 tokens 540 us, chunks over 30 K keys 925 us; each row's page looked up: 720 and 1342)
    const auto near = [](int64_t stride) { return stride >= 0 && stride < (1 << 26); };
    if (a.cache.page_size % 16 == 0 && near(a.cache.k_stride_token) && near(a.cache.v_stride_token)) {
        prefill_kernel<D, FP8, true><<<grid, kThreads, 0, s>>>(args);
    } else {
        prefill_kernel<D, FP8, false><<<grid, kThreads, 0, s>>>(args);
    }
    if (p.splits > 1) {
        const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.num_heads;
        constexpr int kPer = kThreads / (D / 4);
        const unsigned groups = static_cast<unsigned>((rows + kPer - 1) / kPer);
        if (p.splits == 2) {
            prefill_combine_kernel<D, 2><<<groups, kThreads, 0, s>>>(a, w, p.splits);
        } else if (p.splits <= 4) {
            prefill_combine_kernel<D, 4><<<groups, kThreads, 0, s>>>(a, w, p.splits);
        } else {
            prefill_combine_kernel<D, 8><<<groups, kThreads, 0, s>>>(a, w, p.splits);
        }
    }
}

}  // namespace
}  // namespace kda

extern "C" size_t kda_paged_attention_workspace_bytes(const KdaPagedAttentionArgs *args) {
    using namespace kda;
    if (check_sizes(args) != KDA_OK || args->num_tokens == 0) {
        return 0;
    }
    return plan_of(*args).bytes;
}

extern "C" int kda_paged_attention_launch(const KdaPagedAttentionArgs *args, void *workspace, size_t workspace_bytes,
                                          void *stream) {
    using namespace kda;
    if (const int rc = check(args); rc != KDA_OK) {
        return rc;
    }
    Params a{*args, args->num_heads / args->cache.kv_heads};
    if (a.num_tokens == 0) {
        return KDA_OK;
    }
    if (a.q == nullptr || a.out == nullptr || misaligned(a.q, 2) || misaligned(a.out, 2) || a.cu_seqlens == nullptr ||
        misaligned(a.cu_seqlens, (a.wide & KDA_WIDE_CU_SEQLENS) != 0 ? 8 : 4) ||
        (a.num_seqs > 0 && (a.kv_lens == nullptr || misaligned(a.kv_lens, (a.wide & KDA_WIDE_KV_LENS) != 0 ? 8 : 4))) ||
        (a.num_seqs > 0 && a.max_pages > 0 &&
         (a.page_table == nullptr || misaligned(a.page_table, (a.wide & KDA_WIDE_PAGE_TABLE) != 0 ? 8 : 4)))) {
        return KDA_ERR_INVALID_ARGUMENT;
    }
    const Plan p = plan_of(a);
    // a grid counts its threads in 32 bits (splits are made where units are few, so the join's grid is small)
    if (!p.decode && p.tiles * a.cache.kv_heads * p.splits > (INT64_C(1) << 24) - 1) {
        return KDA_ERR_TOO_LARGE;
    }
    if (p.bytes > 0 && (workspace == nullptr || misaligned(workspace, 256) || workspace_bytes < p.bytes)) {
        return KDA_ERR_WORKSPACE;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *ws = static_cast<char *>(workspace);
    const bool fp8 = a.cache.dtype == KDA_FP8_E4M3;
    (void)hipGetLastError();
    if (a.cache.head_dim == 128) {
        fp8 ? launch_attention<128, true>(a, p, ws, s) : launch_attention<128, false>(a, p, ws, s);
    } else {
        fp8 ? launch_attention<64, true>(a, p, ws, s) : launch_attention<64, false>(a, p, ws, s);
    }
    return hipGetLastError() == hipSuccess ? KDA_OK : KDA_ERR_LAUNCH;
}
