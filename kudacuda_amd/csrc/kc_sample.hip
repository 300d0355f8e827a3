// Next tokens of rows of logits: temperature, top-k, top-p and min-p, drawn with
// one given uniform number a row.
//
//     w_i = exp((l_i - max) / T), tokens ordered by (l descending, id ascending);
//     kept: the first top_k; of these the tokens before which the weights sum to
//     less than top_p * (sum of the first top_k); of these the tokens with
//     w >= min_p; the first token always;
//     token = the lowest id whose kept weights, summed by id, pass u * (their sum).
//
// Weights are whole numbers, w rounded to 2^-42 (exp in 64 bits): their sums are
// exact and do not depend on the order of atomics, so equal inputs give equal
// tokens, and a sum over 2^20 tokens fits in 64 bits.  A token below 2^-43 of the
// most likely one weighs nothing.
//
// No row is sorted.  Tokens fall into buckets of 1/64 in log2 w; which bucket ends
// the kept tokens follows from the buckets' counts and sums, and only that bucket's
// tokens (a few to some hundred) are ordered.  Launches, each over (blocks of a row,
// rows):
//   1. the row's largest logit, and the largest of every 128 ids;
//   2. buckets (for top-k and top-p; with top-k only those down to the k-th of the
//      largest of 128, below which no kept token lies);
//   3. tokens of the deciding buckets to a list, sums of the surely kept tokens of
//      each chunk of 2048 ids;
//   4. one block a row: the last kept token of the list, the chunk and in it
//      the token that u falls on.
// The row is read by the first three (once from memory, then from the caches) and
// one chunk of it by the last.  A logit is first compared with the least one that
// matters, in 32 bits; 64-bit arithmetic is for those that do.
#include "kc_device.h"
#include "kc_kernels.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunk = 8 * kThreads;  // ids of a chunk: 8 a thread
constexpr int kAhead = 4;             // chunks that a block requests together
constexpr int kGroups = kThreads / 16;  // groups of 128 ids of a chunk, 16 lanes each
constexpr int kUnits = 64;            // buckets of a factor of two
constexpr int kDepth = 43 * kUnits;   // buckets of the weights' range
constexpr int kBuckets = 11 * kThreads;
constexpr int kPer = kBuckets / kThreads;
constexpr int kCoarse = 64;           // buckets that are summed together, a wave's
static_assert(kBuckets % kCoarse == 0 && kBuckets / kCoarse <= 64, "the sums fit a wave");
constexpr int kList = 2048;           // most tokens that are ordered in LDS
constexpr int kWeightBits = 42;
// Blocks of the first and third launch, and large blocks of the second: more rows than
// fill these take more chunks a block (128 rows of mixed settings in their own order: 2048 and
// 256 87 us, 2048 and 512 90, 1280 and 256 88; 32 rows with top-p: 256 large blocks 50 us, 512 61).
constexpr int64_t kBlocks = 2048;
constexpr int64_t kLargeBlocks = 256;
// From so many rows on the rows with the most work start first, and the second launch's
// blocks go to the rows that have work there, two to a row of which all logits count for
// one to a row of few (128 rows of mixed settings: in their own order 82 us, so 74, three
// to one 79; 256 133 and 109; 32 42.9 and 43.4; 64 rows of one setting alone 64 and 65).
constexpr int64_t kOrderedRows = 64;
constexpr int kDenseShare = 2;
constexpr int kMaxChunks = static_cast<int>(kSampleMaxVocab / kChunk);
constexpr int kIdBits = 20;
constexpr uint64_t kIdMask = (uint64_t{1} << kIdBits) - 1;
static_assert(kSampleMaxVocab <= (int64_t{1} << kIdBits), "ids of an order word");
static_assert(kDepth < kBuckets, "a bucket for every weight");

// 2^(-j / 64).
__device__ constexpr double kPowers[kUnits] = {
    0x1.0000000000000p+0, 0x1.fa7c1819e90d8p-1, 0x1.f50765b6e4540p-1, 0x1.efa1bee615a27p-1,
    0x1.ea4afa2a490dap-1, 0x1.e502ee78b3ff6p-1, 0x1.dfc97337b9b5fp-1, 0x1.da9e603db3285p-1,
    0x1.d5818dcfba487p-1, 0x1.d072d4a07897cp-1, 0x1.cb720dcef9069p-1, 0x1.c67f12e57d14bp-1,
    0x1.c199bdd85529cp-1, 0x1.bcc1e904bc1d2p-1, 0x1.b7f76f2fb5e47p-1, 0x1.b33a2b84f15fbp-1,
    0x1.ae89f995ad3adp-1, 0x1.a9e6b5579fdbfp-1, 0x1.a5503b23e255dp-1, 0x1.a0c667b5de565p-1,
    0x1.9c49182a3f090p-1, 0x1.97d829fde4e50p-1, 0x1.93737b0cdc5e5p-1, 0x1.8f1ae99157736p-1,
    0x1.8ace5422aa0dbp-1, 0x1.868d99b4492edp-1, 0x1.82589994cce13p-1, 0x1.7e2f336cf4e62p-1,
    0x1.7a11473eb0187p-1, 0x1.75feb564267c9p-1, 0x1.71f75e8ec5f74p-1, 0x1.6dfb23c651a2fp-1,
    0x1.6a09e667f3bcdp-1, 0x1.6623882552225p-1, 0x1.6247eb03a5585p-1, 0x1.5e76f15ad2148p-1,
    0x1.5ab07dd485429p-1, 0x1.56f4736b527dap-1, 0x1.5342b569d4f82p-1, 0x1.4f9b2769d2ca7p-1,
    0x1.4bfdad5362a27p-1, 0x1.486a2b5c13cd0p-1, 0x1.44e086061892dp-1, 0x1.4160a21f72e2ap-1,
    0x1.3dea64c123422p-1, 0x1.3a7db34e59ff7p-1, 0x1.371a7373aa9cbp-1, 0x1.33c08b26416ffp-1,
    0x1.306fe0a31b715p-1, 0x1.2d285a6e4030bp-1, 0x1.29e9df51fdee1p-1, 0x1.26b4565e27cddp-1,
    0x1.2387a6e756238p-1, 0x1.2063b88628cd6p-1, 0x1.1d4873168b9aap-1, 0x1.1a35beb6fcb75p-1,
    0x1.172b83c7d517bp-1, 0x1.1429aaea92de0p-1, 0x1.11301d0125b51p-1, 0x1.0e3ec32d3d1a2p-1,
    0x1.0b5586cf9890fp-1, 0x1.0874518759bc8p-1, 0x1.059b0d3158574p-1, 0x1.02c9a3e778061p-1,
};

// What launch 3 tells launch 4 of a row.
struct Decision {
    uint64_t best;        // order word of the row's largest logit
    uint64_t k_weight;    // weights of the buckets before k_bucket (of all: top-k off)
    uint64_t low_weight;  // weights of the buckets before low
    int32_t k_count;      // tokens of the buckets before k_bucket
    int32_t low;          // tokens of buckets below are kept (if min_p lets them)
    int32_t high;         // [low, high]: top-p, or the bucket of the k-th token, decides
    int32_t k_bucket;     // bucket of the k-th token (kBuckets: top-k off or too large)
};
static_assert(sizeof(Decision) <= 64, "the row's workspace");

// Workspace of a row, in this order.
struct RowSpace {
    uint64_t* weights;   // [kBuckets]
    uint64_t* list;      // [kList] order words
    uint64_t* sums;      // [chunks]
    uint64_t* best;      // [chunks] order word of each block's largest logit
    Decision* decision;
    uint32_t* listed;
    uint32_t* counts;    // [kBuckets]
    uint64_t* coarse_weights;  // [64] of kCoarse buckets each
    uint32_t* coarse_counts;   // [64]
    float* largest;      // [chunks * kGroups] of 128 ids each
};
__host__ __device__ inline int64_t row_bytes(int64_t chunks) {
    return kBuckets * 12 + kList * 8 + chunks * (16 + kGroups * 4) + 64 + 16 + 64 * 12;
}
__device__ __forceinline__ RowSpace row_space(uint8_t* base, int64_t row, int chunks) {
    uint8_t* p = base + row * row_bytes(chunks);
    RowSpace s;
    s.weights = reinterpret_cast<uint64_t*>(p);
    p += kBuckets * 8;
    s.list = reinterpret_cast<uint64_t*>(p);
    p += kList * 8;
    s.sums = reinterpret_cast<uint64_t*>(p);
    p += chunks * 8;
    s.best = reinterpret_cast<uint64_t*>(p);
    p += chunks * 8;
    s.decision = reinterpret_cast<Decision*>(p);
    p += 64;
    s.listed = reinterpret_cast<uint32_t*>(p);
    p += 16;
    s.coarse_weights = reinterpret_cast<uint64_t*>(p);
    p += 64 * 8;
    s.coarse_counts = reinterpret_cast<uint32_t*>(p);
    p += 64 * 4;
    s.counts = reinterpret_cast<uint32_t*>(p);
    p += kBuckets * 4;
    s.largest = reinterpret_cast<float*>(p);
    return s;
}

// ---------------------------------------------------------------- one logit
struct F32 {
    static __device__ __forceinline__ float load(float v) { return v; }
};
template <typename T>
struct Raw {
    typedef uint16_t type;
};
template <>
struct Raw<F32> {
    typedef float type;
};
__device__ __forceinline__ uint16_t lowest(Bf16) { return 0xff80u; }
__device__ __forceinline__ uint16_t lowest(F16) { return 0xfc00u; }
__device__ __forceinline__ float lowest(F32) { return -__builtin_huge_valf(); }

// 8 logits from id on as they are stored; -inf where the row ends.
template <typename T>
struct Piece {
    uint4 w[sizeof(typename Raw<T>::type) / 2];
};
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const typename Raw<T>::type* row, int64_t id, int64_t vocab) {
    const auto* const p = row + id;
    Piece<T> v;
    if (id + 8 <= vocab && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(v) / 16; ++i) {
            v.w[i] = reinterpret_cast<const uint4*>(p)[i];
        }
    } else {
        typename Raw<T>::type x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = id + i < vocab ? p[i] : lowest(T{});
        }
        __builtin_memcpy(&v, x, sizeof(v));
    }
    return v;
}
// As fp32, and then: NaN counts as -inf, -0 as 0.
template <typename T>
__device__ __forceinline__ void unpack(float (&x)[8], const Piece<T>& v) {
    typename Raw<T>::type raw[8];
    __builtin_memcpy(raw, &v, sizeof(v));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = T::load(raw[i]);
    }
}
__device__ __forceinline__ float settle(float x) { return x == x ? x + 0.0f : -__builtin_huge_valf(); }
// Their largest (a NaN does not count).
__device__ __forceinline__ float largest_of(const float (&x)[8]) {
    return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
}
template <typename T>
__device__ __forceinline__ const typename Raw<T>::type* row_logits(const SampleArgs& a, int64_t row) {
    return static_cast<const typename Raw<T>::type*>(a.logits) + row * a.stride;
}

// The thread's pieces of chunks c0, c0 + STRIDE, .. that lie before `end`, kAhead of them.
template <typename T>
struct Round {
    Piece<T> piece[kAhead];
};
template <typename T, int STRIDE = 1>
__device__ __forceinline__ Round<T> load_round(const typename Raw<T>::type* logits, int64_t vocab, int c0, int end) {
    Round<T> r;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int c = c0 + j * STRIDE;
        if (c < end) {
            r.piece[j] = load_piece<T>(logits, static_cast<int64_t>(c) * kChunk + threadIdx.x % kThreads * 8, vocab);
        }
    }
    return r;
}
// f(chunk, first id, the thread's 8 logits from there) for every STRIDE-th chunk of
// [begin, end), a round requested while the one before is worked on; the first is
// there already.
template <typename T, int STRIDE = 1, typename F>
__device__ __forceinline__ void for_chunks(const typename Raw<T>::type* logits, int64_t vocab, int begin, int end,
                                           Round<T> round, F f) {
    for (int c0 = begin; c0 < end; c0 += kAhead * STRIDE) {
        const Round<T> next = load_round<T, STRIDE>(logits, vocab, c0 + kAhead * STRIDE, end);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int c = c0 + j * STRIDE;
            if (c < end) {
                float x[8];
                unpack<T>(x, round.piece[j]);
                f(c, static_cast<int64_t>(c) * kChunk + threadIdx.x % kThreads * 8, x);
            }
        }
        round = next;
    }
}
template <typename T, typename F>
__device__ __forceinline__ void for_chunks(const typename Raw<T>::type* logits, int64_t vocab, int begin, int end, F f) {
    for_chunks<T>(logits, vocab, begin, end, load_round<T>(logits, vocab, begin, end), f);
}

// Order word of a token: larger comes first in (logit descending, id ascending).
__device__ __forceinline__ uint64_t order_word(float x, int64_t id) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t key = u ^ ((u & 0x80000000u) != 0 ? 0xffffffffu : 0x80000000u);
    return static_cast<uint64_t>(key) << kIdBits | (kIdMask - static_cast<uint64_t>(id));
}
__device__ __forceinline__ float order_logit(uint64_t word) {
    const uint32_t key = static_cast<uint32_t>(word >> kIdBits);
    return __uint_as_float(key ^ ((key & 0x80000000u) != 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int64_t order_id(uint64_t word) { return static_cast<int64_t>(kIdMask - (word & kIdMask)); }

// A row's settings.
struct Row {
    bool greedy;
    bool plain;      // top and scale are finite
    float top;       // largest logit
    double scale;    // 64 log2(e) / T: buckets of a logit
    int k;           // 0: off
    double p;        // 1: off
    uint64_t least;  // smallest weight that min_p lets pass
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t row) {
    Row r;
    const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.plain = false;
    r.top = 0.0f;
    r.scale = r.greedy ? 0.0 : kUnits * 0x1.71547652b82fep+0 / static_cast<double>(t);
    const int32_t k = a.top_k != nullptr ? a.top_k[row] : 0;
    r.k = k > 0 && k < a.vocab ? k : 0;  // (a row of one token has nothing to decide)
    const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
    r.p = p < 1.0f ? static_cast<double>(p) : 1.0;
    if (p <= 0.0f) {
        r.k = 1;  // the first token alone
        r.p = 1.0;
    }
    const float m = a.min_p != nullptr ? a.min_p[row] : 0.0f;
    const double least = m > 0.0f ? (m < 1.0f ? static_cast<double>(m) : 1.0) : 0.0;
    r.least = static_cast<uint64_t>(ceil(least * static_cast<double>(uint64_t{1} << kWeightBits)));
    return r;
}
__device__ __forceinline__ bool decides(const Row& r) { return r.k > 0 || r.p < 1.0; }
// Top-k that the largest logits of 128 ids each bound.
__device__ __forceinline__ bool bounded(const Row& r, int chunks) { return r.k > 0 && r.k <= chunks * kGroups; }

// Rows by the work that the second and third launch have with them, behind all rows'
// workspaces: where each class ends, then the rows class by class.
constexpr int kClasses = 4;  // all logits in both; all in the third alone; few; none
__device__ __forceinline__ int32_t* row_order(const SampleArgs& a, int chunks) {
    return reinterpret_cast<int32_t*>(a.workspace + a.rows * row_bytes(chunks));
}
__device__ __forceinline__ int class_of(const Row& r, int chunks) {
    if (r.greedy) {
        return 3;
    }
    return bounded(r, chunks) ? 2 : (decides(r) ? 0 : 1);
}

__device__ __forceinline__ void set_top(Row& r, uint64_t best) {
    r.top = order_logit(best);
    r.plain = fabsf(r.top) < __builtin_huge_valf() && r.scale < static_cast<double>(__builtin_huge_val());
}

// How far a logit lies below the largest, in buckets; kDepth: it weighs nothing.
__device__ __forceinline__ double depth_of(const Row& r, float x) {
    const double d = (static_cast<double>(r.top) - static_cast<double>(x)) * r.scale;
    const double within = d < kDepth && x > -__builtin_huge_valf() ? d : kDepth;  // (NaN: kDepth)
    return x == r.top ? 0.0 : within;
}
__device__ __forceinline__ int bucket_of(double depth) { return static_cast<int>(depth); }

// The least logit that may lie in a bucket below `buckets` (rounded down: a filter).
__device__ __forceinline__ float least_logit(const Row& r, int buckets) {
    if (r.top == __builtin_huge_valf()) {
        return r.top;
    }
    const double c = static_cast<double>(r.top) - (buckets + 1) / r.scale;
    return static_cast<float>(c - fabs(c) * 0x1p-23);
}
// Bits of the logits that are at least `least` (and above -inf).
__device__ __forceinline__ uint32_t passing(const float (&x)[8], float least) {
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mask |= x[i] >= least && x[i] > -__builtin_huge_valf() ? 1u << i : 0u;
    }
    return mask;
}
// Tokens before which the weights sum to less than this are in top_p of `total`.
__device__ __forceinline__ uint64_t top_p_end(const Row& r, uint64_t total) {
    return static_cast<uint64_t>(ceil(r.p * static_cast<double>(total)));
}
// One of 8 values by a running index.
__device__ __forceinline__ float pick(const float (&x)[8], int i) {
    const float a = (i & 1) != 0 ? x[1] : x[0];
    const float b = (i & 1) != 0 ? x[3] : x[2];
    const float c = (i & 1) != 0 ? x[5] : x[4];
    const float d = (i & 1) != 0 ? x[7] : x[6];
    const float e = (i & 2) != 0 ? b : a;
    const float f = (i & 2) != 0 ? d : c;
    return (i & 4) != 0 ? f : e;
}

// f(i, logit, depth) for the logits that `least` lets pass (f tells the ones that lie
// too deep): one by one where they are few, all eight in line where half of the
// wave's lanes have one.
template <typename F>
__device__ __forceinline__ void for_passing(const Row& r, const float (&x)[8], float least, F f) {
    const uint64_t lanes = __ballot(largest_of(x) >= least);
    if (lanes == 0) {
        return;
    }
    if (r.plain && __builtin_popcountll(lanes) >= 32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // (of a NaN and of -inf no number below any limit)
            f(i, x[i], (static_cast<double>(r.top) - static_cast<double>(x[i])) * r.scale);
        }
        return;
    }
    float settled[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        settled[i] = settle(x[i]);
    }
    for (uint32_t mask = passing(settled, least); mask != 0; mask &= mask - 1) {
        const int i = __builtin_ctz(mask);
        const float v = pick(settled, i);
        f(i, v, depth_of(r, v));
    }
}

// 2^(42 - depth / 64) rounded to a whole number, 0 <= depth < kDepth: a table's power
// for the whole buckets of the fraction, the Taylor polynomial of degree 5 of
// 2^(-z / 64) for the rest (z < 1: off by 2^-48.6), and the addition of 2^52 that rounds.
__device__ __forceinline__ uint64_t weight_of(double depth, const double* powers) {
    const int whole = static_cast<int>(depth);
    const double z = depth - whole;
    double e = -0x1.5d87fe78a6731p-40;  // (-ln 2 / 64)^n / n!
    e = fma(e, z, 0x1.3b2ab6fba4e77p-31);
    e = fma(e, z, -0x1.c6b08d704a0c0p-23);
    e = fma(e, z, 0x1.ebfbdff82c58fp-15);
    e = fma(e, z, -0x1.62e42fefa39efp-7);
    e = fma(e, z, 1.0);
    const double y = powers[whole % kUnits] * e;
    const int64_t shift = static_cast<int64_t>(kWeightBits - whole / kUnits) << 52;
    const double w = __longlong_as_double(__double_as_longlong(y) + shift) + 0x1p52;
    return static_cast<uint64_t>(__double_as_longlong(w)) & ((uint64_t{1} << 52) - 1);
}

// ------------------------------------------------------------ block helpers
__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Largest of a block's values, in every thread.
template <int WAVES = kWaves>
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* s_part) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        v = max_u64(v, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), o, 64)));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        s_part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = s_part[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        v = max_u64(v, s_part[w]);
    }
    return v;
}

// Sum of the values of the threads before this one; total in every thread.
template <typename V, int WAVES = kWaves>
__device__ __forceinline__ V block_before(V v, uint64_t* s_part, V& total) {
    V sum = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        V left;
        if constexpr (sizeof(V) == 8) {
            left = static_cast<V>(__shfl_up(static_cast<unsigned long long>(sum), o, 64));
        } else {
            left = static_cast<V>(__shfl_up(static_cast<unsigned int>(sum), o, 64));
        }
        sum += static_cast<int>(threadIdx.x & 63) >= o ? left : 0;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        s_part[threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        before += w < static_cast<int>(threadIdx.x >> 6) ? static_cast<V>(s_part[w]) : 0;
        total += static_cast<V>(s_part[w]);
    }
    return before + sum - v;
}
// Sum of a block's values, in every thread.
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* s_part) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        v += static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(v), o, 64));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        s_part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        v += s_part[w];
    }
    return v;
}

// The thread's largest of the first launch's blocks' order words.
__device__ __forceinline__ uint64_t load_best(const RowSpace& s, int blocks) {
    uint64_t v = 0;
    for (int i = threadIdx.x; i < blocks; i += static_cast<int>(blockDim.x)) {
        v = max_u64(v, s.best[i]);
    }
    return v;
}
// The block's copy of the powers.
__device__ __forceinline__ void load_powers(double* s_powers) {
    if (threadIdx.x < kUnits) {
        s_powers[threadIdx.x] = kPowers[threadIdx.x];
    }
}
__device__ __forceinline__ int chunks_end(int chunks, int per) {
    const int end = (static_cast<int>(blockIdx.x) + 1) * per;
    return end < chunks ? end : chunks;
}

// ---------------------------------------------------------------- launches
// By the first launch's first block.
__device__ __forceinline__ void write_order(const SampleArgs& a, int chunks) {
    __shared__ int s_total[kClasses];
    __shared__ int s_count[kWaves][kClasses];
    const int rows = static_cast<int>(a.rows);
    const int tid = static_cast<int>(threadIdx.x);
    int32_t* const order = row_order(a, chunks);
    if (tid < kClasses) {
        s_total[tid] = 0;
    }
    __syncthreads();
    for (int i = tid; i < rows; i += kThreads) {
        atomicAdd(&s_total[class_of(row_of(a, i), chunks)], 1);
    }
    __syncthreads();
    int at[kClasses];
    int end = 0;
#pragma unroll
    for (int c = 0; c < kClasses; ++c) {
        at[c] = end;
        end += s_total[c];
        if (tid == 0) {
            order[c] = end;
        }
    }
    for (int i0 = 0; i0 < rows; i0 += kThreads) {
        const int mine = i0 + tid < rows ? class_of(row_of(a, i0 + tid), chunks) : -1;
        int place = 0;
#pragma unroll
        for (int c = 0; c < kClasses; ++c) {
            const uint64_t same = __ballot(mine == c);
            if ((tid & 63) == 0) {
                s_count[tid >> 6][c] = __builtin_popcountll(same);
            }
            place = mine == c ? at[c] + __builtin_popcountll(same & ((uint64_t{1} << (tid & 63)) - 1)) : place;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kClasses; ++c) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                place += mine == c && w < (tid >> 6) ? s_count[w][c] : 0;
                at[c] += s_count[w][c];
            }
        }
        if (mine >= 0) {
            order[kClasses + place] = i0 + tid;
        }
        __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a, int chunks, int per, bool ordered) {
    __shared__ uint64_t s_part[kWaves];
    if (ordered && blockIdx.x == 0 && blockIdx.y == 0) {
        write_order(a, chunks);
    }
    const int64_t row = blockIdx.y;
    const RowSpace s = row_space(a.workspace, row, chunks);
    const int blocks = static_cast<int>(gridDim.x);
    for (int i = static_cast<int>(blockIdx.x) * kThreads + threadIdx.x; i < kBuckets; i += blocks * kThreads) {
        s.weights[i] = 0;
        s.counts[i] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x < 64) {
        s.coarse_weights[threadIdx.x] = 0;
        s.coarse_counts[threadIdx.x] = 0;
        if (threadIdx.x == 0) {
            *s.listed = 0;
        }
    }
    const auto* const logits = row_logits<T>(a, row);
    const int begin = static_cast<int>(blockIdx.x) * per;
    float best = -__builtin_huge_valf();
    int chunk = begin;  // the first that holds the thread's largest
    for_chunks<T>(logits, a.vocab, begin, chunks_end(chunks, per), [&](int c, int64_t, const float(&x)[8]) {
        float most = largest_of(x);
        chunk = most > best ? c : chunk;
        best = fmaxf(best, most);
        most = fmaxf(most, row_ror<8>(most));
        most = fmaxf(most, row_ror<4>(most));
        most = fmaxf(most, row_ror<2>(most));
        most = fmaxf(most, row_ror<1>(most));
        if (threadIdx.x % 16 == 0) {
            s.largest[c * kGroups + threadIdx.x / 16] = settle(most);
        }
    });
    // its place in the chunk's piece
    const int64_t id = static_cast<int64_t>(chunk) * kChunk + threadIdx.x * 8;
    uint64_t word = 0;
    if (id < a.vocab) {
        float x[8];
        unpack<T>(x, load_piece<T>(logits, id, a.vocab));
        int at = 0;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            at = settle(x[i]) == best ? i : at;
        }
        word = order_word(settle(best), id + at);
    }
    word = block_max(word, s_part);
    if (threadIdx.x == 0) {
        s.best[blockIdx.x] = word;
    }
}

// Large blocks: every block adds the buckets that it has filled to the row's, in
// memory that all XCDs share.
constexpr int kLarge = 1024;

template <typename T>
__global__ __launch_bounds__(kLarge) void sample_buckets_kernel(SampleArgs a, int chunks, int per, int max_blocks,
                                                                bool ordered) {
    constexpr int kStride = kLarge / kThreads;
    __shared__ unsigned long long s_weights[kBuckets];
    __shared__ uint32_t s_counts[kBuckets];
    __shared__ uint64_t s_part[kLarge / 64];
    __shared__ double s_powers[kUnits];
    __shared__ int s_limit;
    int64_t row = blockIdx.y;
    int part = static_cast<int>(blockIdx.x);
    if (ordered) {
        // (no more parts than blocks and, of one part each, rows: the grid has both)
        const int32_t* const order = row_order(a, chunks);
        const int dense = order[0];
        const int sparse = order[2] - order[1];
        const int total = kDenseShare * dense + sparse;
        const int blocks = static_cast<int>(gridDim.x - a.rows);
        const int most = (chunks + kStride - 1) / kStride;
        const auto parts_of = [&](int n) {
            const int v = total > 0 ? blocks * n / total : 1;
            return v < 1 ? 1 : (v < most ? v : most);
        };
        const int dense_parts = parts_of(kDenseShare);
        const bool is_dense = part < dense * dense_parts;
        const int parts = is_dense ? dense_parts : parts_of(1);
        const int place = is_dense ? part : part - dense * dense_parts;
        if (!is_dense && place >= sparse * parts) {
            return;
        }
        row = order[kClasses + (is_dense ? 0 : order[1]) + place / parts];
        part = place % parts;
        per = ((chunks + parts - 1) / parts + kStride - 1) / kStride * kStride;
        if (part * per >= chunks) {
            return;
        }
    }
    Row r = row_of(a, row);
    if (r.greedy || !decides(r)) {
        return;
    }
    const auto* const logits = row_logits<T>(a, row);
    const int begin = part * per + static_cast<int>(threadIdx.x) / kThreads;
    const int end = (part + 1) * per < chunks ? (part + 1) * per : chunks;
    const Round<T> round = load_round<T, kStride>(logits, a.vocab, begin, end);
    const RowSpace s = row_space(a.workspace, row, chunks);
    const uint64_t best = load_best(s, max_blocks);
    const int groups = chunks * kGroups;
    const bool by_groups = bounded(r, chunks);
    constexpr int kHeld = 2;  // largest logits of a thread that are requested at once
    float largest[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int at = i * kLarge + static_cast<int>(threadIdx.x);
        largest[i] = by_groups && at < groups ? s.largest[at] : -__builtin_huge_valf();
    }
    for (int i = threadIdx.x; i < kBuckets; i += kLarge) {
        s_weights[i] = 0;
        s_counts[i] = 0;
    }
    load_powers(s_powers);
    set_top(r, block_max<kLarge / 64>(best, s_part));
    int limit = kDepth;
    if (by_groups) {
        // k of the groups' largest logits are at least the k-th of them: the k-th token
        // lies no deeper
        if (threadIdx.x == 0) {
            s_limit = kDepth;
        }
        const auto put = [&](float x) __attribute__((always_inline)) {
            const double d = depth_of(r, x);
            if (d < kDepth) {
                atomicAdd(&s_counts[bucket_of(d)], 1u);
            }
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            put(largest[i]);
        }
        for (int i = kHeld * kLarge + threadIdx.x; i < groups; i += kLarge) {
            put(s.largest[i]);
        }
        __syncthreads();
        const int b0 = static_cast<int>(threadIdx.x) * kPer;
        uint32_t count[kPer];
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            count[i] = b0 < kBuckets ? s_counts[b0 + i] : 0;
            mine += count[i];
        }
        uint32_t total;
        uint32_t c = block_before<uint32_t, kLarge / 64>(mine, s_part, total);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (c < static_cast<uint32_t>(r.k) && c + count[i] >= static_cast<uint32_t>(r.k)) {
                s_limit = b0 + i + 1;
            }
            c += count[i];
            if (b0 < kBuckets) {
                s_counts[b0 + i] = 0;
            }
        }
        __syncthreads();
        limit = s_limit;
    }
    const float least = least_logit(r, limit);
    for_chunks<T, kStride>(logits, a.vocab, begin, end, round, [&](int, int64_t, const float(&x)[8]) {
        for_passing(r, x, least, [&](int, float, double d) __attribute__((always_inline)) {
            if (d < limit) {
                if (r.k > 0) {
                    atomicAdd(&s_counts[bucket_of(d)], 1u);
                }
                if (r.p < 1.0) {
                    atomicAdd(&s_weights[bucket_of(d)], static_cast<unsigned long long>(weight_of(d, s_powers)));
                }
            }
        });
    });
    __syncthreads();
    for (int i = threadIdx.x; i < kBuckets; i += kLarge) {
        uint32_t count = s_counts[i];
        uint64_t weight = s_weights[i];
        if (!__any(count != 0 || weight != 0)) {
            continue;
        }
        if (count != 0) {
            atomicAdd(&s.counts[i], count);
        }
        if (weight != 0) {
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[i]), static_cast<unsigned long long>(weight));
        }
        // the wave's buckets together
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            count += __shfl_xor(count, o, 64);
            weight += static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(weight), o, 64));
        }
        if ((threadIdx.x & 63) == 0) {
            atomicAdd(&s.coarse_counts[i / kCoarse], count);
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.coarse_weights[i / kCoarse]),
                      static_cast<unsigned long long>(weight));
        }
    }
}

// Sum over the wave's lanes up to this one.
template <typename V>
__device__ __forceinline__ V wave_until(V v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        V left;
        if constexpr (sizeof(V) == 8) {
            left = static_cast<V>(__shfl_up(static_cast<unsigned long long>(v), o, 64));
        } else {
            left = __shfl_up(v, o, 64);
        }
        v += static_cast<int>(threadIdx.x & 63) >= o ? left : 0;
    }
    return v;
}
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane);
    const uint32_t high = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane);
    return static_cast<uint64_t>(high) << 32 | low;
}
__device__ __forceinline__ int first_lane(bool v) { return __builtin_ctzll(__ballot(v) | uint64_t{1} << 63); }

// The deciding buckets, by every wave for itself: a lane holds the sums of kCoarse
// buckets, then one of the buckets that the sums point to.
__device__ __forceinline__ Decision decide(const Row& r, const RowSpace& s, uint32_t count, uint64_t weight) {
    const int lane = static_cast<int>(threadIdx.x & 63);
    Decision d{};
    const uint64_t weights = r.p < 1.0 ? wave_until(weight) : 0;
    const uint64_t all_weights = from_lane(weights, 63);
    // the bucket of the k-th token; top-k off or larger than the row: none
    d.k_bucket = kBuckets;
    d.k_weight = all_weights;
    uint64_t upper = all_weights;  // the most that the first top_k tokens can weigh
    const uint32_t k = static_cast<uint32_t>(r.k);
    if (r.k > 0) {
        const uint32_t counts = wave_until(count);
        if (static_cast<uint32_t>(__builtin_amdgcn_readlane(counts, 63)) >= k) {
            const int at = first_lane(counts >= k);
            const uint32_t fine = s.counts[at * kCoarse + lane];
            const uint64_t fine_weight = r.p < 1.0 ? s.weights[at * kCoarse + lane] : 0;
            const uint32_t until = static_cast<uint32_t>(__builtin_amdgcn_readlane(counts - count, at)) + wave_until(fine);
            const int of = first_lane(until >= k);
            d.k_bucket = at * kCoarse + of;
            d.k_count = __builtin_amdgcn_readlane(until - fine, of);
            if (r.p < 1.0) {
                const uint64_t w = from_lane(weights - weight, at) + wave_until(fine_weight);
                upper = from_lane(w, of);
                d.k_weight = from_lane(w - fine_weight, of);
            }
        }
    }
    d.low = d.k_bucket;
    d.high = d.k_bucket < kBuckets ? d.k_bucket : kBuckets - 1;
    d.low_weight = d.k_weight;
    if (r.p < 1.0) {
        // of the k-th token's bucket some of the weight counts, at most all of it
        const auto find = [&](uint64_t target, uint64_t& before) __attribute__((always_inline)) {
            const int at = first_lane(weights >= target);
            const uint64_t fine = s.weights[at * kCoarse + (at * kCoarse + lane < kBuckets ? lane : 0)];
            const uint64_t until = from_lane(weights - weight, at) + wave_until(fine);
            const int of = first_lane(until >= target);
            before = from_lane(until - fine, of);
            return at * kCoarse + of;
        };
        const uint64_t least = top_p_end(r, d.k_weight);
        const uint64_t most = top_p_end(r, upper);
        d.low = find(least, d.low_weight);
        uint64_t unused;
        d.high = least == most ? d.low : find(most, unused);
    }
    return d;
}

__device__ __forceinline__ bool listed_bucket(const Decision& d, int b) {
    return (b >= d.low && b <= d.high) || b == d.k_bucket;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_sums_kernel(SampleArgs a, int chunks, int per, int max_blocks, bool ordered) {
    __shared__ uint64_t s_part[kWaves];
    __shared__ uint64_t s_list[kList];
    __shared__ uint64_t s_sums[kWaves * kAhead];
    __shared__ double s_powers[kUnits];
    __shared__ uint32_t s_listed, s_at;
    // rows with the most work start first
    const int64_t row = ordered ? row_order(a, chunks)[kClasses + blockIdx.y] : static_cast<int64_t>(blockIdx.y);
    Row r = row_of(a, row);
    const RowSpace s = row_space(a.workspace, row, chunks);
    if (r.greedy && blockIdx.x != 0) {
        return;
    }
    // everything that does not wait for the decision is requested first
    const auto* const logits = row_logits<T>(a, row);
    const int begin = static_cast<int>(blockIdx.x) * per;
    const int end = chunks_end(chunks, per);
    const Round<T> round = load_round<T>(logits, a.vocab, begin, end);
    const uint64_t mine = load_best(s, max_blocks);
    const bool deciding = !r.greedy && decides(r);
    const int lane = static_cast<int>(threadIdx.x & 63);
    const uint32_t count = deciding ? s.coarse_counts[lane] : 0;
    const uint64_t weight = deciding ? s.coarse_weights[lane] : 0;
    const uint64_t best = block_max(mine, s_part);
    set_top(r, best);
    Decision d{};
    d.low = kBuckets;
    d.high = kBuckets - 1;
    d.k_bucket = kBuckets;
    if (deciding) {
        d = decide(r, s, count, weight);
    }
    d.best = best;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *s.decision = d;
    }
    if (r.greedy) {
        return;
    }
    if (threadIdx.x == 0) {
        s_listed = 0;
    }
    load_powers(s_powers);
    __syncthreads();
    const int deepest = d.low > kDepth ? kDepth : max(max(d.low, d.high), d.k_bucket < kBuckets ? d.k_bucket : 0) + 1;
    const float least = least_logit(r, deepest);
    int in_round = 0;
    for_chunks<T>(logits, a.vocab, begin, end, round, [&](int c, int64_t id, const float(&x)[8]) {
        uint64_t sum = 0;
        for_passing(r, x, least, [&](int i, float v, double depth) __attribute__((always_inline)) {
            if (depth < kDepth) {
                const int b = bucket_of(depth);
                if (b < d.low) {
                    const uint64_t w = weight_of(depth, s_powers);
                    sum += w >= r.least ? w : 0;
                } else if (listed_bucket(d, b)) {
                    const uint32_t at = atomicAdd(&s_listed, 1u);
                    if (at < kList) {
                        s_list[at] = order_word(settle(v), id + i);
                    }
                }
            }
        });
        // the waves' sums of a round of chunks meet at its end
        if (__any(sum != 0)) {
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) {
                sum += static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(sum), o, 64));
            }
        }
        if ((threadIdx.x & 63) == 0) {
            s_sums[in_round * kWaves + (threadIdx.x >> 6)] = sum;
        }
        if (++in_round == kAhead || c + 1 == end) {
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < in_round) {
                uint64_t total = 0;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    total += s_sums[threadIdx.x * kWaves + w];
                }
                s.sums[c + 1 - in_round + threadIdx.x] = total;
            }
            in_round = 0;
            __syncthreads();
        }
    });
    __syncthreads();
    // (tokens past the list are counted: the last launch does without it then)
    if (threadIdx.x == 0 && s_listed != 0) {
        s_at = atomicAdd(s.listed, s_listed);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < s_listed && i < kList && s_at + i < kList; i += kThreads) {
        s.list[s_at + i] = s_list[i];
    }
}

// ------------------------------------------------------------- the last launch
// The order word of the first of the block's tokens (those of `in`), in order, up to
// which their values reach the target, digit by digit from the first in which they
// differ, until one is left; 0: it is never reached.
template <int MINE>
__device__ __forceinline__ uint64_t select_in_list(const uint64_t (&word)[MINE], const uint64_t (&value)[MINE], uint32_t in,
                                                uint64_t before, uint64_t target, unsigned long long* s_bins,
                                                uint32_t* s_counts, uint64_t* s_part) {
    static_assert(kThreads == 256, "a thread a digit");
    __shared__ uint64_t s_prefix, s_before;
    __shared__ int s_found;  // tokens of the digit
    uint64_t largest = 0;
    uint64_t smallest = 0;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        largest = (in >> j & 1) != 0 ? max_u64(largest, word[j]) : largest;
        smallest = (in >> j & 1) != 0 ? max_u64(smallest, ~word[j]) : smallest;
    }
    largest = block_max(largest, s_part);
    smallest = ~block_max(smallest, s_part);
    if (largest < smallest) {
        return 0;  // none
    }
    int shift = largest == smallest ? 0 : 64 - __builtin_clzll(largest ^ smallest);
    uint64_t prefix = largest >> shift;
    do {
        const int bits = shift >= 8 ? 8 : shift;
        shift -= bits;
        __syncthreads();
        s_bins[threadIdx.x] = 0;
        s_counts[threadIdx.x] = 0;
        if (threadIdx.x == 0) {
            s_found = 0;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < MINE; ++j) {
            if ((in >> j & 1) != 0 && (word[j] >> shift) >> bits == prefix) {
                const int digit = static_cast<int>(word[j] >> shift) & ((1 << bits) - 1);
                atomicAdd(&s_bins[digit], static_cast<unsigned long long>(value[j]));
                atomicAdd(&s_counts[digit], 1u);
            }
        }
        __syncthreads();
        // bins from the highest digit down: thread i holds digit last - i
        const int digit = (1 << bits) - 1 - static_cast<int>(threadIdx.x);
        const uint64_t mine = digit >= 0 ? s_bins[digit] : 0;
        uint64_t total;
        const uint64_t until = before + block_before<uint64_t>(mine, s_part, total);
        if (until < target && until + mine >= target) {
            s_prefix = prefix << bits | static_cast<uint64_t>(digit);
            s_before = until;
            s_found = static_cast<int>(s_counts[digit]);
        }
        __syncthreads();
        if (s_found == 0) {
            return 0;
        }
        prefix = s_prefix;
        before = s_before;
    } while (shift > 0 && s_found > 1);
    // the one that has these digits
    uint64_t found = 0;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        found = (in >> j & 1) != 0 && word[j] >> shift == prefix ? word[j] : found;
    }
    return block_max(found, s_part);
}

// Where more tokens than the list holds share the deciding buckets (flat rows: high
// temperatures, or 16-bit logits so far from zero that thousands are equal):
// the order word of the first token, in order, up to which the count (k > 0) or the
// weight over buckets [low, high] reaches the target, digit by digit over the whole row;
// 0: it is never reached.  One block reads its row up to seven times: a call with such
// rows takes about a millisecond (151936 logits, top-p 0.95, bf16 normal logits around 16
// or at temperature 60: one row 1.0 ms, 128 1.1; with a top-k of 20000 1.5 and 1.7), where
// others take 26 to 110 us.
template <typename T>
__device__ __forceinline__ uint64_t select_in_row(const SampleArgs& a, const Row& r, const typename Raw<T>::type* logits,
                                               int low, int high, uint64_t before, int k, uint64_t target,
                                               unsigned long long* s_bins, uint64_t* s_part, const double* s_powers) {
    static_assert(kThreads == 256, "a thread a digit");
    __shared__ uint64_t s_prefix, s_before;
    __shared__ int s_found;
    uint64_t prefix = 0;
    int shift = 32 + kIdBits;
    while (shift > 0) {
        const int bits = shift >= 8 ? 8 : shift;
        shift -= bits;
        __syncthreads();
        s_bins[threadIdx.x] = 0;
        if (threadIdx.x == 0) {
            s_found = 0;
        }
        __syncthreads();
        for_chunks<T>(logits, a.vocab, 0, static_cast<int>((a.vocab + kChunk - 1) / kChunk),
                      [&](int, int64_t id, const float(&x)[8]) {
                          for (int i = 0; i < 8; ++i) {
                              const float v = settle(x[i]);
                              const double depth = depth_of(r, v);
                              if (depth < kDepth) {
                                  const int b = bucket_of(depth);
                                  const uint64_t word = order_word(v, id + i);
                                  if (b >= low && b <= high && (word >> shift) >> bits == prefix) {
                                      atomicAdd(&s_bins[(word >> shift) & ((1u << bits) - 1)],
                                                static_cast<unsigned long long>(k > 0 ? 1 : weight_of(depth, s_powers)));
                                  }
                              }
                          }
                      });
        __syncthreads();
        // bins from the highest digit down: thread i holds digit last - i
        const int digit = (1 << bits) - 1 - static_cast<int>(threadIdx.x);
        const uint64_t mine = digit >= 0 ? s_bins[digit] : 0;
        uint64_t total;
        const uint64_t until = before + block_before<uint64_t>(mine, s_part, total);
        if (until < target && until + mine >= target) {
            s_prefix = prefix << bits | static_cast<uint64_t>(digit);
            s_before = until;
            s_found = 1;
        }
        __syncthreads();
        if (s_found == 0) {
            return 0;
        }
        prefix = s_prefix;
        before = s_before;
    }
    return prefix;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_finish_kernel(SampleArgs a, int chunks) {
    constexpr int kMine = kList / kThreads;  // list entries of a thread
    __shared__ uint64_t s_part[kWaves];
    __shared__ uint64_t s_list[kList];
    __shared__ uint64_t s_weights[kThreads];
    __shared__ unsigned long long s_sums[kMaxChunks];
    __shared__ unsigned long long s_bins[kThreads];
    __shared__ uint32_t s_counts[kThreads];
    __shared__ double s_powers[kUnits];
    __shared__ uint64_t s_last, s_rest;
    __shared__ int s_chunk;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    Row r = row_of(a, row);
    const RowSpace s = row_space(a.workspace, row, chunks);
    const Decision d = *s.decision;
    const float u = a.random[row];
    const uint64_t listed = s.list[tid];  // (of no use where the list is shorter)
    set_top(r, d.best);
    if (r.greedy || r.top == -__builtin_huge_valf()) {
        if (tid == 0) {
            const bool none = r.top == -__builtin_huge_valf();  // no token: no logit above -inf
            a.tokens[row] = none ? 0 : static_cast<int32_t>(order_id(d.best));
            if (a.chances != nullptr) {
                a.chances[row] = none ? 0.0f : 1.0f;
            }
        }
        return;
    }
    const auto* const logits = row_logits<T>(a, row);
    const int n = static_cast<int>(*s.listed);
    uint64_t last = 0;  // order word of the last kept token
    load_powers(s_powers);
    for (int c = tid; c < chunks; c += kThreads) {
        s_sums[c] = s.sums[c];
    }
    if (tid == 0) {
        s_last = 0;
    }
    if (n > 0 && n <= kThreads) {
        // a token a thread: what comes before it, by comparing it with every other
        const uint64_t word = tid < n ? listed : 0;
        __syncthreads();
        const double depth = tid < n ? depth_of(r, order_logit(word)) : 0.0;
        const uint64_t weight = tid < n ? weight_of(depth, s_powers) : 0;
        const int b = tid < n ? bucket_of(depth) : -1;
        const bool in_k = b == d.k_bucket;
        const bool in_p = b >= d.low && b <= d.high;
        s_list[tid] = word;
        s_weights[tid] = weight | static_cast<uint64_t>(in_k) << 63 | static_cast<uint64_t>(in_p) << 62;
        __syncthreads();
        uint32_t rank = 0;
        uint64_t before = d.low_weight;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const uint64_t w = s_weights[j];
            const bool earlier = s_list[j] > word;
            rank += earlier ? static_cast<uint32_t>(w >> 63) : 0;
            before += earlier && (w >> 62 & 1) != 0 ? w & ((uint64_t{1} << 62) - 1) : 0;
        }
        uint64_t k_weight = d.k_weight;
        if (d.k_bucket < kBuckets) {
            const int place = d.k_count + static_cast<int>(rank);
            k_weight += block_sum(in_k && place < r.k ? weight : 0, s_part);
            if (in_k && place + 1 == r.k) {
                s_last = word;
            }
        }
        __syncthreads();
        last = s_last;
        if (r.p < 1.0) {
            // the last token with less than the target before it: the smallest word
            const bool under = in_p && before < top_p_end(r, k_weight);
            last = max_u64(last, ~block_max(under ? ~word : 0, s_part));
        }
    } else if (n > 0 && n <= kList) {
        uint64_t word[kMine], weight[kMine];
        uint32_t in_k = 0;
        uint32_t in_p = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int i = j * kThreads + tid;
            word[j] = i < n ? s.list[i] : 0;
            s_list[i] = word[j];
            const double depth = i < n ? depth_of(r, order_logit(word[j])) : 0.0;
            weight[j] = i < n ? weight_of(depth, s_powers) : 0;
            const int b = i < n ? bucket_of(depth) : -1;
            in_k |= b == d.k_bucket ? 1u << j : 0u;
            in_p |= b >= d.low && b <= d.high ? 1u << j : 0u;
        }
        uint64_t k_weight = d.k_weight;
        if (d.k_bucket < kBuckets) {
            uint64_t one[kMine];
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                one[j] = 1;
            }
            last = select_in_list<kMine>(word, one, in_k, static_cast<uint64_t>(d.k_count), static_cast<uint64_t>(r.k), s_bins,
                                         s_counts, s_part);
            uint64_t mine = 0;
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                mine += (in_k >> j & 1) != 0 && word[j] >= last ? weight[j] : 0;
            }
            k_weight += block_sum(mine, s_part);
        }
        if (r.p < 1.0) {
            last = max_u64(last, select_in_list<kMine>(word, weight, in_p, d.low_weight, top_p_end(r, k_weight), s_bins,
                                                       s_counts, s_part));
        }
    } else if (n > kList) {
        __syncthreads();
        uint64_t k_weight = d.k_weight;
        if (d.k_bucket < kBuckets) {
            last = select_in_row<T>(a, r, logits, d.k_bucket, d.k_bucket, static_cast<uint64_t>(d.k_count), r.k,
                                    static_cast<uint64_t>(r.k), s_bins, s_part, s_powers);
            uint64_t mine = 0;
            for_chunks<T>(logits, a.vocab, 0, chunks, [&](int, int64_t id, const float(&x)[8]) {
                for (int i = 0; i < 8; ++i) {
                    const float v = settle(x[i]);
                    const double depth = depth_of(r, v);
                    if (depth < kDepth && bucket_of(depth) == d.k_bucket && order_word(v, id + i) >= last) {
                        mine += weight_of(depth, s_powers);
                    }
                }
            });
            k_weight += block_sum(mine, s_part);
        }
        if (r.p < 1.0) {
            last = max_u64(last, select_in_row<T>(a, r, logits, d.low, d.high, d.low_weight, 0,
                                                  top_p_end(r, k_weight), s_bins, s_part, s_powers));
        }
    }
    // the first token stays, whatever the settings
    last = last < d.best ? last : d.best;
    __syncthreads();
    if (n > 0 && n <= kList) {
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t word = s_list[i];
            const uint64_t w = weight_of(depth_of(r, order_logit(word)), s_powers);
            if (word >= last && w >= r.least) {
                atomicAdd(&s_sums[order_id(word) / kChunk], static_cast<unsigned long long>(w));
            }
        }
    } else if (n > kList) {
        for_chunks<T>(logits, a.vocab, 0, chunks, [&](int c, int64_t id, const float(&x)[8]) {
            uint64_t sum = 0;
            for (int i = 0; i < 8; ++i) {
                const float v = settle(x[i]);
                const double depth = depth_of(r, v);
                if (depth < kDepth && bucket_of(depth) >= d.low && order_word(v, id + i) >= last) {
                    const uint64_t w = weight_of(depth, s_powers);
                    sum += w >= r.least ? w : 0;
                }
            }
            atomicAdd(&s_sums[c], static_cast<unsigned long long>(sum));
        });
    }
    __syncthreads();
    // the chunk that u falls on
    static_assert(kMaxChunks == 2 * kThreads, "two chunks a thread");
    const uint64_t first = 2 * tid < chunks ? s_sums[2 * tid] : 0;
    const uint64_t second = 2 * tid + 1 < chunks ? s_sums[2 * tid + 1] : 0;
    uint64_t total;
    const uint64_t before = block_before<uint64_t>(first + second, s_part, total);
    const double share = u > 0.0f ? (u < 1.0f ? static_cast<double>(u) : 1.0) : 0.0;
    uint64_t target = static_cast<uint64_t>(share * static_cast<double>(total));
    target = target < total ? target : total - 1;
    if (before <= target && target < before + first + second) {
        const bool later = target >= before + first;
        s_chunk = 2 * tid + (later ? 1 : 0);
        s_rest = target - before - (later ? first : 0);
    }
    __syncthreads();
    const int64_t id = static_cast<int64_t>(s_chunk) * kChunk + tid * 8;
    const uint64_t rest = s_rest;
    float x[8];
    unpack<T>(x, load_piece<T>(logits, id, a.vocab));
    uint64_t w[8];
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = settle(x[i]);
        const double depth = id + i < a.vocab ? depth_of(r, v) : kDepth;
        w[i] = depth < kDepth ? weight_of(depth, s_powers) : 0;
        w[i] = w[i] >= r.least && order_word(v, id + i) >= last ? w[i] : 0;
        mine += w[i];
    }
    uint64_t all;
    uint64_t from = block_before<uint64_t>(mine, s_part, all);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (from <= rest && rest < from + w[i]) {
            a.tokens[row] = static_cast<int32_t>(id + i);
            if (a.chances != nullptr) {
                a.chances[row] = static_cast<float>(static_cast<double>(w[i]) / static_cast<double>(total));
            }
        }
        from += w[i];
    }
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
    const int chunks = static_cast<int>((a.vocab + kChunk - 1) / kChunk);
    // with few rows a chunk a block (the large blocks: four), at most about the blocks
    // that the chip holds at a time
    const auto share = [&](int64_t most, int64_t least) {
        const int64_t per = (chunks * a.rows + most - 1) / most;
        return static_cast<int>(per > least ? per : least);
    };
    const auto grid = [&](int per) {
        return dim3(static_cast<unsigned>((chunks + per - 1) / per), static_cast<unsigned>(a.rows));
    };
    const int per = share(kBlocks, 1);
    const int large = share(kLargeBlocks, kLarge / kThreads);
    const int blocks = static_cast<int>(grid(per).x);
    const bool ordered = a.rows >= kOrderedRows;
    hipLaunchKernelGGL(sample_max_kernel<T>, grid(per), dim3(kThreads), 0, stream, a, chunks, per, ordered);
    hipError_t status = hipGetLastError();
    if (status == hipSuccess && (a.top_k != nullptr || a.top_p != nullptr)) {
        const dim3 shared(static_cast<unsigned>(kLargeBlocks + a.rows));
        hipLaunchKernelGGL(sample_buckets_kernel<T>, ordered ? shared : grid(large), dim3(kLarge), 0, stream, a, chunks, large,
                           blocks, ordered);
        status = hipGetLastError();
    }
    if (status == hipSuccess) {
        hipLaunchKernelGGL(sample_sums_kernel<T>, grid(per), dim3(kThreads), 0, stream, a, chunks, per, blocks, ordered);
        status = hipGetLastError();
    }
    if (status == hipSuccess) {
        hipLaunchKernelGGL(sample_finish_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, stream, a, chunks);
        status = hipGetLastError();
    }
    return status;
}

}  // namespace

int64_t sample_workspace_bytes(int64_t rows, int64_t vocab) {
    const int64_t bytes = row_bytes((vocab + kChunk - 1) / kChunk);
    return rows * bytes + (kClasses + rows + 3) / 4 * 16;
}

hipError_t launch_sample(int dtype, const SampleArgs& a, hipStream_t stream) {
    if (dtype == 0) {
        return launch<F32>(a, stream);
    }
    return dtype == 1 ? launch<Bf16>(a, stream) : launch<F16>(a, stream);
}

}  // namespace kc
