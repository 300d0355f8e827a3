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
// No row is sorted.  Tokens fall into 2048 buckets by log2 w; which bucket ends
// the kept tokens follows from the buckets' counts and sums, and only that
// bucket's tokens (tens to hundreds of them) are ordered.  Launches, each over
// (blocks of a row, rows):
//   1. the row's largest logit;  2. buckets (for top-k and top-p);
//   3. tokens of the deciding buckets to a list, sums of the surely kept tokens
//      of each chunk of 2048 ids;  4. one block a row: the list ordered, the last
//      kept token, the chunk and in it the token that u falls on.
// The row is read by the first three (once from memory, then from the caches) and
// one chunk of it by the last.
#include "kc_device.h"
#include "kc_kernels.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8 * kThreads;  // ids of a chunk: 8 a thread
constexpr int kBuckets = 2048;
constexpr int kList = 2048;           // most tokens that are ordered in LDS
constexpr int kFinish = 1024;         // threads of the last launch
constexpr int kWeightBits = 42;
constexpr double kDepth = 43.0;       // log2 of the weights' range
constexpr int kMaxChunks = static_cast<int>(kSampleMaxVocab / kChunk);
constexpr int kIdBits = 20;
constexpr uint64_t kIdMask = (uint64_t{1} << kIdBits) - 1;
static_assert(kSampleMaxVocab <= (int64_t{1} << kIdBits), "ids of an order word");

// What launch 3 tells launch 4 of a row's deciding buckets.
struct Decision {
    int32_t low;         // tokens of buckets below are kept (if min_p lets them)
    int32_t high;        // [low, high]: top-p, or the bucket of the k-th token, decides
    int32_t k_bucket;    // bucket of the k-th token (kBuckets: top-k off or too large)
    int32_t listed;      // tokens of these buckets
    uint64_t k_weight;   // weights and tokens of the buckets before k_bucket (of all: top-k off)
    int64_t k_count;
    uint64_t low_weight;  // weights of the buckets before low
};

// Workspace of a row, in this order.
struct RowSpace {
    uint64_t* weights;   // [kBuckets]
    uint32_t* counts;    // [kBuckets]
    uint64_t* list;      // [kList] order words
    uint64_t* sums;      // [chunks]
    uint64_t* best;      // [chunks] order word of each block's largest logit
    Decision* decision;
    uint32_t* listed;
};
__host__ __device__ inline int64_t row_bytes(int64_t chunks) {
    return kBuckets * 12 + kList * 8 + chunks * 16 + 64 + 16;
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
    s.counts = reinterpret_cast<uint32_t*>(p);
    return s;
}
static_assert(sizeof(Decision) <= 64, "the row's workspace");

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

// 8 logits from id on; -inf where the row ends.  NaN counts as -inf, -0 as 0.
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const typename Raw<T>::type* row, int64_t id, int64_t vocab) {
    typedef typename Raw<T>::type raw;
    const raw* p = row + id;
    if (id + 8 <= vocab && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        raw v[8];
        uint4 w[sizeof(raw) / 2];
#pragma unroll
        for (unsigned i = 0; i < sizeof(raw) / 2; ++i) {
            w[i] = reinterpret_cast<const uint4*>(p)[i];
        }
        __builtin_memcpy(v, w, sizeof(v));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = T::load(v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = id + i < vocab ? T::load(p[i]) : -__builtin_huge_valf();
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = x[i] == x[i] ? x[i] + 0.0f : -__builtin_huge_valf();
    }
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
    float top;       // largest logit
    double scale;    // log2(e) / T
    int64_t k;       // 0: off
    double p;        // >= 1: off
    uint64_t least;  // smallest weight that min_p lets pass
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t row) {
    Row r;
    const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.top = 0.0f;
    r.scale = r.greedy ? 0.0 : 0x1.71547652b82fep+0 / static_cast<double>(t);
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

// How far a logit lies below the largest, in log2 of the weight; >= kDepth: no weight.
__device__ __forceinline__ double depth_of(const Row& r, float x) {
    if (x == r.top) {
        return 0.0;
    }
    const double d = (static_cast<double>(r.top) - static_cast<double>(x)) * r.scale;
    return d == d && x > -__builtin_huge_valf() ? d : kDepth;
}
__device__ __forceinline__ int bucket_of(double depth) {
    const int b = static_cast<int>(depth * (kBuckets / kDepth));
    return b < kBuckets ? b : kBuckets - 1;  // (the product may round up to kBuckets)
}

// 2^(42 - depth) rounded to a whole number, 0 <= depth < 43: e^z of the fraction
// less a half by its Taylor polynomial of degree 12 (|z| <= 0.35: 2^-52).
__device__ __forceinline__ uint64_t weight_of(double depth) {
    const double y = kWeightBits - depth;
    const double n = floor(y);
    const double z = (y - n - 0.5) * 0x1.62e42fefa39efp-1;
    double e = 1.0 / 479001600.0;
    e = fma(e, z, 1.0 / 39916800.0);
    e = fma(e, z, 1.0 / 3628800.0);
    e = fma(e, z, 1.0 / 362880.0);
    e = fma(e, z, 1.0 / 40320.0);
    e = fma(e, z, 1.0 / 5040.0);
    e = fma(e, z, 1.0 / 720.0);
    e = fma(e, z, 1.0 / 120.0);
    e = fma(e, z, 1.0 / 24.0);
    e = fma(e, z, 1.0 / 6.0);
    e = fma(e, z, 0.5);
    e = fma(e, z, 1.0);
    e = fma(e, z, 1.0) * 0x1.6a09e667f3bcdp+0;
    return static_cast<uint64_t>(ldexp(e, static_cast<int>(n)) + 0.5);
}

// ------------------------------------------------------------ block helpers
__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Largest of a block's values, in every thread.
template <int WAVES>
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
template <int WAVES>
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t* s_part, uint64_t& total) {
    uint64_t sum = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t left = static_cast<uint64_t>(__shfl_up(static_cast<unsigned long long>(sum), o, 64));
        sum += static_cast<int>(threadIdx.x & 63) >= o ? left : 0;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        s_part[threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        before += w < static_cast<int>(threadIdx.x >> 6) ? s_part[w] : 0;
        total += s_part[w];
    }
    return before + sum - v;
}

template <typename T>
__device__ __forceinline__ const typename Raw<T>::type* row_logits(const SampleArgs& a, int64_t row) {
    return static_cast<const typename Raw<T>::type*>(a.logits) + row * a.stride;
}

// The row's largest logit and its order word from the first launch's blocks.
template <int WAVES>
__device__ __forceinline__ uint64_t row_best(const RowSpace& s, int blocks, uint64_t* s_part) {
    uint64_t v = 0;
    for (int i = threadIdx.x; i < blocks; i += WAVES * 64) {
        v = max_u64(v, s.best[i]);
    }
    return block_max<WAVES>(v, s_part);
}

// ---------------------------------------------------------------- launches
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a, int chunks, int per) {
    __shared__ uint64_t s_part[kThreads / 64];
    const int64_t row = blockIdx.y;
    const RowSpace s = row_space(a.workspace, row, chunks);
    const int blocks = static_cast<int>(gridDim.x);
    for (int i = static_cast<int>(blockIdx.x) * kThreads + threadIdx.x; i < kBuckets; i += blocks * kThreads) {
        s.weights[i] = 0;
        s.counts[i] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *s.listed = 0;
    }
    const auto* const logits = row_logits<T>(a, row);
    const int end = (static_cast<int>(blockIdx.x) + 1) * per < chunks ? (static_cast<int>(blockIdx.x) + 1) * per : chunks;
    uint64_t best = 0;
    for (int c = static_cast<int>(blockIdx.x) * per; c < end; ++c) {
        const int64_t id = static_cast<int64_t>(c) * kChunk + threadIdx.x * 8;
        if (id < a.vocab) {
            float x[8];
            load8<T>(x, logits, id, a.vocab);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                best = max_u64(best, id + i < a.vocab ? order_word(x[i], id + i) : 0);
            }
        }
    }
    best = block_max<kThreads / 64>(best, s_part);
    if (threadIdx.x == 0) {
        s.best[blockIdx.x] = best;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_buckets_kernel(SampleArgs a, int chunks, int per) {
    __shared__ unsigned long long s_weights[kBuckets];
    __shared__ uint32_t s_counts[kBuckets];
    __shared__ uint64_t s_part[kThreads / 64];
    const int64_t row = blockIdx.y;
    Row r = row_of(a, row);
    if (r.greedy || !decides(r)) {
        return;
    }
    for (int i = threadIdx.x; i < kBuckets; i += kThreads) {
        s_weights[i] = 0;
        s_counts[i] = 0;
    }
    const RowSpace s = row_space(a.workspace, row, chunks);
    r.top = order_logit(row_best<kThreads / 64>(s, static_cast<int>(gridDim.x), s_part));
    const auto* const logits = row_logits<T>(a, row);
    const int end = (static_cast<int>(blockIdx.x) + 1) * per < chunks ? (static_cast<int>(blockIdx.x) + 1) * per : chunks;
    for (int c = static_cast<int>(blockIdx.x) * per; c < end; ++c) {
        const int64_t id = static_cast<int64_t>(c) * kChunk + threadIdx.x * 8;
        if (id < a.vocab) {
            float x[8];
            load8<T>(x, logits, id, a.vocab);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double d = depth_of(r, x[i]);
                if (d < kDepth) {
                    atomicAdd(&s_counts[bucket_of(d)], 1u);
                    if (r.p < 1.0) {
                        atomicAdd(&s_weights[bucket_of(d)], static_cast<unsigned long long>(weight_of(d)));
                    }
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBuckets; i += kThreads) {
        if (s_counts[i] != 0) {
            atomicAdd(&s.counts[i], s_counts[i]);
            if (r.p < 1.0) {
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.weights[i]), s_weights[i]);
            }
        }
    }
}

// The deciding buckets, from the row's counts and weights (all threads of a block).
__device__ __forceinline__ Decision decide(const Row& r, const RowSpace& s, uint64_t* s_part, Decision* s_decision) {
    constexpr int kPer = kBuckets / kThreads;
    constexpr int kWaves = kThreads / 64;
    const int b0 = static_cast<int>(threadIdx.x) * kPer;
    uint32_t count[kPer];
    uint64_t weight[kPer];
    uint64_t counts = 0;
    uint64_t weights = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        count[i] = s.counts[b0 + i];
        weight[i] = s.weights[b0 + i];
        counts += count[i];
        weights += weight[i];
    }
    uint64_t all_counts, all_weights;
    const uint64_t counts_before = block_before<kWaves>(counts, s_part, all_counts);
    const uint64_t weights_before = block_before<kWaves>(weights, s_part, all_weights);
    if (threadIdx.x == 0) {
        s_decision->k_bucket = kBuckets;
        s_decision->k_weight = all_weights;
        s_decision->k_count = static_cast<int64_t>(all_counts);
        s_decision->low = kBuckets;
        s_decision->high = kBuckets - 1;
        s_decision->low_weight = all_weights;
        s_decision->listed = 0;
    }
    __shared__ uint64_t s_upper;  // the most that the first top_k tokens can weigh
    if (threadIdx.x == 0) {
        s_upper = all_weights;
    }
    __syncthreads();
    if (r.k > 0) {
        uint64_t c = counts_before;
        uint64_t w = weights_before;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (c < static_cast<uint64_t>(r.k) && c + count[i] >= static_cast<uint64_t>(r.k)) {
                s_decision->k_bucket = b0 + i;
                s_decision->k_weight = w;
                s_decision->k_count = static_cast<int64_t>(c);
                s_decision->low = b0 + i;
                s_decision->high = b0 + i;
                s_decision->low_weight = w;
                s_upper = w + weight[i];
            }
            c += count[i];
            w += weight[i];
        }
    }
    __syncthreads();
    if (r.p < 1.0) {
        // the k-th token's bucket holds some of its weight, at most all of it
        const double least = r.p * static_cast<double>(s_decision->k_weight);
        const double most = r.p * static_cast<double>(s_upper);
        uint64_t w = weights_before;
        bool is_low[kPer], is_high[kPer];
        uint64_t low_weight = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const bool first = b0 + i == 0;
            const double before = static_cast<double>(w);
            const double after = static_cast<double>(w + weight[i]);
            is_low[i] = after >= least && (first || before < least);
            is_high[i] = after >= most && (first || before < most);
            low_weight = is_low[i] ? w : low_weight;
            w += weight[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (is_low[i]) {
                s_decision->low = b0 + i;
                s_decision->low_weight = low_weight;
            }
            if (is_high[i]) {
                s_decision->high = b0 + i;
            }
        }
    }
    __syncthreads();
    uint64_t listed = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int b = b0 + i;
        listed += (b >= s_decision->low && b <= s_decision->high) || b == s_decision->k_bucket ? count[i] : 0;
    }
    uint64_t all_listed;
    (void)block_before<kWaves>(listed, s_part, all_listed);
    if (threadIdx.x == 0) {
        s_decision->listed = static_cast<int32_t>(all_listed);
    }
    __syncthreads();
    return *s_decision;
}

__device__ __forceinline__ bool listed_bucket(const Decision& d, int b) {
    return (b >= d.low && b <= d.high) || b == d.k_bucket;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_sums_kernel(SampleArgs a, int chunks, int per) {
    __shared__ uint64_t s_part[kThreads / 64];
    __shared__ uint64_t s_list[kList];
    __shared__ Decision s_decision;
    __shared__ uint32_t s_listed, s_at;
    const int64_t row = blockIdx.y;
    Row r = row_of(a, row);
    if (r.greedy) {
        return;
    }
    const RowSpace s = row_space(a.workspace, row, chunks);
    r.top = order_logit(row_best<kThreads / 64>(s, static_cast<int>(gridDim.x), s_part));
    Decision d{};
    d.low = kBuckets;
    d.high = kBuckets - 1;
    d.k_bucket = kBuckets;
    if (decides(r)) {
        d = decide(r, s, s_part, &s_decision);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *s.decision = d;
    }
    if (threadIdx.x == 0) {
        s_listed = 0;
    }
    __syncthreads();
    const auto* const logits = row_logits<T>(a, row);
    const int end = (static_cast<int>(blockIdx.x) + 1) * per < chunks ? (static_cast<int>(blockIdx.x) + 1) * per : chunks;
    for (int c = static_cast<int>(blockIdx.x) * per; c < end; ++c) {
        const int64_t id = static_cast<int64_t>(c) * kChunk + threadIdx.x * 8;
        uint64_t sum = 0;
        if (id < a.vocab) {
            float x[8];
            load8<T>(x, logits, id, a.vocab);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double depth = depth_of(r, x[i]);
                if (depth < kDepth) {
                    const int b = bucket_of(depth);
                    if (b < d.low) {
                        const uint64_t w = weight_of(depth);
                        sum += w >= r.least ? w : 0;
                    } else if (d.listed <= kList && listed_bucket(d, b)) {
                        s_list[atomicAdd(&s_listed, 1u) % kList] = order_word(x[i], id + i);
                    }
                }
            }
        }
        uint64_t total;
        (void)block_before<kThreads / 64>(sum, s_part, total);
        if (threadIdx.x == 0) {
            s.sums[c] = total;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && s_listed != 0) {
        s_at = atomicAdd(s.listed, s_listed);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < s_listed; i += kThreads) {
        s.list[s_at + i] = s_list[i];
    }
}

// ------------------------------------------------------------- the last launch
// Where more tokens than the list holds share the deciding buckets (flat rows):
// the order word of the first token, in order, up to which count (k > 0) or weight
// over buckets [low, high] reaches the target, digit by digit over the whole row;
// 0: it is never reached.
template <typename T>
__device__ __noinline__ uint64_t select_in_row(const SampleArgs& a, const Row& r, const typename Raw<T>::type* logits,
                                               int low, int high, uint64_t before, int64_t k, double target,
                                               unsigned long long* s_bins, uint64_t* s_part) {
    constexpr int kWaves = kFinish / 64;
    __shared__ uint64_t s_prefix, s_before;
    __shared__ int s_found;
    uint64_t prefix = 0;
    int shift = 52;
    while (shift > 0) {
        const int bits = shift >= 8 ? 8 : shift;
        shift -= bits;
        __syncthreads();
        if (threadIdx.x < 256) {
            s_bins[threadIdx.x] = 0;
        }
        if (threadIdx.x == 0) {
            s_found = 0;
        }
        __syncthreads();
        for (int64_t id = threadIdx.x * 8; id < a.vocab; id += kFinish * 8) {
            float x[8];
            load8<T>(x, logits, id, a.vocab);
            for (int i = 0; i < 8; ++i) {
                const double depth = depth_of(r, x[i]);
                if (depth < kDepth) {
                    const int b = bucket_of(depth);
                    const uint64_t word = order_word(x[i], id + i);
                    if (b >= low && b <= high && (word >> shift) >> bits == prefix) {
                        atomicAdd(&s_bins[(word >> shift) & ((1u << bits) - 1)],
                                  static_cast<unsigned long long>(k > 0 ? 1 : weight_of(depth)));
                    }
                }
            }
        }
        __syncthreads();
        // bins from the highest digit down: thread i holds digit last - i
        const int last = (1 << bits) - 1;
        const int digit = last - static_cast<int>(threadIdx.x);
        const uint64_t mine = digit >= 0 ? s_bins[digit] : 0;
        uint64_t total;
        const uint64_t until = before + block_before<kWaves>(mine, s_part, total);
        const bool short_of = k > 0 ? until < static_cast<uint64_t>(k) : static_cast<double>(until) < target;
        const bool reaches = k > 0 ? until + mine >= static_cast<uint64_t>(k) : static_cast<double>(until + mine) >= target;
        if (mine != 0 && short_of && reaches) {
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
__global__ __launch_bounds__(kFinish) void sample_finish_kernel(SampleArgs a, int chunks, int blocks) {
    constexpr int kWaves = kFinish / 64;
    __shared__ uint64_t s_part[kWaves];
    __shared__ uint64_t s_list[kList];
    __shared__ unsigned long long s_sums[kMaxChunks];
    __shared__ unsigned long long s_bins[256];
    __shared__ uint64_t s_last, s_rest;
    __shared__ int s_chunk;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    Row r = row_of(a, row);
    const RowSpace s = row_space(a.workspace, row, chunks);
    const uint64_t best = row_best<kWaves>(s, blocks, s_part);
    r.top = order_logit(best);
    if (r.greedy || r.top == -__builtin_huge_valf()) {
        if (tid == 0) {
            const bool none = r.top == -__builtin_huge_valf();  // no token: no logit above -inf
            a.tokens[row] = none ? 0 : static_cast<int32_t>(order_id(best));
            if (a.chances != nullptr) {
                a.chances[row] = none ? 0.0f : 1.0f;
            }
        }
        return;
    }
    const auto* const logits = row_logits<T>(a, row);
    const Decision d = *s.decision;
    const int n = d.listed;
    uint64_t last = 0;  // order word of the last kept token
    for (int c = tid; c < chunks; c += kFinish) {
        s_sums[c] = s.sums[c];
    }
    if (n > 0 && n <= kList) {
        // the list in order: a bitonic network over the next power of two
        int size = 2;
        while (size < n) {
            size *= 2;
        }
        for (int i = tid; i < size; i += kFinish) {
            s_list[i] = i < n ? s.list[i] : 0;
        }
        for (int width = 2; width <= size; width *= 2) {
            for (int step = width / 2; step >= 1; step /= 2) {
                __syncthreads();
                for (int i = tid; i < size / 2; i += kFinish) {
                    const int x = 2 * i - (i & (step - 1));
                    const int y = x + step;
                    const bool down = (x & width) == 0;
                    const uint64_t u = s_list[x];
                    const uint64_t v = s_list[y];
                    if ((u < v) == down) {
                        s_list[x] = v;
                        s_list[y] = u;
                    }
                }
            }
        }
        if (tid == 0) {
            s_last = 0;
        }
        __syncthreads();
        // two tokens a thread: weights, and which buckets they are in
        uint64_t word[2], weight[2];
        bool in_k[2], in_p[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * tid + j;
            word[j] = i < n ? s_list[i] : 0;
            const double depth = i < n ? depth_of(r, order_logit(word[j])) : kDepth;
            weight[j] = i < n ? weight_of(depth) : 0;
            const int b = i < n ? bucket_of(depth) : -1;
            in_k[j] = b == d.k_bucket;
            in_p[j] = b >= d.low && b <= d.high;
        }
        uint64_t k_weight = d.k_weight;
        if (d.k_bucket < kBuckets) {
            uint64_t all;
            uint64_t rank = block_before<kWaves>((in_k[0] ? 1 : 0) + (in_k[1] ? 1 : 0), s_part, all);
            uint64_t mine = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (in_k[j]) {
                    const uint64_t place = static_cast<uint64_t>(d.k_count) + rank;
                    mine += place < static_cast<uint64_t>(r.k) ? weight[j] : 0;
                    if (place + 1 == static_cast<uint64_t>(r.k)) {
                        s_last = word[j];
                    }
                    ++rank;
                }
            }
            (void)block_before<kWaves>(mine, s_part, all);
            k_weight += all;
        }
        __syncthreads();
        last = s_last;
        if (r.p < 1.0) {
            const double target = r.p * static_cast<double>(k_weight);
            uint64_t all;
            uint64_t before = d.low_weight + block_before<kWaves>((in_p[0] ? weight[0] : 0) + (in_p[1] ? weight[1] : 0),
                                                                  s_part, all);
            // the last token with less than the target before it
            uint64_t mine = ~uint64_t{0};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (in_p[j]) {
                    mine = static_cast<double>(before) < target ? word[j] : mine;
                    before += weight[j];
                }
            }
            // order words fall along the list: the smallest is the last
            const uint64_t p_last = ~block_max<kWaves>(~mine, s_part);
            last = max_u64(last, p_last);
        }
    } else if (n > kList) {
        uint64_t k_weight = d.k_weight;
        if (d.k_bucket < kBuckets) {
            last = select_in_row<T>(a, r, logits, d.k_bucket, d.k_bucket, static_cast<uint64_t>(d.k_count), r.k, 0.0,
                                    s_bins, s_part);
            uint64_t mine = 0;
            for (int64_t id = tid * 8; id < a.vocab; id += kFinish * 8) {
                float x[8];
                load8<T>(x, logits, id, a.vocab);
                for (int i = 0; i < 8; ++i) {
                    const double depth = depth_of(r, x[i]);
                    if (depth < kDepth && bucket_of(depth) == d.k_bucket && order_word(x[i], id + i) >= last) {
                        mine += weight_of(depth);
                    }
                }
            }
            uint64_t all;
            (void)block_before<kWaves>(mine, s_part, all);
            k_weight += all;
        }
        if (r.p < 1.0) {
            last = max_u64(last, select_in_row<T>(a, r, logits, d.low, d.high, d.low_weight, 0,
                                                  r.p * static_cast<double>(k_weight), s_bins, s_part));
        }
    }
    // the first token stays, whatever the settings
    last = last < best ? last : best;
    __syncthreads();
    if (n > 0 && n <= kList) {
        for (int i = tid; i < n; i += kFinish) {
            const uint64_t word = s_list[i];
            const double depth = depth_of(r, order_logit(word));
            const uint64_t w = weight_of(depth);
            if (word >= last && w >= r.least) {
                atomicAdd(&s_sums[order_id(word) / kChunk], static_cast<unsigned long long>(w));
            }
        }
    } else if (n > kList) {
        for (int64_t id = tid * 8; id < a.vocab; id += kFinish * 8) {
            float x[8];
            load8<T>(x, logits, id, a.vocab);
            uint64_t sum = 0;
            for (int i = 0; i < 8; ++i) {
                const double depth = depth_of(r, x[i]);
                if (depth < kDepth && bucket_of(depth) >= d.low && order_word(x[i], id + i) >= last) {
                    const uint64_t w = weight_of(depth);
                    sum += w >= r.least ? w : 0;
                }
            }
            atomicAdd(&s_sums[id / kChunk], static_cast<unsigned long long>(sum));
        }
    }
    __syncthreads();
    // the chunk that u falls on
    static_assert(kMaxChunks <= kFinish, "one chunk a thread");
    const uint64_t mine = tid < chunks ? s_sums[tid] : 0;
    uint64_t total;
    const uint64_t before = block_before<kWaves>(mine, s_part, total);
    const double u = static_cast<double>(a.random[row]);
    uint64_t target = u > 0.0 ? static_cast<uint64_t>((u < 1.0 ? u : 1.0) * static_cast<double>(total)) : 0;
    target = target < total ? target : total - 1;
    if (before <= target && target < before + mine) {
        s_chunk = tid;
        s_rest = target - before;
    }
    __syncthreads();
    const int64_t id0 = static_cast<int64_t>(s_chunk) * kChunk;
    const uint64_t rest = s_rest;
    uint64_t w[2] = {0, 0};
    if (tid < kChunk / 8) {
        float x[8];
        load8<T>(x, logits, id0 + tid * 8, a.vocab);
        uint64_t* const out = s_list;  // [kChunk] weights
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double depth = depth_of(r, x[i]);
            uint64_t v = 0;
            if (depth < kDepth && id0 + tid * 8 + i < a.vocab) {
                v = weight_of(depth);
                v = v >= r.least && order_word(x[i], id0 + tid * 8 + i) >= last ? v : 0;
            }
            out[tid * 8 + i] = v;
        }
    }
    __syncthreads();
    static_assert(kChunk == 2 * kFinish && kChunk <= kList, "two ids of the chunk a thread");
    w[0] = s_list[2 * tid];
    w[1] = s_list[2 * tid + 1];
    uint64_t all;
    const uint64_t at = block_before<kWaves>(w[0] + w[1], s_part, all);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint64_t from = j == 0 ? at : at + w[0];
        if (from <= rest && rest < from + w[j]) {
            a.tokens[row] = static_cast<int32_t>(id0 + 2 * tid + j);
            if (a.chances != nullptr) {
                a.chances[row] = static_cast<float>(static_cast<double>(w[j]) / static_cast<double>(total));
            }
        }
    }
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t stream) {
    const int chunks = static_cast<int>((a.vocab + kChunk - 1) / kChunk);
    // about eight blocks a CU; with few rows a chunk a block
    const int64_t per = (chunks * a.rows + 2047) / 2048;
    const int blocks = static_cast<int>((chunks + per - 1) / per);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.rows));
    hipLaunchKernelGGL(sample_max_kernel<T>, grid, dim3(kThreads), 0, stream, a, chunks, static_cast<int>(per));
    hipError_t status = hipGetLastError();
    if (status == hipSuccess && (a.top_k != nullptr || a.top_p != nullptr)) {
        hipLaunchKernelGGL(sample_buckets_kernel<T>, grid, dim3(kThreads), 0, stream, a, chunks, static_cast<int>(per));
        status = hipGetLastError();
    }
    if (status == hipSuccess) {
        hipLaunchKernelGGL(sample_sums_kernel<T>, grid, dim3(kThreads), 0, stream, a, chunks, static_cast<int>(per));
        status = hipGetLastError();
    }
    if (status == hipSuccess) {
        hipLaunchKernelGGL(sample_finish_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(kFinish), 0, stream, a, chunks,
                           blocks);
        status = hipGetLastError();
    }
    return status;
}

}  // namespace

int64_t sample_workspace_bytes(int64_t rows, int64_t vocab) { return rows * row_bytes((vocab + kChunk - 1) / kChunk); }

hipError_t launch_sample(int dtype, const SampleArgs& a, hipStream_t stream) {
    if (dtype == 0) {
        return launch<F32>(a, stream);
    }
    return dtype == 1 ? launch<Bf16>(a, stream) : launch<F16>(a, stream);
}

}  // namespace kc
