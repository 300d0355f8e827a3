// Attention of a ragged batch of new tokens over a paged KV cache.
//
// Sequence i brings q_len new tokens (rows query_starts[i] .. query_starts[i + 1]
// of the queries) and has kv_len cached rows, its new tokens' among them; token t
// of it stands at position kv_len - q_len + t and sees the keys up to there:
//     out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - max)
// in one pass over the keys with a running maximum and sum (fp32).  A row that
// sees no key is zero.
//
// The query heads of a KV head share its keys, so the rows of one (sequence, KV
// head) are its tokens times those heads, row r = token r / G, head r % G, and a
// block takes a tile of them as the columns of S^T = K Q^T and O^T = V^T P^T.  In
// that orientation a lane's scores belong to one column, and they lie in the
// order in which the second product takes its weights if V's keys are read in
// the same order: the weights never leave their lane.  V's rows go to LDS as they
// are and are read transposed (ds_read_b64_tr_b16: a group of 16 lanes reads 4
// keys x 16 dims and each lane receives the 4 keys of one dim).
#include <type_traits>

#include "kc_device.h"
#include "kc_kernels.h"

namespace kc {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kThreads = 256;

// ------------------------------------------------------------ element types
__device__ __forceinline__ floatx4 mfma16(Bf16, uint4 a, uint4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma16(F16, uint4 a, uint4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma32(Bf16, uint4 a, uint4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma32(F16, uint4 a, uint4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
// Two fp32 values rounded to nearest, the first in the low half; and back.
__device__ __forceinline__ uint32_t pack(Bf16, float lo, float hi) { return pack2(lo, hi); }
__device__ __forceinline__ uint32_t pack(F16, float lo, float hi) {
    typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
    const halfx2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
}
// sum + both halves of v, in fp32.
__device__ __forceinline__ float add_pair(Bf16, uint32_t v, float sum) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
}
__device__ __forceinline__ float add_pair(F16, uint32_t v, float sum) {
    typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(halfx2, v), __builtin_bit_cast(halfx2, 0x3c003c00u), sum, false);
}
// Weights are 2^(score - maximum + kUp): in fp16 they use the type's upper range, up to
// 2^15, so that the many small ones of a long cache keep their bits (an fp16 number loses
// the first below 2^-14 and the last below 2^-25: 2^-36 of the largest weight).  The row
// tiles' maximum may lag by kLag powers of two.  The sums of weights and of values have
// the factor alike, it cancels in their quotient; partials tell the maximum less kUp.
template <typename T>
struct Weights {
    static constexpr float kUp = 0.0f;
    static constexpr float kLag = 8.0f;
    static constexpr float kFewUp = 0.0f;
};
template <>
struct Weights<F16> {
    static constexpr float kUp = 11.0f;
    static constexpr float kLag = 4.0f;
    static constexpr float kFewUp = 14.0f;
};
template <typename T>
__device__ __forceinline__ float low(uint32_t v) {
    return T::load(static_cast<uint16_t>(v & 0xffffu));
}
template <typename T>
__device__ __forceinline__ float high(uint32_t v) {
    return T::load(static_cast<uint16_t>(v >> 16));
}

// Transposed read of 4 keys x 16 dims by 16 lanes (each lane: 8 bytes of a row).
__device__ __forceinline__ uint2 read_transposed(const uint8_t* p) {
    const auto lds = (__attribute__((address_space(3))) shortx4*)(__attribute__((address_space(3))) const uint8_t*)p;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds));
}

// ------------------------------------------------------------- the sequence
// What a block needs of its sequence.  Lengths come from device memory; whatever
// they hold, rows stay inside [0, tokens) and keys inside the sequence's table
// row.  A kv_len that does not fit the table row gives NaN rows.
struct Sequence {
    int first;     // row of the first new token
    int q_len;
    int kv_len;
    bool bad;
};
__device__ __forceinline__ Sequence sequence(const PagedAttnArgs& a, int index) {
    Sequence s;
    const int tokens = static_cast<int>(a.tokens);
    const int begin = a.starts[index];
    const int end = a.starts[index + 1];
    s.first = begin < 0 ? 0 : (begin < tokens ? begin : tokens);
    const int last = end < tokens ? end : tokens;
    s.q_len = last > s.first ? last - s.first : 0;
    const int kv = a.kv_lens[index];
    s.bad = kv < 0 || kv > (a.table_stride << a.page_shift);
    s.kv_len = s.bad ? 0 : kv;
    return s;
}

// The same where the index is one for the whole wave.
__device__ __forceinline__ Sequence wave_sequence(const PagedAttnArgs& a, int index) {
    Sequence s = sequence(a, index);
    s.first = __builtin_amdgcn_readfirstlane(s.first);
    s.q_len = __builtin_amdgcn_readfirstlane(s.q_len);
    s.kv_len = __builtin_amdgcn_readfirstlane(s.kv_len);
    s.bad = __builtin_amdgcn_readfirstlane(s.bad) != 0;
    return s;
}

// Key j of a sequence: element offset of its row in the pools, and whether its
// page exists (a page id outside the pool is read as page 0 and reported).
__device__ __forceinline__ int64_t key_row(const PagedAttnArgs& a, int page, int key, bool& bad) {
    bad |= static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.num_pages);
    const int64_t id = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages) ? page : 0;
    return id * a.page_stride + static_cast<int64_t>(key & ((1 << a.page_shift) - 1)) * a.token_stride;
}

// The partials' parts: sums [row, head, split, dim], (max, sum) [row, head, split],
// and how many splits a row and head has [row, head].
__device__ __forceinline__ float* split_stats(const PagedAttnArgs& a, int D, int splits) {
    return a.partials + a.tokens * a.q_heads * splits * D;
}
__device__ __forceinline__ int32_t* split_counts(const PagedAttnArgs& a, int D, int splits) {
    return reinterpret_cast<int32_t*>(a.partials + a.tokens * a.q_heads * splits * (D + 2));
}

// ----------------------------------------------------------- careful columns
// Columns [c0, c0 + count) of a (sequence, KV head) over keys [begin, end) in
// plain fp32, 16 lanes a column: where a product met an infinity or NaN of a key
// that a column does not see (0 * inf), or a page id is outside the pool (the
// columns that see it become NaN).
template <typename T, int D>
__device__ __forceinline__ void careful_columns(const PagedAttnArgs& a, const Sequence& s, const int32_t* table, int g,
                                                int c0, int count, int begin, int end, int split, int splits) {
    constexpr int kDims = D / 16;
    const int G = static_cast<int>(a.group);
    const int d0 = static_cast<int>(threadIdx.x) % 16 * kDims;
    for (int c = c0 + static_cast<int>(threadIdx.x) / 16; c < c0 + count; c += static_cast<int>(blockDim.x) / 16) {
        const int token = c / G;
        const int head = g * G + c % G;
        const int pos = s.kv_len - s.q_len + token;
        const int stop = end < pos + 1 ? end : pos + 1;
        const int64_t row = s.first + token;
        const uint16_t* qp = a.q + row * a.q_stride + head * D + d0;
        float acc[kDims] = {};
        float m = kNegInf;
        float l = 0.0f;
        for (int key = begin; key < stop; ++key) {
            bool bad = false;
            const int64_t at = key_row(a, table[key >> a.page_shift], key, bad) + g * a.head_stride + d0;
            float dot = 0.0f;
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                dot = fmaf(T::load(qp[d]), T::load(a.k[at + d]), dot);
            }
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) {
                dot += __shfl_xor(dot, o, 16);
            }
            const float sc = bad ? __builtin_nanf("") : dot * a.scale_log2;
            const float m_new = fmaxf(m, sc);
            const float m_sub = m_new == kNegInf ? 0.0f : m_new;
            const float corr = __builtin_amdgcn_exp2f(m - m_sub);
            const float p = __builtin_amdgcn_exp2f(sc - m_sub);
            l = l * corr + p;
            m = m_new;
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                // (a weight of zero takes nothing from an infinite value)
                acc[d] = acc[d] * corr + (p == 0.0f ? 0.0f : p * T::load(a.v[at + d]));
            }
        }
        if (splits == 1) {
            uint16_t* out = a.out + row * a.out_stride + head * D + d0;
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                out[d] = T::store(l == 0.0f ? 0.0f : acc[d] / l);
            }
        } else {
            const int64_t at = (row * a.q_heads + head) * splits + split;
            float* part = a.partials + at * D + d0;
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                part[d] = acc[d];
            }
            if (d0 == 0) {
                float* ml = split_stats(a, D, splits) + 2 * at;
                ml[0] = m;
                ml[1] = l;
            }
        }
    }
}

// Rows of a sequence whose kv_len does not fit its table.
template <typename T, int D>
__device__ __forceinline__ void nan_columns(const PagedAttnArgs& a, const Sequence& s, int g, int c0, int count,
                                            int splits) {
    const int G = static_cast<int>(a.group);
    for (int i = threadIdx.x; i < count * D; i += blockDim.x) {
        const int c = c0 + i / D;
        const int64_t row = s.first + c / G;
        const int head = g * G + c % G;
        if (splits == 1) {
            a.out[row * a.out_stride + head * D + i % D] = T::store(__builtin_nanf(""));
        } else if (i % D == 0) {
            const int64_t unit = row * a.q_heads + head;
            *reinterpret_cast<float2*>(split_stats(a, D, splits) + 2 * unit * splits) = make_float2(0.0f, __builtin_nanf(""));
            split_counts(a, D, splits)[unit] = 1;
        }
    }
}

// One column's merged result: 8 consecutive dims from d0.
template <typename T, int D>
__device__ __forceinline__ void put_column(const PagedAttnArgs& a, int64_t row, int head, int d0, const float (&v)[8],
                                           float m, float l, int split, int splits) {
    if (splits == 1) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = l == 0.0f ? 0u : pack(T{}, v[2 * i] / l, v[2 * i + 1] / l);
        }
        *reinterpret_cast<uint4*>(a.out + row * a.out_stride + head * D + d0) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
    const int64_t at = (row * a.q_heads + head) * splits + split;
    float* part = a.partials + at * D + d0;
    *reinterpret_cast<float4*>(part) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(part + 4) = make_float4(v[4], v[5], v[6], v[7]);
    if (d0 == 0) {
        *reinterpret_cast<float2*>(split_stats(a, D, splits) + 2 * at) = make_float2(m, l);
    }
}

// How many splits columns [c0, c0 + count) have: told once, by the block with the last.
template <int D>
__device__ __forceinline__ void tell_splits(const PagedAttnArgs& a, const Sequence& s, int g, int c0, int count, int made,
                                            int splits) {
    const int G = static_cast<int>(a.group);
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const int c = c0 + i;
        split_counts(a, D, splits)[(s.first + c / G) * a.q_heads + g * G + c % G] = made;
    }
}

// ------------------------------------------------------------------ few rows
// Sequences of which a KV head has at most kFewRows rows, many and long ones (the plan
// says which): single tokens, bound by the cache's bytes.  All blocks share the cached
// rows of all sequences evenly: the work is the line of (sequence, KV head, tile of 16
// rows, round of 128 keys), cut into one stretch a block, so a batch of unequal lengths
// ends everywhere at once (64 sequences of up to 8192 tokens, 307 MB: 70 us, 4.4 TB/s;
// with a fixed number of splits a sequence 88).  A stretch is whole rounds: 9.25 of them
// a block, as there, are 10 for 474 blocks and none for 38.  In a round the four waves
// take 32 keys each, K straight from memory into the first product's operand, V through
// the wave's own LDS, the next keys requested as soon as the registers of these are free.
// With more rows the keys would be read once a tile of 16, and the row tiles below are
// faster: 32 rows of 64 sequences of 2000 keys 58 us here and 38 there, of up to 8192
// keys 104 and 82, of one with 120000 55 and 35; of 64 with 100 keys 9.9 and 12.
constexpr int kFewRows = 16;
constexpr int kUnit = 32;
constexpr int kRound = 4 * kUnit;
constexpr int64_t kFewBlocks = 512;

// A sequence's part of the line: tiles of 16 rows, rounds of each.  Without splits a
// tile is one piece of work.
struct Line {
    int tiles;
    int rounds;
};
__device__ __forceinline__ Line line_of(const PagedAttnArgs& a, const Sequence& s, int few_rows, int splits) {
    const int64_t rows = static_cast<int64_t>(s.q_len) * a.group;
    Line line;
    line.tiles = rows <= few_rows ? static_cast<int>((rows + 15) / 16) : 0;
    const int rounds = (s.kv_len + kRound - 1) / kRound;
    line.rounds = splits > 1 && rounds > 1 ? rounds : 1;
    return line;
}
__device__ __forceinline__ int length_of(const PagedAttnArgs& a, const Line& line) {
    return static_cast<int>(a.kv_heads) * line.tiles * line.rounds;
}

template <typename T, int D>
__device__ __forceinline__ void few_rows_tile(const PagedAttnArgs& a, const Sequence& s, int index, int g, int c0,
                                              int begin, int end, int split, int splits, uint8_t* s_mem,
                                              float (*s_ml)[16][2], int* s_redo) {
    constexpr int kSteps = D / 32;   // products of 32 dims a score
    constexpr int kPieces = D / 8;   // 16-byte pieces of a row
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;
    const int q = lane >> 4;
    const int G = static_cast<int>(a.group);
    const int rows = s.q_len * G;
    const int32_t* const table = a.table + static_cast<int64_t>(index) * a.table_stride;
    const uint16_t* const kbase = a.k + g * a.head_stride;
    const uint16_t* const vbase = a.v + g * a.head_stride;
    uint8_t* const s_v = s_mem + wave * (kUnit * D * 2);

    const int count = rows - c0 < 16 ? rows - c0 : 16;
    const int column = c0 + (r < count ? r : count - 1);
    const int pos = s.kv_len - s.q_len + column / G;  // the last key that the column sees
    const int head = g * G + column % G;
    const int ends = s.kv_len - s.q_len + (c0 + count - 1) / G + 1;
    const int keys = ends > 0 ? ends : 0;
    const int units = (keys + kUnit - 1) / kUnit;
    const int u_end = end * 4 < units ? end * 4 : units;
    int unit = begin * 4 + wave;

    uint4 qf[kSteps];
    {
        const uint16_t* const src = a.q + static_cast<int64_t>(s.first + column / G) * a.q_stride + head * D + 8 * q;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            qf[i] = *reinterpret_cast<const uint4*>(src + 32 * i);
        }
    }
    bool bad = false;
    int64_t at[2];
    int page[2];
    const auto pages = [&](int u) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = u * kUnit + 16 * t + r;
            page[t] = table[(key < keys ? key : keys - 1) >> a.page_shift];
        }
    };
    const auto place = [&](int u) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = u * kUnit + 16 * t + r;
            at[t] = key_row(a, page[t], key < keys ? key : keys - 1, bad) + 8 * q;
        }
    };
    uint4 kf[2][kSteps], vf[2][kSteps];
    const auto fetch = [&](uint4 (&f)[2][kSteps], const uint16_t* base) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                f[t][i] = load_stream(reinterpret_cast<const uint4*>(base + at[t] + 32 * i));
            }
        }
    };
    floatx4 acc[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        acc[i] = floatx4{};
    }
    float m_run = kNegInf;
    float l_run = 0.0f;
    if (unit < u_end) {
        pages(unit);
        place(unit);
        fetch(kf, kbase);
        fetch(vf, vbase);
        pages(unit + 4);
    }
    for (; unit < u_end; unit += 4) {
        // V's rows, their 16-byte pieces swizzled so that the 8 rows of a
        // transposed half-wave read lie in different banks
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int row = 16 * t + r;
                const int piece = (4 * i + q) ^ (((row & 7) << 1) % kPieces);
                *reinterpret_cast<uint4*>(s_v + row * (D * 2) + piece * 16) = vf[t][i];
            }
        }
        const bool more = unit + 4 < u_end;
        if (more) {
            place(unit + 4);
            fetch(vf, vbase);
            pages(unit + 8);
        }
        floatx4 sc[2] = {floatx4{}, floatx4{}};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            sc[0] = mfma16(T{}, kf[0][i], qf[i], sc[0]);
            sc[1] = mfma16(T{}, kf[1][i], qf[i], sc[1]);
        }
        if (more) {
            fetch(kf, kbase);
        }
        // sc[t][i]: key 16 t + 4 q + i of the unit
        const int rel = pos - unit * kUnit - 4 * q;
        float mx = kNegInf;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[t][i] = 16 * t + i <= rel ? sc[t][i] * a.scale_log2 : kNegInf;
                mx = fmaxf(mx, sc[t][i]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run, mx);
        const float m_sub = m_new == kNegInf ? 0.0f : m_new;
        const float corr = __builtin_amdgcn_exp2f(m_run - m_sub);
        m_run = m_new;
        l_run *= corr;
        // weights as two 16-bit parts (16 bits of the fp32 weight in bf16; in fp16 22,
        // one fewer for each power of two below 2^-17 of the largest, none below 2^-39:
        // 2^20 such keys would be 2^-19 of it, in l_run alone): this form waits for
        // memory, the second product is free
        const float m_w = m_sub - Weights<T>::kFewUp;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(sc[e / 2][2 * (e % 2)] - m_w);
            const float p1 = __builtin_amdgcn_exp2f(sc[e / 2][2 * (e % 2) + 1] - m_w);
            l_run += p0 + p1;
            hi[e] = pack(T{}, p0, p1);
            lo[e] = pack(T{}, p0 - low<T>(hi[e]), p1 - high<T>(hi[e]));
        }
        const uint4 ph = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        const uint4 pl = make_uint4(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            uint2 part[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int row = 16 * t + 4 * q + r / 4;
                const int piece = (2 * i + (r & 3) / 2) ^ (((row & 7) << 1) % kPieces);
                part[t] = read_transposed(s_v + row * (D * 2) + piece * 16 + (r & 1) * 8);
            }
            const uint4 vt = make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[i][e] *= corr;
            }
            acc[i] = mfma16(T{}, vt, ph, acc[i]);
            acc[i] = mfma16(T{}, vt, pl, acc[i]);
        }
    }
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    // the waves' columns meet in LDS, each in the wave's own part: [column][dim]
    __syncthreads();
    if (tid == 0) {
        *s_redo = 0;
    }
    float* const s_acc = reinterpret_cast<float*>(s_mem);  // [wave][16][D / 2]: half of the dims a round
    if (q == 0) {
        s_ml[wave][r][0] = m_run - Weights<T>::kFewUp;
        s_ml[wave][r][1] = l_run;
    }
    bool redo = bad;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
        // a padded, rotated row: the 16 columns of a store start in different banks
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int dim = 16 * i + 4 * q;
            *reinterpret_cast<float4*>(s_acc + (wave * 16 + r) * (D / 2) + (dim ^ ((r & 7) * 4))) =
                make_float4(acc[half * (D / 32) + i][0], acc[half * (D / 32) + i][1], acc[half * (D / 32) + i][2],
                            acc[half * (D / 32) + i][3]);
        }
        __syncthreads();
        constexpr int kChunks = D / 16;  // 8 dims of a half row
        if (tid < 16 * kChunks) {
            const int c = tid / kChunks;
            const int d = tid % kChunks * 8;
            float m = s_ml[0][c][0];
#pragma unroll
            for (int w = 1; w < 4; ++w) {
                m = fmaxf(m, s_ml[w][c][0]);
            }
            const float m_sub = m == kNegInf ? 0.0f : m;
            float l = 0.0f;
            float v[8] = {};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(s_ml[w][c][0] - m_sub);
                l = fmaf(s_ml[w][c][1], f, l);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float4 p = *reinterpret_cast<const float4*>(s_acc + (w * 16 + c) * (D / 2) +
                                                                     ((d + 4 * j) ^ ((c & 7) * 4)));
                    v[4 * j] = fmaf(p.x, f, v[4 * j]);
                    v[4 * j + 1] = fmaf(p.y, f, v[4 * j + 1]);
                    v[4 * j + 2] = fmaf(p.z, f, v[4 * j + 2]);
                    v[4 * j + 3] = fmaf(p.w, f, v[4 * j + 3]);
                }
            }
            float zero = l * 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                zero = fmaf(v[j], 0.0f, zero);
            }
            redo |= zero != zero;
            if (c < count) {
                const int col = c0 + c;
                put_column<T, D>(a, s.first + col / G, g * G + col % G, half * (D / 2) + d, v, m, l, split, splits);
            }
        }
    }
    if (redo) {
        *s_redo = 1;
    }
    __syncthreads();
    if (*s_redo != 0) {
        careful_columns<T, D>(a, s, table, g, c0, count, begin * kRound, u_end * kUnit, split, splits);
    }
    __syncthreads();
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void paged_attention_few_kernel(PagedAttnArgs a, int splits, int few_rows) {
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[4 * kUnit * D * 2];
    __shared__ float s_ml[4][16][2];
    __shared__ int s_part[4], s_most[4];
    __shared__ int s_found[6];
    __shared__ int s_redo;
    const int tid = threadIdx.x;
    const int sequences = static_cast<int>(a.sequences);
    // (the line's length fits in 31 bits: the plan splits nothing where it might not)
    // a thread's run of sequences (one of up to 256): the run's part of the line, where
    // it begins, and its first sequence
    const int per_thread = (sequences + kThreads - 1) / kThreads;
    int mine = 0;
    int mine_before = 0;
    Sequence own = {};
    int total, most;
    if (sequences == 1) {
        const Line line = line_of(a, wave_sequence(a, 0), few_rows, splits);
        total = length_of(a, line);
        most = line.rounds;
    } else {
        const int run_end = (tid + 1) * per_thread < sequences ? (tid + 1) * per_thread : sequences;
        int longest = 1;
        bool descending = false;  // (such starts name no rows: their lengths need not fit the line)
        for (int i = tid * per_thread; i < run_end; ++i) {
            own = sequence(a, i);
            descending |= a.starts[i + 1] < a.starts[i];
            const Line line = line_of(a, own, few_rows, splits);
            mine += length_of(a, line);
            longest = line.tiles > 0 && line.rounds > longest ? line.rounds : longest;
        }
        longest = descending ? 0x7fffffff : longest;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int left = __shfl_up(sum, o, 64);
            const int other = __shfl_xor(longest, o, 64);
            sum += (tid & 63) >= o ? left : 0;
            longest = other > longest ? other : longest;
        }
        if ((tid & 63) == 63) {
            s_part[tid >> 6] = sum;
            s_most[tid >> 6] = longest;
        }
        __syncthreads();
        total = __builtin_amdgcn_readfirstlane(s_part[0] + s_part[1] + s_part[2] + s_part[3]);
        most = __builtin_amdgcn_readfirstlane(max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3])));
        if (most == 0x7fffffff) {
            return;
        }
        mine_before = sum - mine;
        for (int w = 0; w < (tid >> 6); ++w) {
            mine_before += s_part[w];
        }
    }
    // a stretch: an even share, and long enough that no tile lies in more than `splits`
    const int blocks = static_cast<int>(gridDim.x);
    int stretch = (total + blocks - 1) / blocks;
    const int least = splits > 1 ? (most + splits - 2) / (splits - 1) : 1;
    stretch = stretch > least ? stretch : least;
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * stretch;
    if (begin >= total) {
        return;
    }
    int at = static_cast<int>(begin);
    const int stop = at + stretch < total ? at + stretch : total;
    int index, before;
    Sequence s;
    if (sequences == 1) {
        index = 0;
        before = 0;
        s = wave_sequence(a, 0);
    } else {
        // the thread whose sequences the stretch begins in tells which
        if (mine_before <= at && at < mine_before + mine) {
            int i = tid * per_thread;
            for (; per_thread > 1; ++i) {
                own = sequence(a, i);
                const int next = mine_before + length_of(a, line_of(a, own, few_rows, splits));
                if (at < next) {
                    break;
                }
                mine_before = next;
            }
            s_found[0] = i;
            s_found[1] = mine_before;
            s_found[2] = own.first;
            s_found[3] = own.q_len;
            s_found[4] = own.kv_len;
            s_found[5] = own.bad;
        }
        __syncthreads();
        index = __builtin_amdgcn_readfirstlane(s_found[0]);
        before = __builtin_amdgcn_readfirstlane(s_found[1]);
        s.first = __builtin_amdgcn_readfirstlane(s_found[2]);
        s.q_len = __builtin_amdgcn_readfirstlane(s_found[3]);
        s.kv_len = __builtin_amdgcn_readfirstlane(s_found[4]);
        s.bad = __builtin_amdgcn_readfirstlane(s_found[5]) != 0;
    }
    for (;;) {
        const Line line = line_of(a, s, few_rows, splits);
        const int next = before + length_of(a, line);
        while (at < stop && at < next) {
            const int piece = (at - before) / line.rounds;
            const int first = before + piece * line.rounds;
            const int to = stop - first < line.rounds ? stop - first : line.rounds;
            const int g = piece / line.tiles;
            const int c0 = piece % line.tiles * 16;
            const int rest = s.q_len * static_cast<int>(a.group) - c0;
            const int count = rest < 16 ? rest : 16;
            const int split = splits > 1 ? static_cast<int>(blockIdx.x) - first / stretch : 0;
            if (s.bad) {
                nan_columns<T, D>(a, s, g, c0, count, splits);
            } else {
                if (to == line.rounds && splits > 1) {
                    tell_splits<D>(a, s, g, c0, count, split + 1, splits);
                }
                few_rows_tile<T, D>(a, s, index, g, c0, at - first, splits > 1 ? to : 0x7fffffff / kRound, split, splits,
                                    s_mem, s_ml, &s_redo);
            }
            at = first + to;
        }
        if (at >= stop) {
            return;
        }
        before = next;
        s = wave_sequence(a, ++index);
    }
}

// ----------------------------------------------------------------- row tiles
// 128 columns of a (sequence, KV head): four waves of 32 over the same 64 keys,
// whose K and V rows go straight to LDS, one window ahead.  Two waves a SIMD hide
// each other's waits and arithmetic: from two such blocks on a CU, or, where there
// are fewer tiles, from one block of two K-groups, which take alternate windows and
// meet in LDS at the end.
//
// A wave takes 32 products of 32 cycles a window (D = 128) and about as long in fp32
// arithmetic (exp of 32 scores a lane).  Weights enter the second product rounded to
// 16 bits and their sum adds the rounded ones: half a step of the type a weight, at
// random, next to the result's own half step (2-norm error of a prompt of 8192 bf16
// tokens 2.1e-3, 1.9e-3 with a maximum that never lags at 284 us for 265, of the
// result's rounding alone 1.6e-3).  A second part of each weight costs half as many
// products again and its forming: that prompt 354 us for 266, six mixed fp16 chunks with
// heads of 64 63 for 49.  Measured, 8192 tokens of 16 heads over 2 KV heads:
// 346 us at first, 318 with loads that bypass the compiler's waits, 293 with operands
// read ahead and the maximum allowed to lag, 287 with page bases as scalars, 262 with the
// waves' priorities and the order of blocks, 266 with the second loop that follows here
// in one kernel (1035 TFLOP/s; a library product of 8192^3 1405).  Forming the next
// window's scores between this window's weights (250 VGPRs) took 293.
//
// Sequences of at most kFineRows rows a KV head (single tokens, drafts) are one wave's
// columns: their products have room, and their weights keep both 16-bit parts, as in the
// kernel for few rows (16 bits of the fp32 weight in bf16, up to 22 in fp16); their sum
// adds them as they are.  What that costs is forming the second parts, fp32 arithmetic of one
// wave: a token over 2000 keys 14.2 us (one part: 14.0), over 120000 33.4 (32.7), 16
// over up to 4000 20.5 (18.1), two chunks of 256 beside 8 tokens 30.4 (30.1; with the
// waves of both K-groups on one SIMD 35).
constexpr int kTileRows = 128;
constexpr int kFineRows = 32;
constexpr int kWindow = 64;

// 16 bytes a lane from base + offset straight into LDS, lane after lane from `lds`.
// (As an instruction of its own: behind the builtin the compiler waits for the load
// before the next LDS read, whatever that reads.  It writes no register; the wait is
// the window's own.  Nothing else in these kernels keeps a value in m0.)
__device__ __forceinline__ void load_lds16(const uint8_t* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void load_lds16(const uint16_t* src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
}
__device__ __forceinline__ float halves_max(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Tile slots: sequence i owns slots from floor(starts[i] G / 128) + i on, at least
// as many as it has tiles, so the grid follows from the token count alone.
template <typename T, int D, int GROUPS>
__global__ __launch_bounds__(kThreads * GROUPS, D == 64 && GROUPS == 2 ? 4 : 2) void paged_attention_tile_kernel(PagedAttnArgs a, int slots,
                                                                                    int tile_splits, int splits,
                                                                                    int few_rows) {
    constexpr int kSteps = D / 16;
    constexpr int kRowBytes = D * 2;
    constexpr int kPieces = D / 8;
    constexpr int kTileBytes = kWindow * kRowBytes;
    constexpr int kLoadRows = 1024 / kRowBytes;      // rows of a wave's load
    constexpr int kLoads = kWindow / (4 * kLoadRows);  // loads of a wave for a tile of K (and of V)
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[GROUPS][2][2 * kTileBytes];
    __shared__ float s_stats[GROUPS > 1 ? kTileRows : 1][2];
    __shared__ int s_index;
    __shared__ int s_redo;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
    const int group = __builtin_amdgcn_readfirstlane(tid >> 8);  // the K-group
    const int r = lane & 31;
    const int q = lane >> 5;
    const int G = static_cast<int>(a.group);
    const int kv_heads = static_cast<int>(a.kv_heads);
    // Later tiles see more keys: they start first, and of the first two blocks of a CU
    // the second is the lighter the heavier the first is.
    int order = static_cast<int>(blockIdx.x);
    if (GROUPS == 1) {
        const int total = static_cast<int>(gridDim.x);
        const int end = total < 512 ? total : 512;
        order = order >= 256 && order < end ? 255 + end - order : order;
    }
    const int g = order % kv_heads;
    const int split = order / kv_heads % tile_splits;
    const int slot = slots - 1 - order / kv_heads / tile_splits;
    if (tid == 0) {
        s_index = 0;
        s_redo = 0;
    }
    __syncthreads();
    for (int i = tid; i < static_cast<int>(a.sequences); i += kThreads * GROUPS) {
        const int64_t base = static_cast<int64_t>(a.starts[i]) * G / kTileRows + i;
        if (base <= slot) {
            atomicMax(&s_index, i);
        }
    }
    __syncthreads();
    const int index = __builtin_amdgcn_readfirstlane(s_index);
    const Sequence s = wave_sequence(a, index);
    const int64_t total = static_cast<int64_t>(s.q_len) * G;
    const int64_t tile = slot - (static_cast<int64_t>(s.first) * G / kTileRows + index);
    const int64_t c0 = tile * kTileRows;
    if (tile < 0 || c0 >= total || total <= few_rows) {
        return;
    }
    const int count = static_cast<int>(total - c0 < kTileRows ? total - c0 : kTileRows);
    if (s.bad) {
        if (split == 0) {
            nan_columns<T, D>(a, s, g, static_cast<int>(c0), count, splits);
        }
        return;
    }
    if (split == 0 && splits > 1) {
        tell_splits<D>(a, s, g, static_cast<int>(c0), count, tile_splits, splits);
    }
    const int32_t* const table = a.table + static_cast<int64_t>(index) * a.table_stride;
    const uint16_t* const kbase = a.k + g * a.head_stride;
    const uint16_t* const vbase = a.v + g * a.head_stride;
    const int before = s.kv_len - s.q_len;  // position of the first new token
    const int ends = before + (static_cast<int>(c0) + count - 1) / G + 1;
    const int keys = ends > 0 ? ends : 0;
    const int windows = (keys + kWindow - 1) / kWindow;
    const int per_split = (windows + tile_splits - 1) / tile_splits;
    const int w_begin = split * per_split;
    const int w_end = w_begin + per_split < windows ? w_begin + per_split : windows;

    // the K-groups' waves of the same columns on different SIMDs, for tiles of few columns
    const int strip = (wave + 2 * group) & 3;
    const int local = strip * 32 + r;
    const int column = static_cast<int>(c0) + (local < count ? local : count - 1);
    const int head = g * G + column % G;
    const int pos = before + column / G;
    const int wave_column = static_cast<int>(c0) + (strip * 32 < count ? strip * 32 : count - 1);
    const int first_pos = before + wave_column / G;  // lowest and highest positions of the wave's columns
    const int wave_last = strip * 32 + 31 < count ? strip * 32 + 31 : count - 1;
    const int last_pos = strip * 32 < count ? before + (static_cast<int>(c0) + wave_last) / G : -1;

    uint4 qf[kSteps];
    {
        const uint16_t* const src = a.q + static_cast<int64_t>(s.first + column / G) * a.q_stride + head * D + 8 * q;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            qf[i] = *reinterpret_cast<const uint4*>(src + 16 * i);
        }
    }
    bool bad = false;
    // K's pieces are swizzled by row against the 16 (D = 64: 8) rows that a read
    // takes together, V's so that the 4 rows of a transposed half-wave read lie
    // in different banks; the lane fetches the piece that belongs in its place
    const int lane_row = lane / kPieces;  // of a load's kLoadRows rows, which begin at a multiple of that
    const auto piece_of = [&](int row, bool value) __attribute__((always_inline)) {
        const int k = D == 128 ? row & 15 : (row >> 1) & 7;
        const int v = D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
        return (lane % kPieces) ^ (value ? v : k);
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(s_mem[group][0]) + wave * 1024);
    // Whole windows of pages that hold a load's rows together (and begin within 4 GB
    // of a pool's beginning times a page id): a load's base is the wave's, its lanes'
    // offsets are the same in every window.  Bytes from here on.
    const int page_mask = (1 << a.page_shift) - 1;
    const bool together = page_mask + 1 >= kLoadRows && a.token_stride < (1 << 26) && a.page_stride < (1 << 30);
    const uint32_t page_bytes = static_cast<uint32_t>(2 * a.page_stride);
    const uint32_t token_bytes = static_cast<uint32_t>(2 * a.token_stride);
    const uint8_t* k_at[kLoads];
    const uint8_t* v_at[kLoads];
    uint32_t k_lane[kLoads];
    uint32_t v_lane[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int row0 = (j * 4 + wave) * kLoadRows;
        const int64_t in_page = static_cast<int64_t>(row0 & page_mask) * token_bytes;
        k_at[j] = reinterpret_cast<const uint8_t*>(kbase) + in_page;
        v_at[j] = reinterpret_cast<const uint8_t*>(vbase) + in_page;
        k_lane[j] = lane_row * token_bytes + 16 * piece_of(row0 + lane_row, false);
        v_lane[j] = lane_row * token_bytes + 16 * piece_of(row0 + lane_row, true);
    }
    // pages of the window's groups of kLoadRows keys, one a lane
    int pages = 0;
    const auto look = [&](int w) __attribute__((always_inline)) {
        const int key = w * kWindow + lane % (4 * kLoads) * kLoadRows;
        pages = table[(key < keys ? key : keys - 1) >> a.page_shift];
    };
    const auto fetch = [&](int w, int buffer) __attribute__((always_inline)) {
        const uint32_t lds = lds0 + buffer * (2 * kTileBytes);
        if (together && (w + 1) * kWindow <= keys) {
            const bool out = static_cast<uint32_t>(pages) >= static_cast<uint32_t>(a.num_pages);
            bad |= out;
            const int page = out ? 0 : pages;
            // (pages of more than a window: where the window begins in its page)
            const int64_t shift = static_cast<int64_t>((w * kWindow) & page_mask) * token_bytes;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const uint32_t id = __builtin_amdgcn_readlane(page, j * 4 + wave);
                const int64_t at = static_cast<int64_t>(static_cast<uint64_t>(id) * page_bytes) + shift;
                load_lds16(k_at[j] + at, k_lane[j], lds + j * 4096);
                load_lds16(v_at[j] + at, v_lane[j], lds + kTileBytes + j * 4096);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int row = (j * 4 + wave) * kLoadRows + lane_row;
                const int key = w * kWindow + row < keys ? w * kWindow + row : keys - 1;
                const int64_t at = key_row(a, table[key >> a.page_shift], key, bad);
                load_lds16(kbase + at + 8 * piece_of(row, false), lds + j * 4096);
                load_lds16(vbase + at + 8 * piece_of(row, true), lds + kTileBytes + j * 4096);
            }
        }
    };
    floatx16 acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        acc[i] = floatx16{};
    }
    float m_run = kNegInf;
    float l_run = 0.0f;
    if (w_begin + group < w_end) {
        look(w_begin + group);
        fetch(w_begin + group, 0);
        look(w_begin + group + GROUPS);
    }
    const auto sweep = [&](auto parts) __attribute__((always_inline)) {
        constexpr bool kFine = decltype(parts)::value == 2;
        int buffer = 0;
        for (int w0 = w_begin; w0 < w_end; w0 += GROUPS, buffer ^= 1) {
            const int w = w0 + group;
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the window is in LDS
            __syncthreads();
            if (w + GROUPS < w_end) {
                fetch(w + GROUPS, buffer ^ 1);
                look(w + 2 * GROUPS);
            }
            const int key0 = w * kWindow;
            if (w >= w_end || key0 > last_pos) {
                continue;  // no window for this group, or no column of this wave sees it
            }
            const uint8_t* const s_k = s_mem[group][buffer];
            const uint8_t* const s_v = s_k + kTileBytes;
            const auto read_k = [&](uint4 (&k)[2], int i) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int row = 32 * t + r;
                    const int piece = (2 * i + q) ^ (D == 128 ? row & 15 : (row >> 1) & 7);
                    k[t] = *reinterpret_cast<const uint4*>(s_k + row * kRowBytes + piece * 16);
                }
            };
            const auto read_v = [&](uint4& v, int n, int i) __attribute__((always_inline)) {
                uint2 part[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    // 16 lanes: keys 16 n + 8 t + 4 q .. + 3, dims 32 i + 16 (lane / 16 % 2) .. + 15
                    const int row = 16 * n + 8 * t + 4 * q + (lane & 15) / 4;
                    const int piece = (4 * i + 2 * ((lane >> 4) & 1) + (lane & 3) / 2) ^
                                      (D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2);
                    part[t] = read_transposed(s_v + row * kRowBytes + piece * 16 + (lane & 1) * 8);
                }
                v = make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
            };
            // operands are read ahead of their products, held there by the scheduling
            // barriers; a wave that multiplies goes before one that does arithmetic
            floatx16 sc[2] = {floatx16{}, floatx16{}};
            constexpr int kAhead = D == 128 ? 2 : 1;
            uint4 kf[kAhead + 1][2], vf[D / 32];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                read_k(kf[i], i);
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (i + kAhead < kSteps) {
                    read_k(kf[(i + kAhead) % (kAhead + 1)], i + kAhead);
                }
                if (i + 2 >= kSteps) {
#pragma unroll
                    for (int d = 0; d < D / 64; ++d) {
                        read_v(vf[(i + 2 - kSteps) * (D / 64) + d], 0, (i + 2 - kSteps) * (D / 64) + d);
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    sc[t] = mfma32(T{}, kf[i % (kAhead + 1)][t], qf[i], sc[t]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            // sc[t][e]: key 32 t + 8 (e / 4) + 4 q + e % 4 of the window
            if (__builtin_amdgcn_readfirstlane(static_cast<int>(key0 + kWindow > first_pos + 1)) != 0) {
                const int rel = pos - key0 - 4 * q;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        sc[t][e] = 32 * t + 8 * (e / 4) + e % 4 <= rel ? sc[t][e] : kNegInf;
                    }
                }
            }
            float mx = kNegInf;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    mx = fmaxf(mx, sc[t][e]);
                }
            }
            // the maximum may lag behind (larger weights are as exact): sums are rescaled a
            // few times a row, not in every window
            const float m_new = fmaxf(m_run, halves_max(mx) * a.scale_log2);
            if (__any(m_new > m_run + Weights<T>::kLag)) {
                const float corr = __builtin_amdgcn_exp2f(m_run - (m_new == kNegInf ? 0.0f : m_new));
                l_run *= corr;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        acc[i][e] *= corr;
                    }
                }
                m_run = m_new;
            }
            const float m_sub = (m_run == kNegInf ? 0.0f : m_run) - Weights<T>::kUp;
            // steps of 16 keys: the lane's weights of scores 8 (n % 2) .. + 7 of half n / 2;
            // between the products of a step the next step's weights are formed and its V read
            uint32_t p[2][4], rest[2][kFine ? 4 : 1];
            const auto weights = [&](int n, int e) __attribute__((always_inline)) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[n / 2][8 * (n % 2) + 2 * e], a.scale_log2, -m_sub));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[n / 2][8 * (n % 2) + 2 * e + 1], a.scale_log2, -m_sub));
                p[n & 1][e] = pack(T{}, p0, p1);
                if constexpr (kFine) {
                    rest[n & 1][e] = pack(T{}, p0 - low<T>(p[n & 1][e]), p1 - high<T>(p[n & 1][e]));
                    l_run += p0 + p1;
                } else {
                    l_run = add_pair(T{}, p[n & 1][e], l_run);
                }
            };
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                weights(0, e);
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint4 pf = make_uint4(p[n & 1][0], p[n & 1][1], p[n & 1][2], p[n & 1][3]);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    acc[i] = mfma32(T{}, vf[i], pf, acc[i]);
                    if constexpr (kFine) {
                        const uint32_t(&x)[4] = rest[n & 1];
                        acc[i] = mfma32(T{}, vf[i], make_uint4(x[0], x[1], x[2], x[3]), acc[i]);
                    }
                    if (n < 3) {
#pragma unroll
                        for (int e = 0; e < 128 / D; ++e) {
                            weights(n + 1, i * (128 / D) + e);
                        }
                        read_v(vf[i], n + 1, i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        }
    };
    if (total > kFineRows) {
        sweep(std::integral_constant<int, 1>{});
    } else {
        sweep(std::integral_constant<int, 2>{});
    }
    l_run = halves_sum(l_run);
    {
        float zero = l_run * 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                zero = fmaf(acc[i][e], 0.0f, zero);
            }
        }
        if (bad || zero != zero) {
            s_redo = 1;
        }
    }
    __syncthreads();
    if (s_redo != 0) {
        careful_columns<T, D>(a, s, table, g, static_cast<int>(c0), count, w_begin * kWindow, w_end * kWindow, split,
                              splits);
        return;
    }
    if constexpr (GROUPS > 1) {
        // the second group's columns meet the first's: [wave][4 values][lane]
        float4* const s_acc = reinterpret_cast<float4*>(&s_mem[0][0][0]);
        if (group == 1) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s_acc[(strip * (D / 8) + i * 4 + j) * 64 + lane] =
                        make_float4(acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]);
                }
            }
            s_stats[local][0] = m_run;  // (both halves of the wave hold it)
            s_stats[local][1] = l_run;
        }
        __syncthreads();
        if (group == 1) {
            return;
        }
        const float m1 = s_stats[local][0];
        const float m_all = fmaxf(m_run, m1);
        const float m_sub = m_all == kNegInf ? 0.0f : m_all;
        const float f0 = __builtin_amdgcn_exp2f(m_run - m_sub);
        const float f1 = __builtin_amdgcn_exp2f(m1 - m_sub);
        l_run = l_run * f0 + s_stats[local][1] * f1;
        m_run = m_all;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 v = s_acc[(strip * (D / 8) + i * 4 + j) * 64 + lane];
                acc[i][4 * j] = acc[i][4 * j] * f0 + v.x * f1;
                acc[i][4 * j + 1] = acc[i][4 * j + 1] * f0 + v.y * f1;
                acc[i][4 * j + 2] = acc[i][4 * j + 2] * f0 + v.z * f1;
                acc[i][4 * j + 3] = acc[i][4 * j + 3] * f0 + v.w * f1;
            }
        }
    }
    if (local >= count) {
        return;
    }
    // acc[i][e]: dim 32 i + 8 (e / 4) + 4 q + e % 4 of the lane's column
    const int64_t row = s.first + column / G;
    if (splits == 1) {
        uint16_t* const out = a.out + row * a.out_stride + head * D + 4 * q;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool none = l_run == 0.0f;
                const uint32_t x = none ? 0u : pack(T{}, acc[i][4 * j] / l_run, acc[i][4 * j + 1] / l_run);
                const uint32_t y = none ? 0u : pack(T{}, acc[i][4 * j + 2] / l_run, acc[i][4 * j + 3] / l_run);
                *reinterpret_cast<uint2*>(out + 32 * i + 8 * j) = make_uint2(x, y);
            }
        }
        return;
    }
    const int64_t at = (row * a.q_heads + head) * splits + split;
    float* const part = a.partials + at * D + 4 * q;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<float4*>(part + 32 * i + 8 * j) =
                make_float4(acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]);
        }
    }
    if (q == 0) {
        *reinterpret_cast<float2*>(split_stats(a, D, splits) + 2 * at) = make_float2(m_run - Weights<T>::kUp, l_run);
    }
}

// -------------------------------------------------------------------- merge
// One row and head, or one of PARTS parts of its dims: GROUPS groups of lanes of 8 dims
// each, a group takes every GROUPS-th split, some of them requested together, and the
// groups' sums meet in LDS.  Rows outside [starts[0], starts[sequences]) belong to no sequence and are
// left alone.
template <typename T, int D, int GROUPS, int PARTS>
__global__ __launch_bounds__(kThreads / PARTS) void paged_attention_merge_kernel(PagedAttnArgs a, int splits) {
    constexpr int kLanes = D / 8 / PARTS;
    constexpr int kUnits = kThreads / PARTS / (kLanes * GROUPS);  // rows and heads of a block
    constexpr int kAhead = PARTS > 1 ? 8 : 4;
    __shared__ __attribute__((aligned(16))) float s_v[GROUPS > 1 ? GROUPS : 1][kUnits][GROUPS > 1 ? kLanes * 8 : 1];
    __shared__ float s_ml[GROUPS][kUnits][2];
    const int part = static_cast<int>(threadIdx.x) / kLanes;
    const int mine = part % kUnits;
    const int group = part / kUnits;
    const int64_t unit = static_cast<int64_t>(blockIdx.x / PARTS) * kUnits + mine;
    const int64_t row = unit / a.q_heads;
    const int head = static_cast<int>(unit % a.q_heads);
    const bool live = row < a.tokens && row >= a.starts[0] && row < a.starts[a.sequences];
    const int l0 = static_cast<int>(threadIdx.x) % kLanes * 8;  // of the part's dims
    const int d0 = static_cast<int>(blockIdx.x) % PARTS * (kLanes * 8) + l0;
    float m = kNegInf;
    float l = 0.0f;
    float v[8] = {};
    if (live) {
        const float2* const ml = reinterpret_cast<const float2*>(split_stats(a, D, splits)) + unit * splits;
        const float* const src = a.partials + unit * splits * D + d0;
        const int told = split_counts(a, D, splits)[unit];
        const int made = told < 0 ? 0 : (told < splits ? told : splits);
        for (int s0 = group; s0 < made; s0 += kAhead * GROUPS) {
            float2 w[kAhead];
            float4 x[kAhead], y[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int s = s0 + j * GROUPS < made ? s0 + j * GROUPS : made - 1;
                w[j] = ml[s];
            }
            float m_new = m;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                // (sum 0: no key of the row in this split)
                w[j].y = s0 + j * GROUPS < made ? w[j].y : 0.0f;
                m_new = fmaxf(m_new, w[j].y != 0.0f ? w[j].x : kNegInf);
                if (w[j].y != 0.0f) {
                    x[j] = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s0 + j * GROUPS) * D);
                    y[j] = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s0 + j * GROUPS) * D + 4);
                }
            }
            const float m_sub = m_new == kNegInf ? 0.0f : m_new;
            const float corr = __builtin_amdgcn_exp2f(m - m_sub);
            m = m_new;
            l *= corr;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] *= corr;
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (w[j].y != 0.0f) {
                    const float f = __builtin_amdgcn_exp2f(w[j].x - m_sub);
                    l = fmaf(w[j].y, f, l);
                    v[0] = fmaf(x[j].x, f, v[0]);
                    v[1] = fmaf(x[j].y, f, v[1]);
                    v[2] = fmaf(x[j].z, f, v[2]);
                    v[3] = fmaf(x[j].w, f, v[3]);
                    v[4] = fmaf(y[j].x, f, v[4]);
                    v[5] = fmaf(y[j].y, f, v[5]);
                    v[6] = fmaf(y[j].z, f, v[6]);
                    v[7] = fmaf(y[j].w, f, v[7]);
                }
            }
        }
    }
    if constexpr (GROUPS > 1) {
        *reinterpret_cast<float4*>(&s_v[group][mine][l0]) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(&s_v[group][mine][l0 + 4]) = make_float4(v[4], v[5], v[6], v[7]);
        if (l0 == 0) {
            s_ml[group][mine][0] = m;
            s_ml[group][mine][1] = l;
        }
        __syncthreads();
        if (group != 0) {
            return;
        }
        float m_all = m;
#pragma unroll
        for (int o = 1; o < GROUPS; ++o) {
            m_all = fmaxf(m_all, s_ml[o][mine][0]);
        }
        const float m_sub = m_all == kNegInf ? 0.0f : m_all;
        const float c = __builtin_amdgcn_exp2f(m - m_sub);
        l *= c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] *= c;
        }
#pragma unroll
        for (int o = 1; o < GROUPS; ++o) {
            const float f = __builtin_amdgcn_exp2f(s_ml[o][mine][0] - m_sub);
            l = fmaf(s_ml[o][mine][1], f, l);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = fmaf(s_v[o][mine][l0 + i], f, v[i]);
            }
        }
    }
    if (live) {
        put_column<T, D>(a, row, head, d0, v, m, l, 0, 1);
    }
}

template <typename T, int D, int GROUPS, int PARTS>
hipError_t launch_merge(const PagedAttnArgs& a, int64_t splits, hipStream_t stream) {
    constexpr int kUnits = kThreads / (D / 8 * GROUPS);
    const int64_t blocks = (a.tokens * a.q_heads + kUnits - 1) / kUnits;
    hipLaunchKernelGGL((paged_attention_merge_kernel<T, D, GROUPS, PARTS>), dim3(static_cast<unsigned>(blocks * PARTS)),
                       dim3(kThreads / PARTS), 0, stream, a, static_cast<int>(splits));
    return hipGetLastError();
}

template <typename T, int D>
hipError_t launch(const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    if (plan.few_blocks > 0) {
        hipLaunchKernelGGL((paged_attention_few_kernel<T, D>), dim3(static_cast<unsigned>(plan.few_blocks)), dim3(kThreads), 0,
                           stream, a, static_cast<int>(plan.splits), plan.tile_splits > 0 ? kFewRows : 0x7fffffff);
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) {
            return status;
        }
    }
    if (plan.tile_splits > 0) {
        const dim3 grid(static_cast<unsigned>(plan.slots * a.kv_heads * plan.tile_splits));
        const int few_rows = plan.few_blocks > 0 ? kFewRows : 0;
        if (plan.tile_groups == 1) {
            hipLaunchKernelGGL((paged_attention_tile_kernel<T, D, 1>), grid, dim3(kThreads), 0, stream, a,
                               static_cast<int>(plan.slots), static_cast<int>(plan.tile_splits),
                               static_cast<int>(plan.splits), few_rows);
        } else {
            hipLaunchKernelGGL((paged_attention_tile_kernel<T, D, 2>), grid, dim3(2 * kThreads), 0, stream, a,
                               static_cast<int>(plan.slots), static_cast<int>(plan.tile_splits),
                               static_cast<int>(plan.splits), few_rows);
        }
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) {
            return status;
        }
    }
    if (plan.splits > 1) {
        // many splits of few rows: groups work on them side by side, the parts of a row's
        // dims on as many CUs (16 splits of 16 rows 4.1 us with groups, 11.8 without; 256
        // splits 6.4 with parts, 8.2 without)
        if (plan.splits > 64 && a.tokens * a.q_heads < 256) {
            return launch_merge<T, D, 16, 4>(a, plan.splits, stream);
        }
        return plan.splits > 4 && a.tokens * a.q_heads < 2048 ? launch_merge<T, D, 16, 1>(a, plan.splits, stream)
                                                              : launch_merge<T, D, 1, 1>(a, plan.splits, stream);
    }
    return hipSuccess;
}

}  // namespace

PagedAttnPlan paged_attention_plan(int64_t tokens, int64_t sequences, int64_t max_query_len, int64_t max_kv_len,
                                   int64_t max_keys, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t workspace_bytes) {
    const int64_t group = q_heads / kv_heads;
    PagedAttnPlan p;
    const int64_t longest = max_query_len < tokens ? max_query_len : tokens;
    const int64_t rows = longest * group;
    const auto cap = [](int64_t v, int64_t most) { return v < 1 ? int64_t{1} : (v < most ? v : most); };
    const int64_t windows = (max_kv_len + kWindow - 1) / kWindow;
    // Few rows of every sequence go to the kernel for them where all sequences' windows
    // are at least 28 a CU (64 sequences of up to 8192 keys, 2 KV heads: 71 us, row tiles
    // 84; 32 36 and 43; 24 35 and 35; 16 23.6 and 22.9; 128 of up to 2000 38 and 45, of
    // 1000 30 and 27).
    const bool few = rows <= kFewRows && sequences * kv_heads * windows >= 7168;
    if (!few) {
        p.slots = tokens * group / kTileRows + sequences;
        const int64_t tiles = p.slots * kv_heads;
        // Splits of at least four windows, while the blocks run side by side: a window of a
        // block takes about 0.85 us, a merge 3 and 7 more for the partials of 256 full tiles
        // (600 tokens of 16 heads over 2 KV heads after 4000: 3 splits 39 us, one 67; 1000
        // after none: one 22.5, 2 splits 27.6; 1300 after 4000: 2 of 164 tiles 76, one 78).
        const int64_t side_by_side = tiles > 128 && tiles <= 192 ? 384 : 256;
        const auto cost = [&](int64_t s) { return 85 * windows / s + (s > 1 ? 300 + 700 * tiles * s / 256 : 0); };
        p.tile_splits = 1;
        for (int64_t s = 2; s <= (windows + 3) / 4 && s * tiles <= side_by_side; ++s) {
            p.tile_splits = cost(s) < cost(p.tile_splits) ? s : p.tile_splits;
        }
        // Sequences of one tile a KV head, whose partials are small: splits that even out
        // unequal lengths (64 sequences of 4 tokens and up to 8192 keys: 150 us without, 82
        // with; all of 2000 keys 39.7 and 37.8; of 1 to 5 tokens and up to 4000 keys 56 and
        // 48; but 8 tokens each after 2000 43 and 49).
        if (sequences > 1 && rows <= kTileRows) {
            const int64_t even = cap(1024 / tiles, (windows + 7) / 8);
            p.tile_splits = p.tile_splits > even ? p.tile_splits : even;
        }
        // Blocks of one K-group, two a CU, where they fill the chip; else of two, one a CU
        // (two of D = 64): 8192 tokens 269 us with one and 298 with two, 6000 166 and 175,
        // 4000 90 and 80, 3000 64 and 53; splits past 256 blocks 43 and 47 (D = 128), 60
        // and 56 (D = 64).
        p.tile_groups = tiles >= 512 || (head_dim == 128 && p.tile_splits > 1 && tiles * p.tile_splits > 256) ? 1 : 2;
    }
    // Beside longer sequences they go there where a tile would take more than 50 windows (a
    // chunk of 1000 and a token after 16000: 58 us, with tiles alone 113; 512 and 63 tokens
    // after up to 4000: 60 and 67; two chunks of 256 and 8 tokens: 40 and 30).
    int64_t few_splits = 0;
    if (few || (rows > kFewRows && tokens != sequences * longest && windows > 50 * p.tile_splits)) {
        // two blocks a CU; a stretch of at least one round of keys.  The longest sequence
        // may be cut into twice as many stretches as it were in a batch of such ones.
        const int64_t tiles = sequences * kv_heads * (((rows < kFewRows ? rows : kFewRows) + 15) / 16);
        const int64_t rounds = (max_kv_len + kRound - 1) / kRound;
        p.few_blocks = rounds < kFewBlocks && tiles * rounds < kFewBlocks ? tiles * rounds : kFewBlocks;
        few_splits = cap(2 * ((kFewBlocks + tiles - 1) / tiles) + 1, cap(rounds, 256));
    }
    const int64_t unit = tokens * q_heads * (head_dim + 2) * 4;
    const int64_t counts = tokens * q_heads * 4;
    const int64_t room = unit > 0 ? (workspace_bytes - counts) / unit : 0;
    // the few-row kernel counts its rounds in 31 bits
    const int64_t rounds = (max_keys + kRound - 1) / kRound;
    const bool countable = (tokens * q_heads / 16 + sequences * kv_heads) * rounds < (int64_t{1} << 31);
    const int64_t most = room > 1 && countable ? room : 1;
    few_splits = few_splits < most ? few_splits : most;
    p.tile_splits = p.tile_splits < most ? p.tile_splits : most;
    p.splits = few_splits > p.tile_splits ? few_splits : p.tile_splits;
    p.workspace_bytes = p.splits > 1 ? unit * p.splits + counts : 0;
    return p;
}

hipError_t launch_paged_attention(Act act, const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    if (a.head_dim == 64) {
        return act == Act::kBf16 ? launch<Bf16, 64>(a, plan, stream) : launch<F16, 64>(a, plan, stream);
    }
    return act == Act::kBf16 ? launch<Bf16, 128>(a, plan, stream) : launch<F16, 128>(a, plan, stream);
}

}  // namespace kc
