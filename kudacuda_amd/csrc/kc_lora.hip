// Low-rank adapters of many requests beside a shared projection:
//     out = base + s_a (x A_a^T) B_a^T
// for the rows of adapter a; A_a is [rank, in], B_a [out, rank].  The caller's plan groups
// the rows: a tile is up to 64 rows of one adapter.
//
// Two launches (one where both are small), bound by bytes: the adapters' factors where rows are few (64 adapters of a
// row each, 2048 -> 11008, ranks 8 to 64, 53 MB: 7.0 + 14.4 us, 2.5 TB/s), else the inputs,
// the base rows and the results (2000 rows of one adapter of rank 16, 2048 -> 11008, 97 MB:
// 7.6 + 23.1 us, 3.2 TB/s; 8 chunks of 2996 rows, 11008 -> 2048, 79 MB: 19.9 + 10.4, 2.6 TB/s); one
// row is latency: 6.7 us, places, two products and their sums one after the other.
//
// The first forms u = x A^T, a tile's rows by up to 64 ranks a block, over a share of `in`
// (few tiles are split so that the adapters' bytes come through all CUs); the four waves
// take alternate steps of 32 and meet in LDS.  The second sums the shares in order, splits
// u into two 16-bit parts (normalised by a power of two a row, so that fp16 keeps 22 bits
// of it and bf16 16) and takes 64 outputs a wave: up to rank 16 both parts lie along one
// product's inner axis of 32, above the factor meets one after the other.  Operands come
// straight from memory: both factors' rows are contiguous along the inner axis.  (Lanes
// that read them in their order in memory, as rows through LDS would, gain a tenth of the
// first launch before the exchange is paid for.)  Loads are plain: streamed (nontemporal)
// factors cost 22 %, since several loads touch a line.
#include <type_traits>

#include "kc_device.h"
#include "kc_kernels.h"

namespace kc {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kStep = 32;            // of the inner axis, a matrix instruction
constexpr int kBlockStep = 4 * kStep;  // of the four waves
// Tiles of 16 rows on average or fewer have kernels for 16 rows at a time (calls with 64
// adapters, 2048 -> 11008: a row each of ranks 8 to 64 20.1 us, with room for 64 rows 26.9;
// 16 rows each of rank 16 18.4 and 22.6).
inline bool few_rows(int64_t tokens, int64_t tile_count) { return tokens <= 16 * tile_count; }
// Blocks of the first launch that tiles are split into.  More shorten it and lengthen the
// second, which sums the shares in each of its blocks.  Calls with 256, 512 and 1024, us,
// 11008 -> 2048: few rows a tile, 64 adapters of a row, ranks 8 to 64, 24.2, 21.6, 23.3, 16 of
// rank 64 14.6, 15.1, 15.3; more rows, the 8 chunks above 29.3, 30.5, 32.2, 16 chunks of 100,
// rank 32, 22.4, 25.1, 27.1, 4 of 700, rank 128, 68, 74, 90, 4 of 2000, rank 64, 97, 94, 101.
inline int64_t inner_blocks(int64_t tokens, int64_t tile_count) { return few_rows(tokens, tile_count) ? 512 : 256; }

__device__ __forceinline__ floatx4 mfma16(Bf16, uint4 a, uint4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma16(F16, uint4 a, uint4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pair(Bf16, float lo, float hi) { return pack2(lo, hi); }
__device__ __forceinline__ uint32_t pair(F16, float lo, float hi) {
    typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
    const halfx2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
}

// A tile of the plan; whatever it holds, rows stay inside the order and the adapter inside
// the pools (adapter -1: none).
struct Tile {
    int adapter;
    int rank;
    int first;
    int count;
};
__device__ __forceinline__ Tile tile_of(const LoraArgs& a, int index) {
    const int32_t* const p = a.tiles + 3 * static_cast<int64_t>(index);
    Tile t;
    const int tokens = static_cast<int>(a.tokens);
    t.adapter = __builtin_amdgcn_readfirstlane(p[0]);
    t.first = __builtin_amdgcn_readfirstlane(p[1]);
    t.count = __builtin_amdgcn_readfirstlane(p[2]);
    t.count = t.first < 0 || t.first >= tokens || t.count < 0 ? 0 : t.count;
    t.count = t.count < kLoraTile ? t.count : kLoraTile;
    t.count = t.count < tokens - t.first ? t.count : tokens - t.first;
    t.rank = 0;
    if (t.adapter >= 0 && t.adapter < a.adapters) {
        const int rank = __builtin_amdgcn_readfirstlane(a.ranks[t.adapter]);
        t.rank = rank < 0 ? 0 : (rank < a.max_rank ? rank : static_cast<int>(a.max_rank));
    }
    return t;
}
// Row `i` of a tile in the inputs and outputs, -1 if there is none.
__device__ __forceinline__ int row_of(const LoraArgs& a, const Tile& t, int i) {
    const int row = i < t.count ? a.order[t.first + i] : -1;
    return row < a.tokens ? row : -1;
}

// ------------------------------------------------------------------- x A^T
// RT tiles of 16 ranks from rank0 on, SUBS of 16 rows: a wave's share, its part of every
// kBlockStep.  acc[s][i][e]: rank 16 i + 4 q + e of row 16 s + r.
template <typename T, int RT, int SUBS, int AHEAD>
__device__ __forceinline__ void inner_sums(const LoraArgs& a, const Tile& t, int rank0, int k_begin, int k_end,
                                           floatx4 (&acc)[SUBS][RT]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int r = lane & 15;
    const int q = lane >> 4;
    const uint16_t* const factor = a.a + static_cast<int64_t>(t.adapter) * a.max_rank * a.in_features;
    const uint16_t* arow[RT];
    const uint16_t* xrow[SUBS];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int rank = rank0 + 16 * i + r;
        arow[i] = factor + static_cast<int64_t>(rank < t.rank ? rank : t.rank - 1) * a.in_features;
    }
#pragma unroll
    for (int i = 0; i < SUBS; ++i) {
        const int row = row_of(a, t, 16 * i + r);
        xrow[i] = a.x + static_cast<int64_t>(row < 0 ? 0 : row) * a.x_stride;
    }
#pragma unroll
    for (int s = 0; s < SUBS; ++s) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            acc[s][i] = floatx4{};
        }
    }
    const int tiles = (t.rank - rank0 + 15) / 16;
    // steps on their way while others are multiplied
    uint4 av[AHEAD][RT], xv[AHEAD][SUBS];
    const auto request = [&](int n, int k0) __attribute__((always_inline)) {
        const int k = k0 + 8 * q;
        const bool in = k < k_end;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            av[n][i] = make_uint4(0, 0, 0, 0);
            if (in && i < tiles) {
                av[n][i] = *reinterpret_cast<const uint4*>(arow[i] + k);
            }
        }
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            xv[n][s] = make_uint4(0, 0, 0, 0);
            if (in && 16 * s < t.count) {
                xv[n][s] = *reinterpret_cast<const uint4*>(xrow[s] + k);
            }
        }
    };
    int k0 = k_begin + wave * kStep;
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
        request(n, k0 + n * kBlockStep);
    }
    for (; k0 < k_end; k0 += AHEAD * kBlockStep) {
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int s = 0; s < SUBS; ++s) {
                    acc[s][i] = mfma16(T{}, av[n][i], xv[n][s], acc[s][i]);
                }
            }
            request(n, k0 + (n + AHEAD) * kBlockStep);
        }
    }
}

template <typename T, int RT, int SUBS>
__device__ __forceinline__ void inner_tile(const LoraArgs& a, const Tile& t, int rank0, int k_begin, int k_end,
                                           float* partials, float (*s_u)[16][RT * 16 + 4]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int r = lane & 15;
    const int q = lane >> 4;
    floatx4 acc[SUBS][RT];
    inner_sums<T, RT, SUBS, RT * SUBS <= 2 ? 4 : 2>(a, t, rank0, k_begin, k_end, acc);
    // the waves' shares meet in LDS
#pragma unroll
    for (int s = 0; s < SUBS; ++s) {
        if (16 * s >= t.count) {
            break;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            *reinterpret_cast<float4*>(&s_u[wave][r][16 * i + 4 * q]) =
                make_float4(acc[s][i][0], acc[s][i][1], acc[s][i][2], acc[s][i][3]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * RT * 4; i += kThreads) {
            const int row = i / (RT * 4);
            const int rank = i % (RT * 4) * 4;
            if (16 * s + row < t.count && rank0 + rank < t.rank) {
                float4 sum = *reinterpret_cast<const float4*>(&s_u[0][row][rank]);
#pragma unroll
                for (int w = 1; w < 4; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(&s_u[w][row][rank]);
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                *reinterpret_cast<float4*>(partials + static_cast<int64_t>(t.first + 16 * s + row) * a.pitch + rank0 + rank) = sum;
            }
        }
    }
}

// Sixteen rows after sixteen of a tile, or (SUBS 4) a whole one together.
template <typename Work>
__device__ __forceinline__ void rows_of_tile(const Tile& t, int step, Work work) {
    for (int row = 0; row < t.count; row += step) {
        Tile part = t;
        part.first += row;
        part.count = t.count - row < step ? t.count - row : step;
        if (row > 0) {
            __syncthreads();
        }
        work(part);
    }
}

template <typename T, int RT, int SUBS>
__global__ __launch_bounds__(kThreads) void lora_inner_kernel(LoraArgs a, int splits, int chunks) {
    __shared__ __attribute__((aligned(16))) float s_u[4][16][RT * 16 + 4];
    const int chunk = static_cast<int>(blockIdx.x) % chunks;
    const int split = static_cast<int>(blockIdx.x) / chunks % splits;
    const Tile t = tile_of(a, static_cast<int>(blockIdx.x) / chunks / splits);
    const int rank0 = chunk * RT * 16;
    if (t.count == 0 || rank0 >= t.rank) {
        return;
    }
    const int in = static_cast<int>(a.in_features);
    const int steps = (in + kBlockStep - 1) / kBlockStep;
    const int per_split = (steps + splits - 1) / splits * kBlockStep;
    const int begin = split * per_split < in ? split * per_split : in;
    const int end = begin + per_split < in ? begin + per_split : in;
    float* const partials = a.partials + static_cast<int64_t>(split) * a.tokens * a.pitch;
    rows_of_tile(t, 16 * SUBS, [&](const Tile& part) __attribute__((always_inline)) {
        inner_tile<T, RT, SUBS>(a, part, rank0, begin, end, partials, s_u);
    });
}

// ------------------------------------------------------------------- u B^T
// A block: a tile's rows by `groups` groups of 64 outputs a wave; the first group's factors
// and base rows are requested before anything else.  LDS holds a row's u first in fp32, then
// as pieces of 8 ranks: `half` first parts, then as many second ones.  Up to 16 ranks both
// parts are one instruction's (pieces 0, 1 of each), else a factor's 32 ranks meet the
// first and then the second parts.
constexpr int outer_sets(int rank_tiles, int subs) { return subs == 1 && rank_tiles <= 4 ? 2 : 1; }

template <typename T, int RT, int SUBS, bool WHOLE>
__device__ __forceinline__ void outer_tile(const LoraArgs& a, const Tile& t, int splits, int column0, int groups,
                                           uint8_t* s_row, float* s_factor, float (*s_u)[16][RT * 16 + 4]) {
    constexpr int kRowBytes = RT * 64 + 16;
    constexpr int kFactors = (RT + 1) / 2;  // of 32 ranks
    constexpr int kSets = outer_sets(RT, SUBS);
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;
    const int q = lane >> 4;
    const int pieces = (t.rank + 7) / 8;
    const bool one = pieces <= 2;
    const int half = one ? 2 : (pieces + 3) / 4 * 4;
    const int factors = t.rank > 0 ? (pieces + 3) / 4 : 0;
    const int out = static_cast<int>(a.out_features);
    // Loads without conditions, which would be waited for all together: a factor's rows are a
    // buffer of their bytes (past it and for pieces that are none a load reads nothing), and
    // base rows that are none are read from another (base is output where there is none).
    const uint16_t* const rows_b = a.b + static_cast<int64_t>(t.adapter < 0 ? 0 : t.adapter) * a.max_rank * a.out_features;
    const int row_bytes = 16 * pieces;
    const __amdgpu_buffer_rsrc_t factor =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(rows_b), 0, out * row_bytes, 0x00027000);
    const uint16_t* const base_rows = a.base != nullptr ? a.base : a.out;
    const int64_t base_stride = a.base != nullptr ? a.base_stride : a.out_stride;
    const float scale = t.rank > 0 ? a.scales[t.adapter] : 0.0f;
    int rows[SUBS];
#pragma unroll
    for (int s = 0; s < SUBS; ++s) {
        rows[s] = row_of(a, t, 16 * s + r);
    }
    // The outputs of row r of operand i: lane (r, q) of a result then has outputs 32 h + 8 q
    // .. + 7 of its token, from operands 2 h and 2 h + 1.
    uint4 bv[kSets][kFactors][4], base[kSets][SUBS][2];
    const auto request = [&](int set, int o0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int o = o0 + 32 * (i >> 1) + 8 * (r >> 2) + 4 * (i & 1) + (r & 3);
#pragma unroll
            for (int f = 0; f < kFactors; ++f) {
                const int piece = one ? q & 1 : 4 * f + q;
                bv[set][f][i] = __builtin_bit_cast(
                    uint4, __builtin_amdgcn_raw_buffer_load_b128(factor, piece < pieces ? o * row_bytes + 16 * piece : 0x7ffffff0, 0, 0));
            }
        }
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int o = o0 + 32 * h + 8 * q;
                base[set][s][h] = *reinterpret_cast<const uint4*>(base_rows + static_cast<int64_t>(rows[s] < 0 ? 0 : rows[s]) * base_stride +
                                                                  (o < out ? o : 0));
            }
        }
    };
    request(0, column0 + wave * 64);
    if (t.rank > 0) {
        if constexpr (WHOLE) {
            floatx4 acc[SUBS][RT];
            inner_sums<T, RT, SUBS, RT <= 2 ? 8 : 4>(a, t, 0, 0, static_cast<int>(a.in_features), acc);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                *reinterpret_cast<float4*>(&s_u[wave][r][16 * i + 4 * q]) =
                    make_float4(acc[0][i][0], acc[0][i][1], acc[0][i][2], acc[0][i][3]);
            }
            __syncthreads();
        }
        for (int i = tid; i < 16 * SUBS * RT * 4; i += kThreads) {
            const int row = i / (RT * 4);
            const int rank = i % (RT * 4) * 4;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if constexpr (WHOLE) {
                if (row < t.count && rank < t.rank) {
                    sum = *reinterpret_cast<const float4*>(&s_u[0][row][rank]);
#pragma unroll
                    for (int w = 1; w < 4; ++w) {
                        const float4 v = *reinterpret_cast<const float4*>(&s_u[w][row][rank]);
                        sum.x += v.x;
                        sum.y += v.y;
                        sum.z += v.z;
                        sum.w += v.w;
                    }
                }
            } else if (row < t.count && rank < t.rank) {
                const float* const p = a.partials + static_cast<int64_t>(t.first + row) * a.pitch + rank;
                const int64_t share = a.tokens * a.pitch;
                constexpr int kTogether = 8;  // shares on their way (past the last one it is read again)
                for (int s0 = 0; s0 < splits; s0 += kTogether) {
                    float4 v[kTogether];
#pragma unroll
                    for (int n = 0; n < kTogether; ++n) {
                        v[n] = *reinterpret_cast<const float4*>(p + (s0 + n < splits ? s0 + n : splits - 1) * share);
                    }
#pragma unroll
                    for (int n = 0; n < kTogether; ++n) {
                        const bool more = s0 + n < splits;
                        sum.x = more ? sum.x + v[n].x : sum.x;
                        sum.y = more ? sum.y + v[n].y : sum.y;
                        sum.z = more ? sum.z + v[n].z : sum.z;
                        sum.w = more ? sum.w + v[n].w : sum.w;
                    }
                }
            }
            sum.y = rank + 1 < t.rank ? sum.y : 0.0f;
            sum.z = rank + 2 < t.rank ? sum.z : 0.0f;
            sum.w = rank + 3 < t.rank ? sum.w : 0.0f;
            *reinterpret_cast<float4*>(s_row + row * kRowBytes + rank * 4) = sum;
        }
        __syncthreads();
        const int row = tid / 4;
        const int part = tid % 4;
        float4 u[RT];
        float most = 0.0f;
        if (row < 16 * SUBS) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                u[i] = *reinterpret_cast<const float4*>(s_row + row * kRowBytes + (16 * i + 4 * part) * 4);
                most = fmaxf(most, fmaxf(fmaxf(fabsf(u[i].x), fabsf(u[i].y)), fmaxf(fabsf(u[i].z), fabsf(u[i].w))));
            }
        }
        most = fmaxf(most, __shfl_xor(most, 1, 4));
        most = fmaxf(most, __shfl_xor(most, 2, 4));
        __syncthreads();
        if (row < 16 * SUBS) {
            // u 2^-e lies below 1: its parts fit fp16 (e kept where 2^-e and 2^e are normal)
            int e = static_cast<int>(__float_as_uint(most) >> 23) - 126;
            e = e > -120 ? (e < 120 ? e : 120) : -120;
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            if (part == 0) {
                s_factor[row] = scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int piece = 2 * i + part / 2;
                if (piece < half) {
                    const float v[4] = {u[i].x * down, u[i].y * down, u[i].z * down, u[i].w * down};
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        hi[j] = pair(T{}, v[2 * j], v[2 * j + 1]);
                        const float x = v[2 * j] - T::load(static_cast<uint16_t>(hi[j] & 0xffffu));
                        const float y = v[2 * j + 1] - T::load(static_cast<uint16_t>(hi[j] >> 16));
                        lo[j] = pair(T{}, x == x ? x : 0.0f, y == y ? y : 0.0f);  // (infinities have no rest)
                    }
                    uint8_t* const at = s_row + row * kRowBytes + part % 2 * 8;
                    *reinterpret_cast<uint2*>(at + piece * 16) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(at + (half + piece) * 16) = make_uint2(lo[0], lo[1]);
                }
            }
        }
        __syncthreads();
    }
    const auto multiply = [&](int set, int o0) __attribute__((always_inline)) {
        floatx4 acc[SUBS][4];
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[s][i] = floatx4{};
            }
        }
#pragma unroll
        for (int f = 0; f < kFactors; ++f) {
            if (f < factors) {
#pragma unroll
                for (int s = 0; s < SUBS; ++s) {
                    const uint8_t* const at = s_row + (16 * s + r) * kRowBytes + (4 * f + q) * 16;
                    const uint4 hi = *reinterpret_cast<const uint4*>(at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[s][i] = mfma16(T{}, bv[set][f][i], hi, acc[s][i]);
                    }
                    if (!one) {
                        const uint4 lo = *reinterpret_cast<const uint4*>(at + half * 16);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            acc[s][i] = mfma16(T{}, bv[set][f][i], lo, acc[s][i]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            if (rows[s] < 0) {
                continue;
            }
            const float f = t.rank > 0 ? s_factor[16 * s + r] : 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int o = o0 + 32 * h + 8 * q;
                if (o < out) {
                    float v[8] = {};
                    if (a.base != nullptr) {
                        unpack8<T>(base[set][s][h], v);
                    }
                    if (t.rank > 0) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            v[e] = fmaf(acc[s][2 * h + e / 4][e % 4], f, v[e]);
                        }
                    }
                    *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(rows[s]) * a.out_stride + o) =
                        make_uint4(pair(T{}, v[0], v[1]), pair(T{}, v[2], v[3]), pair(T{}, v[4], v[5]), pair(T{}, v[6], v[7]));
                }
            }
        }
    };
    int o0 = column0 + wave * 64;
    if constexpr (kSets == 2) {
        // (a group past the block's last asks for none)
        int n = 0;
        for (; n + 1 < groups; n += 2) {
            request(1, o0 + 256);
            multiply(0, o0);
            request(0, n + 2 < groups ? o0 + 512 : out);
            multiply(1, o0 + 256);
            o0 += 512;
        }
        if (n < groups) {
            multiply(0, o0);
        }
    } else {
        multiply(0, o0);
        for (int n = 1; n < groups; ++n) {
            o0 += 256;
            request(0, o0);
            multiply(0, o0);
        }
    }
}

template <typename T, int RT, int SUBS, bool WHOLE>
__global__ __launch_bounds__(kThreads, SUBS == 1 && !WHOLE ? 3 : 2) void lora_outer_kernel(LoraArgs a, int splits, int blocks, int groups) {
    __shared__ __attribute__((aligned(16))) uint8_t s_u[WHOLE ? 4 * 16 * (RT * 16 + 4) * 4 : 16];
    __shared__ __attribute__((aligned(16))) uint8_t s_row[16 * SUBS * (RT * 64 + 16)];
    __shared__ float s_factor[16 * SUBS];
    const Tile t = tile_of(a, static_cast<int>(blockIdx.x) / blocks);
    const int column0 = static_cast<int>(blockIdx.x) % blocks * groups * 256;
    if (t.count == 0 || (t.rank == 0 && a.out == a.base)) {
        return;
    }
    rows_of_tile(t, 16 * SUBS, [&](const Tile& part) __attribute__((always_inline)) {
        outer_tile<T, RT, SUBS, WHOLE>(a, part, splits, column0, groups, s_row, s_factor,
                                         reinterpret_cast<float (*)[16][RT * 16 + 4]>(s_u));
    });
}

template <typename T, int RT, int SUBS, bool WHOLE>
hipError_t launch_outer(const LoraArgs& a, const LoraPlan& plan, hipStream_t stream) {
    // One group of 64 outputs a wave, more where there are blocks enough without.  Few rows a
    // tile are bound by what a block does before its first product, and the groups after the
    // first come while others are multiplied: 64 adapters, 64 rows of 11008 outputs, ranks 8
    // to 64 -- two groups 16.1 us, four 14.1, six 16.9, rank 16 alone 9.8, 8.0 and 8.0 (with
    // loads under conditions, waited for all together, four took 16.8 and 11.0); one adapter
    // and row 4.7 with one.  Tiles of 64 rows are bound by their rows: 2000 rows of
    // 11008 outputs -- one group 25.9 us, four 29 (with twice the shares that the first launch
    // makes now: one 23.1).
    constexpr int kSets = outer_sets(RT, SUBS);
    const int64_t columns = (a.out_features + 255) / 256;
    int64_t groups = a.tile_count * columns / (kSets == 2 ? 640 : 2048);
    groups = groups < 2 ? 1 : (groups < 16 ? groups / kSets * kSets : 16);
    const int64_t blocks = (columns + groups - 1) / groups;
    hipLaunchKernelGGL((lora_outer_kernel<T, RT, SUBS, WHOLE>), dim3(static_cast<unsigned>(a.tile_count * blocks)),
                       dim3(kThreads), 0, stream, a, static_cast<int>(plan.splits), static_cast<int>(blocks),
                       static_cast<int>(groups));
    return hipGetLastError();
}

template <typename T, int RT, int SUBS>
hipError_t launch(const LoraArgs& a, const LoraPlan& plan, hipStream_t stream) {
    if constexpr (SUBS == 1 && RT <= 4) {
        // Small factors and few blocks: each forms u for itself, and a launch is saved, 4 us of
        // a call (one row, 2048 -> 2048: rank 16 6.8 us and 3.6 + 4.6 in two launches, rank 32
        // 8.9 and 4.1 + 5.1; but rank 64 13.3 and 5.0 + 6.6, 11008 -> 2048 with rank 16 16.4 and
        // 4.0 + 5.7; rank 16, 16 adapters 8.5 and 4.0 + 4.7, 64 11.4 and 4.6 + 5.6).
        if (a.pitch * a.in_features <= 65536 && a.tile_count * ((a.out_features + 255) / 256) <= 128) {
            return launch_outer<T, RT, SUBS, true>(a, plan, stream);
        }
    }
    constexpr int kChunk = RT < 4 ? RT : 4;  // ranks of 16 that a block of the first product takes
    const int64_t chunks = (a.pitch / 16 + kChunk - 1) / kChunk;
    hipLaunchKernelGGL((lora_inner_kernel<T, kChunk, SUBS>), dim3(static_cast<unsigned>(a.tile_count * plan.splits * chunks)),
                       dim3(kThreads), 0, stream, a, static_cast<int>(plan.splits), static_cast<int>(chunks));
    const hipError_t status = hipGetLastError();
    return status != hipSuccess ? status : launch_outer<T, RT, SUBS, false>(a, plan, stream);
}

template <typename T, int SUBS>
hipError_t launch(const LoraArgs& a, const LoraPlan& plan, hipStream_t stream) {
    const int64_t tiles = a.pitch / 16;
    return tiles <= 1 ? launch<T, 1, SUBS>(a, plan, stream)
                      : (tiles <= 2 ? launch<T, 2, SUBS>(a, plan, stream)
                                    : (tiles <= 4 ? launch<T, 4, SUBS>(a, plan, stream) : launch<T, 8, SUBS>(a, plan, stream)));
}

template <typename T>
hipError_t launch(const LoraArgs& a, const LoraPlan& plan, hipStream_t stream) {
    return few_rows(a.tokens, a.tile_count) ? launch<T, 1>(a, plan, stream) : launch<T, kLoraTile / 16>(a, plan, stream);
}

}  // namespace

LoraPlan lora_plan(int64_t tokens, int64_t tile_count, int64_t max_rank, int64_t in_features) {
    LoraPlan p;
    p.pitch = (max_rank + 15) / 16 * 16;
    const int64_t steps = (in_features + kBlockStep - 1) / kBlockStep;
    const int64_t wanted = tile_count > 0 ? inner_blocks(tokens, tile_count) / tile_count : 1;
    // (at least four steps a split: their loads are on their way together)
    const int64_t most = (steps + 3) / 4;
    p.splits = wanted < 1 ? 1 : (wanted < most ? wanted : most);
    p.workspace_bytes = p.splits * tokens * p.pitch * 4;
    return p;
}

hipError_t launch_lora(Act act, const LoraArgs& a, const LoraPlan& plan, hipStream_t stream) {
    return act == Act::kBf16 ? launch<Bf16>(a, plan, stream) : launch<F16>(a, plan, stream);
}

}  // namespace kc
