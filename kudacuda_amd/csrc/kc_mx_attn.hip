// Attention over a paged cache of microscaled numbers (kc_mx.h): what kc_paged_attn.hip
// computes, on the numbers that the cache holds.
//
// An element times its block's power of two is a number of the queries' type, so rows are
// unpacked on their way to the same matrix products (a conversion a pair, power included),
// and results are those of the attention over the cache's unpacked rows.  A block whose
// byte says NaN unpacks to NaN, and goes the way of the 16-bit cache's NaN: columns that
// do not see it are summed again with care.
#include "kc_mx.h"
#include "kc_paged_attn.h"

namespace kc {
namespace {

// A row's place: its elements' and its blocks' bytes in a pool.
struct MxPlace {
    int64_t elements;
    int64_t blocks;
};

template <typename T, int D, int BITS>
struct MxRow {
    using Place = MxPlace;
    static __device__ __forceinline__ MxPlace place_of(const PagedAttnArgs& a, int page, int key, int g, bool& bad) {
        bad |= static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.num_pages);
        const int64_t id = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages) ? page : 0;
        const int64_t row = (static_cast<int64_t>(g) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
        return {id * a.page_stride + row * (D * BITS / 8), id * a.page_stride + a.block_offset + row * (D / kMxBlock)};
    }
    static __device__ __forceinline__ float element(const uint16_t* pool, const MxPlace& at, int d) {
        const uint8_t* const bytes = reinterpret_cast<const uint8_t*>(pool);
        constexpr std::integral_constant<int, BITS> bits{};
        const float power = mx_power(bytes[at.blocks + d / kMxBlock]);
        const uint32_t byte = bytes[at.elements + d * BITS / 8];
        const uint32_t pair = mx_pair<0>(T{}, bits, byte, power);
        return BITS == 4 && (d & 1) != 0 ? high<T>(pair) : low<T>(pair);
    }
};

// A wave's 32 keys: lane (r, q) holds dims D / 4 * q .. of keys r and 16 + r, which share
// a power of two; the 16 keys' rows lie in one page.
template <typename T, int D, int BITS>
struct MxFewRows : MxRow<T, D, BITS> {
    static constexpr int kSteps = D / 32;
    static constexpr int kBytes = D * BITS / 32;  // of a lane
    static constexpr int kWords = kBytes / 4;
    const PagedAttnArgs& a;
    const int32_t* const table;
    const uint8_t* const kpool;
    const uint8_t* const vpool;
    const int g, keys, r, q;
    bool bad = false;
    int page[2];
    MxPlace at[2];
    uint32_t kw[2][kWords], vw[2][kWords];
    uint32_t kb[2], vb[2];

    static __device__ __forceinline__ int first_dim(int q, int i) { return D / 4 * q + 8 * i; }
    __device__ __forceinline__ MxFewRows(const PagedAttnArgs& args, const int32_t* table_row, int head, int n, int lane_r,
                                         int lane_q)
        : a(args), table(table_row), kpool(reinterpret_cast<const uint8_t*>(args.k)),
          vpool(reinterpret_cast<const uint8_t*>(args.v)), g(head), keys(n), r(lane_r), q(lane_q) {}
    __device__ __forceinline__ void pages(int u) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = u * kUnit + 16 * t;
            page[t] = table[(key < keys ? key : keys - 1) >> a.page_shift];
        }
    }
    __device__ __forceinline__ void place(int u) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = u * kUnit + 16 * t + r;
            // (a key past the end reads the last one, in the page of the 16 or before it)
            at[t] = MxRow<T, D, BITS>::place_of(a, page[t], key < keys ? key : keys - 1, g, bad);
            at[t].elements += q * kBytes;
            at[t].blocks += q * (D / 4) / kMxBlock;
        }
    }
    __device__ __forceinline__ void fetch(uint32_t (&w)[2][kWords], uint32_t (&b)[2], const uint8_t* pool) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            get_words(w[t], pool + at[t].elements);
            b[t] = pool[at[t].blocks];
        }
    }
    __device__ __forceinline__ void fetch_k() { fetch(kw, kb, kpool); }
    __device__ __forceinline__ void fetch_v() { fetch(vw, vb, vpool); }
    template <typename At>
    __device__ __forceinline__ void store_v(uint8_t* s_v, At at_piece) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float power = mx_power(vb[t]);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                *reinterpret_cast<uint4*>(s_v + at_piece(16 * t + r, kSteps * q + i)) =
                    mx_unpack8<T, BITS>(vw[t] + i * (BITS / 4), power);
            }
        }
    }
    __device__ __forceinline__ uint4 k(int t, int i) const {
        return mx_unpack8<T, BITS>(kw[t] + i * (BITS / 4), mx_power(kb[t]));
    }
};

// A window's rows through registers: a lane takes a block of a row, of K and of V (D =
// 64: of one of them).  V's rows are dealt so that 16 lanes' stores, and the transposed
// reads of 4 rows, lie in different banks.
template <typename T, int D, int BITS>
struct MxWindow {
    using Rows = MxRow<T, D, BITS>;
    static constexpr int kParts = D / 64;
    static constexpr int kWords = kMxBlock * BITS / 32;
    static constexpr int kTileBytes = kWindow * D * 2;
    const PagedAttnArgs& a;
    const int32_t* const table;
    const int g, keys;
    uint8_t* const lds;
    int row[kParts];
    int block[kParts];
    bool value[kParts];
    int page[kParts];
    uint32_t words[kParts][kWords];
    uint32_t bytes[kParts];
    bool bad = false;

    static __device__ __forceinline__ int k_place(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int v_place(int row) {
        return (D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
    __device__ __forceinline__ MxWindow(const PagedAttnArgs& args, const int32_t* table_row, int head, int n, int lane, int wave,
                                        uint8_t* buffers)
        : a(args), table(table_row), g(head), keys(n), lds(buffers) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            if constexpr (D == 128) {
                value[p] = p == 1;
                block[p] = lane & 3;
                row[p] = 16 * wave + (value[p] ? (lane >> 4) + 4 * ((lane >> 2) & 3) : lane >> 2);
            } else {
                value[p] = wave >= 2;
                block[p] = lane & 1;
                row[p] = 32 * (wave & 1) + (value[p] ? ((lane >> 1) & 1) + 4 * ((lane >> 2) & 3) + 2 * ((lane >> 4) & 1) +
                                                           16 * (lane >> 5)
                                                     : lane >> 1);
            }
            page[p] = 0;
            bytes[p] = 0;
        }
    }
    __device__ __forceinline__ int key_of(int w, int p) const {
        const int key = w * kWindow + row[p];
        return key < keys ? key : keys - 1;
    }
    __device__ __forceinline__ void look(int w) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            page[p] = table[key_of(w, p) >> a.page_shift];
        }
    }
    __device__ __forceinline__ void fetch(int w, int) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            const MxPlace at = Rows::place_of(a, page[p], key_of(w, p), g, bad);
            const uint8_t* const pool = reinterpret_cast<const uint8_t*>(value[p] ? a.v : a.k);
            get_words(words[p], pool + at.elements + block[p] * (4 * kWords));
            bytes[p] = pool[at.blocks + block[p]];
        }
    }
    __device__ __forceinline__ void arrive(bool live, int buffer) {
        if (!live) {
            return;
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            uint8_t* const at = lds + buffer * (2 * kTileBytes) + (value[p] ? kTileBytes : 0) + row[p] * (D * 2);
            const int place = value[p] ? v_place(row[p]) : k_place(row[p]);
            const float power = mx_power(bytes[p]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<uint4*>(at + ((4 * block[p] + j) ^ place) * 16) =
                    mx_unpack8<T, BITS>(words[p] + j * (BITS / 4), power);
            }
        }
    }
};

template <typename T, int D, int BITS>
hipError_t launch(const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    return launch_kernels<T, D, MxFewRows<T, D, BITS>, MxWindow<T, D, BITS>>(a, plan, stream);
}
template <typename T>
hipError_t launch(int bits, const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    if (a.head_dim == 64) {
        return bits == 4 ? launch<T, 64, 4>(a, plan, stream) : launch<T, 64, 8>(a, plan, stream);
    }
    return bits == 4 ? launch<T, 128, 4>(a, plan, stream) : launch<T, 128, 8>(a, plan, stream);
}

}  // namespace

PagedAttnPlan mx_attention_plan(int, int64_t tokens, int64_t sequences, int64_t max_query_len, int64_t max_kv_len,
                                int64_t max_keys, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                int64_t workspace_bytes) {
    return paged_attention_plan(tokens, sequences, max_query_len, max_kv_len, max_keys, q_heads, kv_heads, head_dim,
                                workspace_bytes);
}

hipError_t launch_mx_attention(Act act, int bits, const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    return act == Act::kBf16 ? launch<Bf16>(bits, a, plan, stream) : launch<F16>(bits, a, plan, stream);
}

}  // namespace kc
