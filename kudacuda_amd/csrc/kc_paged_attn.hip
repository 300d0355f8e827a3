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
#include "kc_paged_attn.h"

namespace kc {
namespace {

// ---------------------------------------------------------------- rows of 16 bits
template <typename T>
struct CachedRow {
    using Place = int64_t;
    static __device__ __forceinline__ Place place_of(const PagedAttnArgs& a, int page, int key, int g, bool& bad) {
        return key_row(a, page, key, bad) + g * a.head_stride;
    }
    static __device__ __forceinline__ float element(const uint16_t* pool, Place at, int d) { return T::load(pool[at + d]); }
};

// A wave's 32 keys: lane (r, q) holds dims 32 i + 8 q .. + 7 of keys r and 16 + r.
template <typename T, int D>
struct FewRows : CachedRow<T> {
    static constexpr int kSteps = D / 32;
    const PagedAttnArgs& a;
    const int32_t* const table;
    const uint16_t* const kbase;
    const uint16_t* const vbase;
    const int keys, r, q;
    bool bad = false;
    int64_t at[2];
    int page[2];
    uint4 kf[2][kSteps], vf[2][kSteps];

    static __device__ __forceinline__ int first_dim(int q, int i) { return 32 * i + 8 * q; }
    __device__ __forceinline__ FewRows(const PagedAttnArgs& args, const int32_t* table_row, int g, int n, int lane_r, int lane_q)
        : a(args), table(table_row), kbase(args.k + g * args.head_stride), vbase(args.v + g * args.head_stride), keys(n),
          r(lane_r), q(lane_q) {}
    __device__ __forceinline__ void pages(int u) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = u * kUnit + 16 * t + r;
            page[t] = table[(key < keys ? key : keys - 1) >> a.page_shift];
        }
    }
    __device__ __forceinline__ void place(int u) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = u * kUnit + 16 * t + r;
            at[t] = key_row(a, page[t], key < keys ? key : keys - 1, bad) + 8 * q;
        }
    }
    __device__ __forceinline__ void fetch(uint4 (&f)[2][kSteps], const uint16_t* base) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                f[t][i] = load_stream(reinterpret_cast<const uint4*>(base + at[t] + 32 * i));
            }
        }
    }
    __device__ __forceinline__ void fetch_k() { fetch(kf, kbase); }
    __device__ __forceinline__ void fetch_v() { fetch(vf, vbase); }
    template <typename At>
    __device__ __forceinline__ void store_v(uint8_t* s_v, At at_piece) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                *reinterpret_cast<uint4*>(s_v + at_piece(16 * t + r, 4 * i + q)) = vf[t][i];
            }
        }
    }
    __device__ __forceinline__ uint4 k(int t, int i) const { return kf[t][i]; }
};

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

// A window's rows straight to LDS.  K's pieces are swizzled by row against the 16 (D = 64:
// 8) rows that a read takes together, V's so that the 4 rows of a transposed half-wave
// read lie in different banks; the lane fetches the piece that belongs in its place.
template <typename T, int D>
struct AsyncWindow {
    using Rows = CachedRow<T>;
    static constexpr int kRowBytes = D * 2;
    static constexpr int kPieces = D / 8;
    static constexpr int kTileBytes = kWindow * kRowBytes;
    static constexpr int kLoadRows = 1024 / kRowBytes;        // rows of a wave's load
    static constexpr int kLoads = kWindow / (4 * kLoadRows);  // loads of a wave for a tile of K (and of V)
    const PagedAttnArgs& a;
    const int32_t* const table;
    const uint16_t* const kbase;
    const uint16_t* const vbase;
    const int keys, lane, wave;
    const int lane_row;  // of a load's kLoadRows rows, which begin at a multiple of that
    const uint32_t lds0;
    // Whole windows of pages that hold a load's rows together (and begin within 4 GB
    // of a pool's beginning times a page id): a load's base is the wave's, its lanes'
    // offsets are the same in every window.  Bytes from here on.
    const int page_mask;
    const bool together;
    const uint32_t page_bytes, token_bytes;
    const uint8_t* k_at[kLoads];
    const uint8_t* v_at[kLoads];
    uint32_t k_lane[kLoads];
    uint32_t v_lane[kLoads];
    int page = 0;  // pages of the window's groups of kLoadRows keys, one a lane
    bool bad = false;

    static __device__ __forceinline__ int k_place(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int v_place(int row) { return D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }
    __device__ __forceinline__ int piece_of(int row, bool value) const {
        return (lane % kPieces) ^ (value ? v_place(row) : k_place(row));
    }
    __device__ __forceinline__ AsyncWindow(const PagedAttnArgs& args, const int32_t* table_row, int g, int n, int lane_id,
                                           int wave_id, const uint8_t* lds)
        : a(args), table(table_row), kbase(args.k + g * args.head_stride), vbase(args.v + g * args.head_stride), keys(n),
          lane(lane_id), wave(wave_id), lane_row(lane_id / kPieces),
          lds0(__builtin_amdgcn_readfirstlane(lds_address(lds) + wave_id * 1024)), page_mask((1 << args.page_shift) - 1),
          together(page_mask + 1 >= kLoadRows && args.token_stride < (1 << 26) && args.page_stride < (1 << 30)),
          page_bytes(static_cast<uint32_t>(2 * args.page_stride)), token_bytes(static_cast<uint32_t>(2 * args.token_stride)) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int row0 = (j * 4 + wave) * kLoadRows;
            const int64_t in_page = static_cast<int64_t>(row0 & page_mask) * token_bytes;
            k_at[j] = reinterpret_cast<const uint8_t*>(kbase) + in_page;
            v_at[j] = reinterpret_cast<const uint8_t*>(vbase) + in_page;
            k_lane[j] = lane_row * token_bytes + 16 * piece_of(row0 + lane_row, false);
            v_lane[j] = lane_row * token_bytes + 16 * piece_of(row0 + lane_row, true);
        }
    }
    __device__ __forceinline__ void look(int w) {
        const int key = w * kWindow + lane % (4 * kLoads) * kLoadRows;
        page = table[(key < keys ? key : keys - 1) >> a.page_shift];
    }
    __device__ __forceinline__ void fetch(int w, int buffer) {
        const uint32_t lds = lds0 + buffer * (2 * kTileBytes);
        if (together && (w + 1) * kWindow <= keys) {
            const bool out = static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.num_pages);
            bad |= out;
            const int inside = out ? 0 : page;
            // (pages of more than a window: where the window begins in its page)
            const int64_t shift = static_cast<int64_t>((w * kWindow) & page_mask) * token_bytes;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const uint32_t id = __builtin_amdgcn_readlane(inside, j * 4 + wave);
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
    }
    __device__ __forceinline__ void arrive(bool, int) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the window is in LDS
    }
};

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
hipError_t launch_merges(const PagedAttnArgs& a, int64_t splits, hipStream_t stream) {
    // many splits of few rows: groups work on them side by side, the parts of a row's
    // dims on as many CUs (16 splits of 16 rows 4.1 us with groups, 11.8 without; 256
    // splits 6.4 with parts, 8.2 without)
    if (splits > 64 && a.tokens * a.q_heads < 256) {
        return launch_merge<T, D, 16, 4>(a, splits, stream);
    }
    return splits > 4 && a.tokens * a.q_heads < 2048 ? launch_merge<T, D, 16, 1>(a, splits, stream)
                                                     : launch_merge<T, D, 1, 1>(a, splits, stream);
}

template <typename T, int D>
hipError_t launch(const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    return launch_kernels<T, D, FewRows<T, D>, AsyncWindow<T, D>>(a, plan, stream);
}

}  // namespace

hipError_t launch_paged_merge(Act act, const PagedAttnArgs& a, int64_t splits, hipStream_t stream) {
    if (a.head_dim == 64) {
        return act == Act::kBf16 ? launch_merges<Bf16, 64>(a, splits, stream) : launch_merges<F16, 64>(a, splits, stream);
    }
    return act == Act::kBf16 ? launch_merges<Bf16, 128>(a, splits, stream) : launch_merges<F16, 128>(a, splits, stream);
}

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
