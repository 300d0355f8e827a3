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
        const uint16_t* const src = a.q + static_cast<int64_t>(s.first + column / G) * a.q_stride + head * D;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            qf[i] = *reinterpret_cast<const uint4*>(src + FewRows<T, D>::first_dim(q, i));
        }
    }
    FewRows<T, D> cached(a, table, g, keys, r, q);
    floatx4 acc[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        acc[i] = floatx4{};
    }
    float m_run = kNegInf;
    float l_run = 0.0f;
    if (unit < u_end) {
        cached.pages(unit);
        cached.place(unit);
        cached.fetch_k();
        cached.fetch_v();
        cached.pages(unit + 4);
    }
    for (; unit < u_end; unit += 4) {
        // V's rows, their 16-byte pieces swizzled so that the 8 rows of a
        // transposed half-wave read lie in different banks
        cached.store_v(s_v, [&](int row, int piece) __attribute__((always_inline)) {
            return row * (D * 2) + (piece ^ (((row & 7) << 1) % kPieces)) * 16;
        });
        const bool more = unit + 4 < u_end;
        if (more) {
            cached.place(unit + 4);
            cached.fetch_v();
            cached.pages(unit + 8);
        }
        floatx4 sc[2] = {floatx4{}, floatx4{}};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            sc[0] = mfma16(T{}, cached.k(0, i), qf[i], sc[0]);
            sc[1] = mfma16(T{}, cached.k(1, i), qf[i], sc[1]);
        }
        if (more) {
            cached.fetch_k();
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
    join_waves<T, D, CachedRow<T>>(a, s, table, g, c0, count, begin * kRound, u_end * kUnit, split, splits, acc, m_run, l_run,
                           cached.bad, s_mem, s_ml, s_redo);
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
        const int sum = wave_scan(mine, [](int x, int y) { return x + y; });
        longest = wave_scan(longest, [](int x, int y) { return x > y ? x : y; });
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
                few_rows_tile<T, D>(a, s, index, g, c0, at - first, splits > 1 ? to : 0x7fffffff / kRound, split, splits, s_mem, s_ml,
                          &s_redo);
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

// --------------------------------------------------------------- windows of 16 bits
// A window's rows straight to LDS.  K's pieces are swizzled by row against the 16 (D = 64:
// 8) rows that a read takes together, V's so that the 4 rows of a transposed half-wave
// read lie in different banks; the lane fetches the piece that belongs in its place.
template <typename T, int D>
struct AsyncWindow {
    using Rows = CachedRow<T>;
    static constexpr int waves(int groups) { return D == 64 && groups == 2 ? 4 : 2; }  // a SIMD
    static constexpr int kRowBytes = D * 2;
    static constexpr int kPieces = D / 8;
    static constexpr int kTileBytes = kWindow * kRowBytes;
    static constexpr int kKeyBytes = kTileBytes;
    static constexpr int kBufferBytes = 2 * kTileBytes;
    static constexpr int kSteps = D / 16;
    static constexpr int kLoadRows = 1024 / kRowBytes;        // rows of a wave's load
    static constexpr int kLoads = kWindow / (4 * kLoadRows);  // loads of a wave for a tile of K (and of V)
    const PagedAttnArgs& a;
    const int32_t* const table;
    const uint16_t* const kbase;
    const uint16_t* const vbase;
    const int keys, lane, wave;
    const int lane_row;  // of a load's kLoadRows rows, which begin at a multiple of that
    const uint8_t* const buffers;
    const uint32_t lds0;
    uint4 qf[kSteps];
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
          lane(lane_id), wave(wave_id), lane_row(lane_id / kPieces), buffers(lds),
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
    __device__ __forceinline__ void start(int w, int step, int) {
        look(w);
        fetch(w, 0);
        look(w + step);
    }
    __device__ __forceinline__ void arrive(int) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the window is in LDS
    }
    __device__ __forceinline__ void next(int w, int step, int w_end, int buffer) {
        if (w < w_end) {
            fetch(w, buffer);
            look(w + step);
        }
    }
    __device__ __forceinline__ void query(const uint16_t* row) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            qf[i] = *reinterpret_cast<const uint4*>(row + 8 * (lane >> 5) + 16 * i);
        }
    }
    template <typename Late>
    __device__ __forceinline__ void scores(floatx16 (&sc)[2], int buffer, Late late) {
        tile_scores<T, D, AsyncWindow>(sc, qf, buffers + buffer * kBufferBytes, lane, late);
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
    const int l0 = static_cast<int>(threadIdx.x) % kLanes * 8;  // of the part's dims
    const int d0 = static_cast<int>(blockIdx.x) % PARTS * (kLanes * 8) + l0;
    const float2* const ml = reinterpret_cast<const float2*>(split_stats(a, D, splits)) + unit * splits;
    const float* const src = a.partials + unit * splits * D + d0;
    float2 w[kAhead];
    float4 x[kAhead], y[kAhead];
    // Groups of few splits ask for their first ones before they know how many there are (the
    // partials have room for `splits`): otherwise four loads wait for one another.  64 rows
    // of 16 heads over up to 9 splits 6.3 us so and 5.4 now.
    if (GROUPS > 1 && row < a.tokens) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int s = group + j * GROUPS;
            if (s < splits) {
                w[j] = ml[s];
                x[j] = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * D);
                y[j] = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * D + 4);
            }
        }
    }
    const bool live = row < a.tokens && row >= a.starts[0] && row < a.starts[a.sequences];
    float m = kNegInf;
    float l = 0.0f;
    float v[8] = {};
    if (live) {
        const int told = split_counts(a, D, splits)[unit];
        const int made = told < 0 ? 0 : (told < splits ? told : splits);
        for (int s0 = group; s0 < made; s0 += kAhead * GROUPS) {
            const bool ahead = GROUPS > 1 && s0 == group;
            if (!ahead) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const int s = s0 + j * GROUPS < made ? s0 + j * GROUPS : made - 1;
                    w[j] = ml[s];
                }
            }
            float m_new = m;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                // (sum 0: no key of the row in this split)
                w[j].y = s0 + j * GROUPS < made ? w[j].y : 0.0f;
                m_new = fmaxf(m_new, w[j].y != 0.0f ? w[j].x : kNegInf);
                if (!ahead && w[j].y != 0.0f) {
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
hipError_t launch_merges(const PagedAttnArgs& a, int64_t splits, bool fours, hipStream_t stream) {
    // (groups of four for up to 16 splits: those 64 rows 4.4 us, with 16 groups 5.4; the
    // attention over 16-bit rows keeps its order of sums)
    if (fours && splits <= 16 && a.tokens * a.q_heads < 2048) {
        return launch_merge<T, D, 4, 1>(a, splits, stream);
    }
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
    if (plan.few_blocks > 0) {
        hipLaunchKernelGGL((paged_attention_few_kernel<T, D>), dim3(static_cast<unsigned>(plan.few_blocks)), dim3(kThreads), 0,
                           stream, a, static_cast<int>(plan.splits), plan.tile_splits > 0 ? kFewRows : 0x7fffffff);
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) {
            return status;
        }
    }
    return launch_tiles<T, D, AsyncWindow<T, D>>(a, plan, kFewRows, false, stream);
}

}  // namespace

hipError_t launch_paged_merge(Act act, const PagedAttnArgs& a, int64_t splits, bool fours, hipStream_t stream) {
    if (a.head_dim == 64) {
        return act == Act::kBf16 ? launch_merges<Bf16, 64>(a, splits, fours, stream) : launch_merges<F16, 64>(a, splits, fours, stream);
    }
    return act == Act::kBf16 ? launch_merges<Bf16, 128>(a, splits, fours, stream) : launch_merges<F16, 128>(a, splits, fours, stream);
}

PagedAttnPlan paged_attention_plan(int64_t tokens, int64_t sequences, int64_t max_query_len, int64_t max_kv_len,
                                   int64_t max_keys, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t workspace_bytes) {
    const int64_t group = q_heads / kv_heads;
    PagedAttnPlan p;
    const int64_t longest = max_query_len < tokens ? max_query_len : tokens;
    const int64_t rows = longest * group;
    const int64_t windows = (max_kv_len + kWindow - 1) / kWindow;
    // Few rows of every sequence go to the kernel for them where all sequences' windows
    // are at least 28 a CU (64 sequences of up to 8192 keys, 2 KV heads: 71 us, row tiles
    // 84; 32 36 and 43; 24 35 and 35; 16 23.6 and 22.9; 128 of up to 2000 38 and 45, of
    // 1000 30 and 27).
    const bool few = rows <= kFewRows && sequences * kv_heads * windows >= 7168;
    if (!few) {
        plan_tiles(p, tokens, sequences, group, rows, windows, kv_heads, head_dim);
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
