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

// ------------------------------------------------------------------ few rows
// The two tiles of 16 keys that a wave takes next: their rows lie in one page each, whose
// place is the wave's; K unpacked into the first product's operand, V through LDS.
//
// (The scaled matrix instructions would meet K as it is stored, the query as e4m3 numbers
// in parts, and save the unpacking.  But they align the products of neighbouring dims to
// the largest of them and drop what lies below 2^-13 of it, where the 16-bit instructions
// keep 2^-23: small dims beside large ones vanish.)
template <typename T, int D, int BITS>
struct MxQuery {
    static constexpr int kSteps = D / 32;
    uint4 part[kSteps];
    __device__ __forceinline__ void load(const uint16_t* row, int q) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            part[i] = *reinterpret_cast<const uint4*>(row + D / 4 * q + 8 * i);
        }
    }
    template <int WORDS>
    __device__ __forceinline__ floatx4 scores(const uint32_t (&key)[WORDS], uint32_t byte) const {
        floatx4 sc = floatx4{};
        const float power = mx_power(byte);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            sc = mfma16(T{}, mx_unpack8<T, BITS>(key + i * (BITS / 4), power), part[i], sc);
        }
        return sc;
    }
};

template <typename T, int D, int BITS>
struct MxFewTile {
    static constexpr int kRowBytes = D * BITS / 8;
    static constexpr int kWords = kRowBytes / 16;  // of a lane's quarter of a row
    static constexpr int kSteps = D / 32;
    static constexpr int kDepth = 2;  // units that are on their way

    struct Raw {
        uint32_t k[2][kWords], v[2][kWords];
        uint32_t k_byte[2], v_byte[2];
    };

    static __device__ __forceinline__ void run(const PagedAttnArgs& a, const Sequence& s, int index, int g, int c0, int begin,
                                               int end, int split, int splits, uint8_t* s_mem, float (*s_ml)[16][2],
                                               int* s_redo) {
        constexpr int kPieces = D / 8;  // 16-byte pieces of an unpacked row
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
        const int first_pos = s.kv_len - s.q_len + c0 / G;
        const int ends = s.kv_len - s.q_len + (c0 + count - 1) / G + 1;
        // (the wave's, and told to be: the loop and the pages' buffers take them as scalars)
        const int keys = __builtin_amdgcn_readfirstlane(ends > 0 ? ends : 0);
        const int units = (keys + kUnit - 1) / kUnit;
        const int u_end = __builtin_amdgcn_readfirstlane(end * 4 < units ? end * 4 : units);
        int unit = __builtin_amdgcn_readfirstlane(begin * 4 + wave);
        const int head = __builtin_amdgcn_readfirstlane(g << a.page_shift);

        // Pages of the wave's next 64 tiles, one a lane: read in the loop, their ids would come
        // behind the rows that are on their way, since loads return in order.
        const int last_tile = (keys > 0 ? keys - 1 : 0) & ~15;
        const int page_mask = (1 << a.page_shift) - 1;
        int pages = 0;
        int pages_from = unit;
        bool bad = false;
        const auto look = [&](int u) __attribute__((always_inline)) {
            const int key = (u + lane / 2 * 4) * kUnit + lane % 2 * 16;
            pages = table[(key < last_tile ? key : last_tile) >> a.page_shift];
            asm volatile("" : "+v"(pages));  // (waited for here, once in 32 units, not wherever it is read)
            pages_from = u;
        };
        const int lane_bytes = q * (kRowBytes / 4);
        const int b_lane = q * (D / 4) / kMxBlock;
        const uint8_t* const kpool = reinterpret_cast<const uint8_t*>(a.k);
        const uint8_t* const vpool = reinterpret_cast<const uint8_t*>(a.v);
        // A unit behind the wave's last one is asked for like the others, from a page of no bytes:
        // loads under a condition would be waited for all together.
        const auto fetch = [&](int u, Raw& raw) __attribute__((always_inline)) {
            if (u == pages_from + 4 * 32 && u < u_end) {
                look(u);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int id = __builtin_amdgcn_readlane(pages, ((u - pages_from) / 2 + t) & 63);
                const bool out = static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.num_pages);
                bad |= out && u < u_end;
                int key = u * kUnit + 16 * t;
                key = key < last_tile ? key : last_tile;
                // (rows past the end read the last one)
                const int row = r < keys - 1 - key ? r : keys - 1 - key;
                const int64_t at = static_cast<int64_t>(out ? 0 : id) * a.page_stride;
                const int bytes = out || u >= u_end ? 0 : static_cast<int>(a.page_stride);
                const auto k_page = page_buffer(kpool + at, bytes);
                const auto v_page = page_buffer(vpool + at, bytes);
                const int first = head + (key & page_mask) + row;
                const int elements = first * kRowBytes;
                const int block = static_cast<int>(a.block_offset) + first * (D / kMxBlock) + b_lane;
                get_words(raw.k[t], k_page, elements + lane_bytes);
                get_words(raw.v[t], v_page, elements + lane_bytes);
                raw.k_byte[t] = __builtin_amdgcn_raw_buffer_load_b8(k_page, block, 0, 0);
                raw.v_byte[t] = __builtin_amdgcn_raw_buffer_load_b8(v_page, block, 0, 0);
            }
        };

        // (the query is requested first: loads return in order)
        MxQuery<T, D, BITS> query;
        query.load(a.q + static_cast<int64_t>(s.first + column / G) * a.q_stride + (g * G + column % G) * D, q);
        Raw raw[kDepth];
        look(unit);
        fetch(unit, raw[0]);
        asm volatile("" ::: "memory");  // (asked for in this order)
        fetch(unit + 4, raw[1]);
        floatx4 acc[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            acc[i] = floatx4{};
        }
        float m_run = kNegInf;
        float l_run = 0.0f;
        const auto step = [&](Raw& now) __attribute__((always_inline)) {
            floatx4 sc[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t] = query.scores(now.k[t], now.k_byte[t]);
            }
            // V's rows, their 16-byte pieces swizzled so that the 8 rows of a
            // transposed half-wave read lie in different banks
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float power = mx_power(now.v_byte[t]);
                const int row = 16 * t + r;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int piece = (kSteps * q + i) ^ (((row & 7) << 1) % kPieces);
                    *reinterpret_cast<uint4*>(s_v + row * (D * 2) + piece * 16) =
                        mx_unpack8<T, BITS>(now.v[t] + i * (BITS / 4), power);
                }
            }
            fetch(unit + 4 * kDepth, now);
            // sc[t][i]: key 16 t + 4 q + i of the unit
            if (unit * kUnit + kUnit > first_pos + 1) {
                const int rel = pos - unit * kUnit - 4 * q;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[t][i] = 16 * t + i <= rel ? sc[t][i] : kNegInf;
                    }
                }
            }
            float mx = kNegInf;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    mx = fmaxf(mx, sc[t][i]);
                }
            }
            const auto p16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = halves_max(fmaxf(__uint_as_float(p16[0]), __uint_as_float(p16[1])));
            const float m_new = fmaxf(m_run, mx * a.scale_log2);
            if (__any(m_new > m_run)) {
                const float corr = __builtin_amdgcn_exp2f(m_run - (m_new == kNegInf ? 0.0f : m_new));
                l_run *= corr;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[i][e] *= corr;
                    }
                }
                m_run = m_new;
            }
            // weights as two 16-bit parts, as over 16-bit rows
            const float m_w = (m_run == kNegInf ? 0.0f : m_run) - Weights<T>::kFewUp;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[e / 2][2 * (e % 2)], a.scale_log2, -m_w));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[e / 2][2 * (e % 2) + 1], a.scale_log2, -m_w));
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
                acc[i] = mfma16(T{}, vt, ph, acc[i]);
                acc[i] = mfma16(T{}, vt, pl, acc[i]);
            }
        };
        // (no way out between the two, which would come back to the first as far as the counts of
        // loads on their way are concerned)
        while (unit + 4 < u_end) {
            step(raw[0]);
            unit += 4;
            step(raw[1]);
            unit += 4;
        }
        if (unit < u_end) {
            step(raw[0]);
        }
        join_waves<T, D, MxRow<T, D, BITS>>(a, s, table, g, c0, count, begin * kRound, u_end * kUnit, split, splits, acc, m_run,
                                            l_run, bad, s_mem, s_ml, s_redo);
    }
};

// A block takes one piece: a share of the rounds of 128 keys of one (sequence, KV head,
// tile of 16 rows).  Sequences are shared evenly into pieces of at most `longest` rounds,
// the least number for which the pieces of the batch fit on the chip at once.  (Blocks of
// equal stretches of all sequences' rounds, as over 16-bit rows, end together, but most of
// them then begin and end two pieces, and what a piece costs beside its rows -- places
// found one after the other, the query, the waves' meeting -- is as long as two or
// three rounds here.)  Bound by memory once rows flow: a round more on 512 blocks of heads of
// 128 in 4 bits is 1.6 us, 5.4 TB/s; beside it 7 us of launch, places, query and meeting.  64
// sequences of up to 8192 keys, 82 MB, 23.5 us, of heads of 64, 41 MB, 18.2; 120000 keys of one
// in 8 bits, 63 MB, 16.9.
constexpr int64_t kFewAtOnce = 512;  // two blocks a CU
constexpr int kMxFewRows = 32;

// Sums over the block's threads up to and with this one, a wave at a time: the waves' sums
// are in s_part behind the barrier.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (*s_part)[N]) {
    const int wave = static_cast<int>(threadIdx.x) >> 6;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = wave_scan(v[i], [](int x, int y) { return x + y; });
    }
    if ((threadIdx.x & 63) == 63) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s_part[wave][i] = v[i];
        }
    }
    __syncthreads();
}
template <int N>
__device__ __forceinline__ int block_sum(int (*s_part)[N], int i) {
    return __builtin_amdgcn_readfirstlane(s_part[0][i] + s_part[1][i] + s_part[2][i] + s_part[3][i]);
}

// Of a batch's pieces: candidates for the longest's rounds, from an even share of all on in
// steps to where every tile may have a short last piece.
constexpr int kTries = 4;
__device__ __forceinline__ int least_piece(int rounds, int tiles, int most, int splits, int& step) {
    const int at_once = static_cast<int>(kFewAtOnce);
    const int spare = at_once - tiles > at_once / 4 ? at_once - tiles : at_once / 4;
    int least = (rounds + at_once - 1) / at_once;
    const int allowed = (most + splits - 1) / splits;
    least = least > allowed ? least : allowed;
    const int enough = (rounds + spare - 1) / spare;
    step = enough > least ? (enough - least + kTries - 2) / (kTries - 1) : 1;
    return least;
}

// ceil(n / d) for n < 2^23: the quotient of the nearest floats is at most one off.
__device__ __forceinline__ int parts_of(int n, int d) {
    const int up = n + d - 1;
    int q = static_cast<int>(static_cast<float>(up) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
    q -= q * d > up ? 1 : 0;
    return q + ((q + 1) * d <= up ? 1 : 0);
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads, 2) void mx_few_kernel(PagedAttnArgs a, int splits, int few_rows) {
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[4 * kUnit * D * 2];
    __shared__ float s_ml[4][16][2];
    __shared__ int s_total[4][2], s_most[4], s_tries[4][kTries];
    __shared__ int s_found[6];
    __shared__ int s_redo;
    const int tid = threadIdx.x;
    const int sequences = static_cast<int>(a.sequences);
    const int kv_heads = static_cast<int>(a.kv_heads);
    const auto pieces_of = [&](const Line& line, int longest) __attribute__((always_inline)) {
        return kv_heads * line.tiles * parts_of(line.rounds, longest);
    };
    int pieces;   // of the batch
    int longest;  // rounds of a piece
    int before = 0;      // pieces before this thread's run of sequences (one of up to 256)
    int own_pieces = 0;  // and in it
    const int per_thread = (sequences + kThreads - 1) / kThreads;
    const int run = tid * per_thread;
    Sequence own = {};
    if (sequences == 1) {
        own = wave_sequence(a, 0);
        const Line line = line_of(a, own, few_rows, splits);
        const int heads = kv_heads * line.tiles;
        const int share = heads > 0 ? static_cast<int>(kFewAtOnce) / heads : 1;  // pieces of a tile
        const int parts = share < 1 ? 1 : (share < splits ? share : splits);
        longest = (line.rounds + parts - 1) / parts;
        pieces = pieces_of(line, longest);
    } else if (sequences <= 64) {
        // a lane a sequence, in every wave alike: no wave waits for another
        const int lane = tid & 63;
        const auto add = [](int x, int y) { return x + y; };
        const auto last = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, 63); };
        Line line = {};
        bool descending = false;
        if (lane < sequences) {
            own = sequence(a, lane);
            descending = a.starts[lane + 1] < a.starts[lane];
            line = line_of(a, own, few_rows, splits);
        }
        const int rounds = last(wave_scan(length_of(a, line), add));
        const int tiles = last(wave_scan(kv_heads * line.tiles, add));
        const int most = last(wave_scan(line.tiles > 0 && line.rounds > 1 ? line.rounds : 1, [](int x, int y) { return x > y ? x : y; }));
        if (__any(descending) || rounds == 0) {
            return;
        }
        int step;
        const int least = least_piece(rounds, tiles, most, splits, step);
        longest = 0;
        pieces = 0;
#pragma unroll
        for (int t = kTries - 1; t >= 0; --t) {
            const int mine = pieces_of(line, least + t * step);
            const int after = wave_scan(mine, add);
            const int sum = last(after);
            if (sum <= static_cast<int>(kFewAtOnce) || t == kTries - 1) {
                longest = least + t * step;
                pieces = sum;
                own_pieces = mine;
                before = after - mine;
            }
        }
    } else {
        const int run_end = run + per_thread < sequences ? run + per_thread : sequences;
        Line line = {};
        int total[2] = {};  // rounds, tiles
        int most = 1;
        bool descending = false;  // (such starts name no rows: their lengths need not fit the line)
        for (int i = run; i < run_end; ++i) {
            own = sequence(a, i);
            descending |= a.starts[i + 1] < a.starts[i];
            line = line_of(a, own, few_rows, splits);
            total[0] += length_of(a, line);
            total[1] += kv_heads * line.tiles;
            most = line.tiles > 0 && line.rounds > most ? line.rounds : most;
        }
        most = wave_scan(descending ? 0x7fffffff : most, [](int x, int y) { return x > y ? x : y; });
        if ((tid & 63) == 63) {
            s_most[tid >> 6] = most;
        }
        block_scan(total, s_total);
        total[0] = block_sum(s_total, 0);
        total[1] = block_sum(s_total, 1);
        most = __builtin_amdgcn_readfirstlane(max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3])));
        if (most == 0x7fffffff || total[0] == 0) {
            return;
        }
        int step;
        const int least = least_piece(total[0], total[1], most, splits, step);
        int tries[kTries] = {};
        for (int i = run; i < run_end; ++i) {
            if (per_thread > 1) {
                line = line_of(a, sequence(a, i), few_rows, splits);
            }
#pragma unroll
            for (int t = 0; t < kTries; ++t) {
                tries[t] += pieces_of(line, least + t * step);
            }
        }
        int mine[kTries];
#pragma unroll
        for (int t = 0; t < kTries; ++t) {
            mine[t] = tries[t];
        }
        block_scan(tries, s_tries);
        longest = 0;
        pieces = 0;
#pragma unroll
        for (int t = kTries - 1; t >= 0; --t) {
            const int sum = block_sum(s_tries, t);
            if (sum <= static_cast<int>(kFewAtOnce) || t == kTries - 1) {  // (more tiles than fit at once: the last)
                longest = least + t * step;
                pieces = sum;
                own_pieces = mine[t];
                before = tries[t] - mine[t];
                for (int w = 0; w < (tid >> 6); ++w) {
                    before += s_tries[w][t];
                }
            }
        }
    }
    const int piece = static_cast<int>(blockIdx.x);
    if (piece >= pieces) {
        return;
    }
    int index = 0;
    int first = 0;  // the first piece of the sequence
    Sequence s = own;
    if (sequences > 1 && sequences <= 64) {
        const uint64_t found = __ballot(before <= piece && piece < before + own_pieces);
        index = __builtin_amdgcn_readfirstlane(__builtin_ctzll(found));  // (pieces are all somebody's)
        first = __builtin_amdgcn_readlane(before, index);
        s.first = __builtin_amdgcn_readlane(own.first, index);
        s.q_len = __builtin_amdgcn_readlane(own.q_len, index);
        s.kv_len = __builtin_amdgcn_readlane(own.kv_len, index);
        s.bad = __builtin_amdgcn_readlane(static_cast<int>(own.bad), index) != 0;
    } else if (sequences > 1) {
        // the thread whose sequences the piece is of tells which
        if (before <= piece && piece < before + own_pieces) {
            int i = run;
            for (; per_thread > 1; ++i) {
                own = sequence(a, i);
                const int next = before + pieces_of(line_of(a, own, few_rows, splits), longest);
                if (piece < next) {
                    break;
                }
                before = next;
            }
            s_found[0] = i;
            s_found[1] = before;
            s_found[2] = own.first;
            s_found[3] = own.q_len;
            s_found[4] = own.kv_len;
            s_found[5] = own.bad;
        }
        __syncthreads();
        index = __builtin_amdgcn_readfirstlane(s_found[0]);
        first = __builtin_amdgcn_readfirstlane(s_found[1]);
        s.first = __builtin_amdgcn_readfirstlane(s_found[2]);
        s.q_len = __builtin_amdgcn_readfirstlane(s_found[3]);
        s.kv_len = __builtin_amdgcn_readfirstlane(s_found[4]);
        s.bad = __builtin_amdgcn_readfirstlane(s_found[5]) != 0;
    }
    const Line line = line_of(a, s, few_rows, splits);
    const int parts = parts_of(line.rounds, longest);
    const int split = (piece - first) % parts;
    const int tile = (piece - first) / parts;
    const int g = tile / line.tiles;
    const int c0 = tile % line.tiles * 16;
    const int rest = s.q_len * static_cast<int>(a.group) - c0;
    const int count = rest < 16 ? rest : 16;
    if (s.bad) {
        if (split == 0) {
            nan_columns<T, D>(a, s, g, c0, count, splits);
        }
        return;
    }
    if (split == 0 && splits > 1) {
        tell_splits<D>(a, s, g, c0, count, parts, splits);
    }
    const int share = (line.rounds + parts - 1) / parts;
    const int end = share * (split + 1) < line.rounds ? share * (split + 1) : line.rounds;
    MxFewTile<T, D, BITS>::run(a, s, index, g, c0, split * share, splits > 1 ? end : 0x7fffffff / kRound, split, splits, s_mem,
                               s_ml, &s_redo);
}

// ----------------------------------------------------------------- row tiles
// A window's rows through registers, unpacked into what the tiles over 16-bit rows have in
// LDS: a wave takes 16 rows of K and of V, which lie in one page, a lane a block of a row of
// both (D = 64: lanes 0 .. 31 K's, the others V's).  V's rows are dealt so that 16 lanes'
// stores, and the transposed reads of 4 rows, lie in different banks.  The products, the
// arithmetic and LDS are each about as busy there, and unpacking adds to two of them: a
// prompt of 8192 tokens takes 283 us in 4 bits and 291 in 8, 970 and 945 TFLOP/s, where it
// takes 279 over 16-bit rows.  In 8 bits the rows' words do not fit beside the rest: 2 to 10
// registers a lane are spilled, in heads of 128 and in heads of 64 with one K-group; none in
// 4 bits.  (Measured instead: the same behind the barrier, a window later, 5 % slower; K kept
// packed, its products by scaled instructions, whose sums are coarse as told above, 1 % faster
// in bf16 heads of 128 in 4 bits, 2 % slower in 8, 9 % in fp16 and 18 % in heads of 64.)
template <typename T, int D, int BITS>
struct MxWindow {
    using Rows = MxRow<T, D, BITS>;
    static constexpr int waves(int groups) { return D == 64 && groups == 1 ? 3 : 2; }  // a SIMD
    static constexpr int kParts = D / 64;
    static constexpr int kRowBytes = D * BITS / 8;
    static constexpr int kWords = kMxBlock * BITS / 32;
    static constexpr int kTileBytes = kWindow * D * 2;
    static constexpr int kKeyBytes = kTileBytes;
    static constexpr int kBufferBytes = 2 * kTileBytes;
    const PagedAttnArgs& a;
    const int32_t* const table;
    const int keys, lane, wave;
    const int64_t head_row;  // the head's first row in a page
    const int last_tile;
    uint8_t* const lds;
    const uint8_t* pool[kParts];
    int row[kParts];  // of the wave's 16
    int block[kParts];
    int place[kParts];  // in LDS
    int page = 0;
    uint32_t words[kParts][kWords];
    uint32_t bytes[kParts];
    uint4 qf[D / 16];
    bool bad = false;

    static __device__ __forceinline__ int k_place(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int v_place(int row) {
        return (D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
    __device__ __forceinline__ MxWindow(const PagedAttnArgs& args, const int32_t* table_row, int head, int n, int lane_id, int wave_id,
                                        uint8_t* buffers)
        : a(args), table(table_row), keys(n), lane(lane_id), wave(wave_id), head_row(static_cast<int64_t>(head) << args.page_shift),
          last_tile((n > 0 ? n - 1 : 0) & ~15), lds(buffers) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            const bool value = D == 128 ? p == 1 : lane >= 32;
            if constexpr (D == 128) {
                block[p] = lane & 3;
                row[p] = value ? (lane >> 4) + 4 * ((lane >> 2) & 3) : lane >> 2;
            } else {
                block[p] = lane & 1;
                row[p] = value ? ((lane >> 1) & 1) + 4 * ((lane >> 2) & 3) + 2 * ((lane >> 4) & 1) : lane >> 1;
            }
            pool[p] = reinterpret_cast<const uint8_t*>(value ? a.v : a.k);
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                words[p][i] = 0;
            }
            place[p] = (value ? kTileBytes : 0) + (16 * wave + row[p]) * (D * 2) +
                       16 * ((4 * block[p]) ^ (value ? v_place(row[p]) : k_place(row[p])));
            bytes[p] = 0;
        }
    }
    __device__ __forceinline__ int tile_of(int w) const {
        const int key = w * kWindow + 16 * wave;
        return key < last_tile ? key : last_tile;
    }
    __device__ __forceinline__ void look(int w) { page = table[tile_of(w) >> a.page_shift]; }
    __device__ __forceinline__ void fetch(int w) {
        const int key = tile_of(w);
        const int id = __builtin_amdgcn_readfirstlane(page);
        const bool out = static_cast<uint32_t>(id) >= static_cast<uint32_t>(a.num_pages);
        bad |= out;
        const int64_t first = head_row + (key & ((1 << a.page_shift) - 1));
        const int64_t at = static_cast<int64_t>(out ? 0 : id) * a.page_stride;
        const int64_t elements = at + first * kRowBytes;
        const int64_t blocks = at + a.block_offset + first * (D / kMxBlock);
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            // (rows past the end read the last one)
            const int mine = row[p] < keys - 1 - key ? row[p] : keys - 1 - key;
            get_words(words[p], pool[p] + elements + static_cast<uint32_t>(mine * kRowBytes + block[p] * (4 * kWords)));
            bytes[p] = (pool[p] + blocks)[static_cast<uint32_t>(mine * (D / kMxBlock) + block[p])];
        }
    }
    // The rows that have come, unpacked into LDS.  (Where there is no such window it is the last
    // rows again, and nobody reads them.)
    __device__ __forceinline__ void arrive(int buffer) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            const float power = mx_power(bytes[p]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<uint4*>(lds + buffer * kBufferBytes + (place[p] ^ (16 * j))) =
                    mx_unpack8<T, BITS>(words[p] + j * (BITS / 4), power);
            }
        }
    }
    __device__ __forceinline__ void start(int w, int step, int) {
        look(w);
        fetch(w);
        look(w + step);
    }
    __device__ __forceinline__ void next(int w, int step, int, int) {
        fetch(w);
        look(w + step);
    }
    __device__ __forceinline__ void query(const uint16_t* row) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            qf[i] = *reinterpret_cast<const uint4*>(row + 8 * (lane >> 5) + 16 * i);
        }
    }
    template <typename Late>
    __device__ __forceinline__ void scores(floatx16 (&sc)[2], int buffer, Late late) {
        tile_scores<T, D, MxWindow>(sc, qf, lds + buffer * kBufferBytes, lane, late);
    }
};

template <typename T, int D, int BITS>
hipError_t launch(const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    if (plan.few_blocks > 0) {
        hipLaunchKernelGGL((mx_few_kernel<T, D, BITS>), dim3(static_cast<unsigned>(plan.few_blocks)), dim3(kThreads), 0, stream,
                           a, static_cast<int>(plan.splits), plan.tile_splits > 0 ? kMxFewRows : 0x7fffffff);
        const hipError_t status = hipGetLastError();
        if (status != hipSuccess) {
            return status;
        }
    }
    return launch_tiles<T, D, MxWindow<T, D, BITS>>(a, plan, kMxFewRows, true, stream);
}
template <typename T>
hipError_t launch(int bits, const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    if (a.head_dim == 64) {
        return bits == 4 ? launch<T, 64, 4>(a, plan, stream) : launch<T, 64, 8>(a, plan, stream);
    }
    return bits == 4 ? launch<T, 128, 4>(a, plan, stream) : launch<T, 128, 8>(a, plan, stream);
}

}  // namespace

PagedAttnPlan mx_attention_plan(int64_t tokens, int64_t sequences, int64_t max_query_len, int64_t max_kv_len,
                                int64_t max_keys, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                int64_t workspace_bytes) {
    const int64_t group = q_heads / kv_heads;
    PagedAttnPlan p;
    const int64_t longest = max_query_len < tokens ? max_query_len : tokens;
    const int64_t rows = longest * group;
    const int64_t windows = (max_kv_len + kWindow - 1) / kWindow;
    const int64_t rounds = (max_kv_len + kRound - 1) / kRound;
    const bool few = rows <= kMxFewRows;
    int64_t even_splits = 1;  // of tiles, as for 16-bit rows
    if (!few) {
        plan_tiles(p, tokens, sequences, group, rows, windows, kv_heads, head_dim);
        even_splits = p.tile_splits;
        // Tiles of one K-group here are two blocks a CU (heads of 64: three), of two K-groups one
        // (kc_paged_attn.hip's are two of heads of 64).  So sequences of one tile each, whose
        // lengths splits even out, take one group where there are blocks enough for it (heads of
        // 64, 64 sequences of 30 tokens after 3000: 71 us with two groups, 57 with one; 32 of 25
        // after 1000 32 and 23), and so do chunks behind a past at least as long, with splits that
        // fill the chip (1500 tokens of 12 heads of 64 over 4 KV heads after 3000: 53 and 45;
        // heads of 128, 16 over 2: 1200 after 2000 62 and 51, 2500 after 3000 138 and 129).
        // Shorter and fewer ones would lose by the merge what they gain: 3 chunks of 800 after
        // 1000 27 (heads of 128 60) and 36 (64), 1200 of heads of 64 after 2000 31 and 34, whole
        // prompts likewise.  (The longest past may be another sequence's than the longest chunk:
        // a whole prompt of 2000 beside a token after 6000 63 us so and 71 with two groups, beside
        // 8 after up to 8000 59 and 63; 1500 of heads of 64 beside 8 36 and 36.)
        const int64_t tiles = p.slots * kv_heads;
        if (sequences > 1 && rows <= kTileRows) {
            p.tile_groups = tiles * p.tile_splits > 256 ? 1 : p.tile_groups;
        } else if (max_kv_len >= 2 * longest && windows >= 40 && tiles > (head_dim == 64 ? 128 : 96) &&
                   tiles < (head_dim == 64 ? 512 : 342)) {
            p.tile_groups = 1;
            p.tile_splits = head_dim == 64 ? (511 + tiles) / tiles : (tiles <= 256 ? 512 : 1024) / tiles;
        }
    }
    // Beside longer sequences few rows go to their kernel where a tile would take more than 50
    // windows, of the splits that even out lengths: those of the chunks above are no help to a
    // token that is one of them (2000 beside a token after 6000 63 us, in tiles 87; 1500 of heads
    // of 64 beside 8 after up to 8000 36 and 56; but 2000 after 3000 beside 16 after up to 4000
    // 115 and 103).
    int64_t few_splits = 0;
    if (few || (tokens != sequences * longest && windows > 50 * even_splits)) {
        // Where no other sequence is split: up to 5 rounds in one piece (a call of a token over
        // 640 keys 10.4 us so, 13.0 split and merged, replayed 8.8 and 7.6; over 768 replayed
        // 10.0 and 7.6).
        const int64_t tiles = sequences * kv_heads * ((cap(rows, kMxFewRows) + 15) / 16);
        few_splits = p.tile_splits <= 1 && rounds <= 5 ? 1 : cap(2 * ((kFewAtOnce + tiles - 1) / tiles) + 1, cap(rounds, 256));
    }
    const int64_t unit = tokens * q_heads * (head_dim + 2) * 4;
    const int64_t counts = tokens * q_heads * 4;
    const int64_t room = unit > 0 ? (workspace_bytes - counts) / unit : 0;
    // the pieces of few rows are counted in 31 bits
    const int64_t all_tiles = kv_heads * (few ? tokens * group / 16 + sequences : sequences * (kMxFewRows / 16));
    const bool countable = all_tiles * ((max_keys + kRound - 1) / kRound) < (int64_t{1} << 31);
    const int64_t most = room > 1 && countable ? room : 1;
    few_splits = few_splits < most ? few_splits : most;
    p.tile_splits = p.tile_splits < most ? p.tile_splits : most;
    p.splits = few_splits > p.tile_splits ? few_splits : p.tile_splits;
    p.workspace_bytes = p.splits > 1 ? unit * p.splits + counts : 0;
    if (few_splits > 0) {
        // a block a piece, whatever the lengths are: at most a quarter of those at once and
        // one more a tile where the tiles alone are more than fit
        const int64_t pieces = all_tiles + kFewAtOnce / 4 > kFewAtOnce ? all_tiles + kFewAtOnce / 4 : kFewAtOnce;
        p.few_blocks = pieces < all_tiles * p.splits ? pieces : all_tiles * p.splits;
    }
    return p;
}

hipError_t launch_mx_attention(Act act, int bits, const PagedAttnArgs& a, const PagedAttnPlan& plan, hipStream_t stream) {
    return act == Act::kBf16 ? launch<Bf16>(bits, a, plan, stream) : launch<F16>(bits, a, plan, stream);
}

}  // namespace kc
