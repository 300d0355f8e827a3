// A paged cache of microscaled numbers: rows on the way in and out.
//
// Into it go queries and keys turned by their positions, as kc_rope.hip turns them, and
// values.  A block of 32 dims takes the power of two that its largest magnitude needs and
// rounds its elements to it; both are decided by the row as the 16-bit cache would hold
// it.  The keys' angles, turns and products are formed in 64 bits, since one rounding
// apart a number on the border of two codes lands in the other one, 2^7 (8 bits: 2^4) bf16
// steps away; the queries' are fp32 as there.
//
// Bound by the bytes of the projections' rows: 19999 tokens of 16 and 2 heads of 128 into
// 8 bits, 195 MB, 41 us, 4.7 TB/s; 8 tokens 4.4 us, a launch and the angles.  Four lanes
// share a block, 8 dims each: 16 bytes in, 4 or 8 out, the largest magnitude by two
// exchanges.  A key's lane also loads the 8 dims that its own are paired with.
#include <type_traits>

#include "kc_kernels.h"
#include "kc_mx.h"
#include "kc_rope.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 64;  // of the caches' largest head

// (cos, sin) of position * freq, times amplitude, in 64 bits: the angle less whole
// quarter turns in two parts, Taylor polynomials of the rest (the first terms left out
// are below 2^-58).
__device__ __forceinline__ double2 turn(int32_t position, double freq, float amplitude) {
    constexpr double kTwoOverPi = 0x1.45f306dc9c883p-1;
    constexpr double kHalfPi = 0x1.921fb54442d18p+0;
    constexpr double kHalfPiRest = 0x1.1a62633145c07p-54;
    const double angle = static_cast<double>(position) * freq;
    const double n = rint(angle * kTwoOverPi);
    const double x = fma(-n, kHalfPiRest, fma(-n, kHalfPi, angle));
    const int quarter = static_cast<int>(n - 4.0 * floor(n * 0.25));
    const double z = x * x;
    double s = 1.0 / 355687428096000.0;
    s = fma(z, s, -1.0 / 1307674368000.0);
    s = fma(z, s, 1.0 / 6227020800.0);
    s = fma(z, s, -1.0 / 39916800.0);
    s = fma(z, s, 1.0 / 362880.0);
    s = fma(z, s, -1.0 / 5040.0);
    s = fma(z, s, 1.0 / 120.0);
    s = fma(z, s, -1.0 / 6.0);
    s = fma(x * z, s, x);
    double c = 1.0 / 20922789888000.0;
    c = fma(z, c, -1.0 / 87178291200.0);
    c = fma(z, c, 1.0 / 479001600.0);
    c = fma(z, c, -1.0 / 3628800.0);
    c = fma(z, c, 1.0 / 40320.0);
    c = fma(z, c, -1.0 / 720.0);
    c = fma(z, c, 1.0 / 24.0);
    c = fma(z, c, -0.5);
    c = fma(z, c, 1.0);
    const double cs = (quarter & 1) != 0 ? s : c;
    const double sn = (quarter & 1) != 0 ? c : s;
    return make_double2(((quarter + 1) & 2) != 0 ? -cs * amplitude : cs * amplitude,
                        (quarter & 2) != 0 ? -sn * amplitude : sn * amplitude);
}

// Eight elements from p, in one piece or one by one.
template <bool WIDE>
__device__ __forceinline__ void get8(uint16_t (&x)[8], const uint16_t* p) {
    if constexpr (WIDE) {
        get<8>(x, p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = p[i];
        }
    }
}

// Dims d0 .. d0 + 7 of a key, turned.  cs: (cos, sin) of the token's pairs.
template <typename T, bool WIDE>
__device__ __forceinline__ void turned8(uint16_t (&x)[8], const MxAppendArgs& a, const double2* cs, const uint16_t* row,
                                        int d0) {
    const int pairs = a.rotary_dim / 2;
    get8<WIDE>(x, row + d0);
    if (d0 >= a.rotary_dim) {
        return;
    }
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (d0 + 2 * i < a.rotary_dim) {
                const double2 t = cs[d0 / 2 + i];
                const double x1 = T::load(x[2 * i]);
                const double x2 = T::load(x[2 * i + 1]);
                x[2 * i] = T::store(static_cast<float>(fma(x1, t.x, -(x2 * t.y))));
                x[2 * i + 1] = T::store(static_cast<float>(fma(x1, t.y, x2 * t.x)));
            }
        }
        return;
    }
    if constexpr (WIDE) {  // the eight pairs' other halves side by side
        const bool first = d0 < pairs;
        uint16_t other[8];
        get8<true>(other, row + (first ? d0 + pairs : d0 - pairs));
        const double2* const t = cs + (first ? d0 : d0 - pairs);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double own = T::load(x[i]);
            const double far = T::load(other[i]);
            x[i] = T::store(static_cast<float>(first ? fma(own, t[i].x, -(far * t[i].y)) : fma(far, t[i].y, own * t[i].x)));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            if (d < a.rotary_dim) {
                const bool first = d < pairs;
                const double own = T::load(x[i]);
                const double far = T::load(row[first ? d + pairs : d - pairs]);
                const double2 t = cs[first ? d : d - pairs];
                x[i] = T::store(static_cast<float>(first ? fma(own, t.x, -(far * t.y)) : fma(far, t.y, own * t.x)));
            }
        }
    }
}

template <typename T, int BITS, bool WIDE, int TOKENS>
__global__ __launch_bounds__(kThreads) void append_kernel(MxAppendArgs a) {
    __shared__ double2 s_turn[TOKENS][kMaxPairs];
    __shared__ float2 s_near[TOKENS][kMaxPairs];
    const int pairs = a.rotary_dim / 2;
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * TOKENS;
    for (int i = threadIdx.x; i < TOKENS * pairs; i += kThreads) {
        const int64_t token = token0 + i / pairs;
        if (token < a.tokens) {
            const double2 t = turn(a.positions[token], a.inv_freq[i % pairs], a.amplitude);
            s_turn[i / pairs][i % pairs] = t;
            s_near[i / pairs][i % pairs] = make_float2(static_cast<float>(t.x), static_cast<float>(t.y));
        }
    }
    __syncthreads();
    constexpr int kLanes = kThreads / TOKENS;  // of a token, whole waves
    const int mine = static_cast<int>(threadIdx.x) / kLanes;
    const int64_t token = token0 + mine;
    if (token >= a.tokens) {
        return;
    }
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= (a.num_pages << a.page_shift)) {
        return;  // padding
    }
    const int64_t page = (slot >> a.page_shift) * a.page_stride;
    const int offset = static_cast<int>(slot & ((int64_t{1} << a.page_shift) - 1));
    const int chunks = a.head_dim / 8;
    // keys and values first: their groups of four lanes stay together
    const int cached = 2 * a.kv_heads * chunks;
    constexpr int kPiece = WIDE ? 8 : 1;
    const int units = a.head_dim / (2 * kPiece);
    const int total = cached + a.q_heads * units;
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    for (int i = lane; i < total; i += kLanes) {
        if (i >= cached) {
            const int head = (i - cached) / units;
            unit<T, kPiece>(a, s_near[mine], (i - cached) % units, true, a.q + token * a.q_stride + head * a.head_dim,
                            a.q_out + token * a.out_stride + head * a.head_dim);
            continue;
        }
        uint16_t x[8];
        const bool value = i >= cached / 2;
        const int head = (value ? i - cached / 2 : i) / chunks;
        const int d0 = i % chunks * 8;
        if (value) {
            get8<WIDE>(x, a.v + token * a.v_stride + head * a.head_dim + d0);
        } else {
            turned8<T, WIDE>(x, a, s_turn[mine], a.k + token * a.k_stride + head * a.head_dim, d0);
        }
        uint32_t most = 0;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t m = x[j] & 0x7fffu;
            most = m > most ? m : most;
            f[j] = T::load(x[j]);
        }
        uint32_t near = __shfl_xor(most, 1, 4);
        most = near > most ? near : most;
        near = __shfl_xor(most, 2, 4);
        most = near > most ? near : most;
        const uint32_t byte = mx_byte<T, BITS>(most);
        uint32_t words[BITS / 4];
        mx_pack8<BITS>(f, byte, words);
        uint8_t* const pool = (value ? a.v_pages : a.k_pages) + page;
        const int64_t row = static_cast<int64_t>(head << a.page_shift) + offset;  // (kv_heads * page_size fits)
        uint8_t* const at = pool + (row * a.head_dim + d0) * BITS / 8;
        if constexpr (BITS == 4) {
            *reinterpret_cast<uint32_t*>(at) = words[0];
        } else {
            *reinterpret_cast<uint2*>(at) = make_uint2(words[0], words[1]);
        }
        if (d0 % kMxBlock == 0) {
            pool[a.block_offset + (row * a.head_dim + d0) / kMxBlock] = static_cast<uint8_t>(byte);
        }
    }
}

template <typename T, int BITS, bool WIDE>
hipError_t launch(const MxAppendArgs& a, hipStream_t stream) {
    // few tokens: one a block, to spread them over the chip, as in kc_rope.hip
    if (a.tokens < 2048) {
        hipLaunchKernelGGL((append_kernel<T, BITS, WIDE, 1>), dim3(static_cast<unsigned>(a.tokens)), dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((append_kernel<T, BITS, WIDE, 4>), dim3(static_cast<unsigned>((a.tokens + 3) / 4)), dim3(kThreads), 0,
                           stream, a);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------- reading back
// A lane unpacks 8 dims at a time: 4 or 8 bytes in, 16 out, so that a wave writes whole
// lines; UNITS of them, whose slots and then whose bytes are asked for together.
template <typename T, int BITS, int UNITS>
__device__ __forceinline__ void read_units(const MxReadArgs& a, int64_t first) {
    const int chunks = a.head_dim / 8;
    const int row_units = 2 * a.kv_heads * chunks;  // of a token
    const int64_t token0 = first / row_units;
    const int rest = static_cast<int>(first - token0 * row_units);
    const uint8_t* page[UNITS];
    int64_t row[UNITS], token[UNITS];
    int unit[UNITS];
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const unsigned i = static_cast<unsigned>(rest + n * kThreads) + threadIdx.x;
        const unsigned ahead = i / static_cast<unsigned>(row_units);
        unit[n] = static_cast<int>(i - ahead * row_units);
        token[n] = token0 + ahead;
        row[n] = token[n] < a.tokens ? a.slots[token[n]] : -1;
    }
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const int64_t slot = row[n];
        const bool value = unit[n] >= row_units / 2;
        page[n] = nullptr;  // padding, or behind the last row
        if (slot >= 0 && slot < (a.num_pages << a.page_shift)) {
            const int head = (value ? unit[n] - row_units / 2 : unit[n]) / chunks;
            page[n] = (value ? a.v_pages : a.k_pages) + (slot >> a.page_shift) * a.page_stride;
            row[n] = static_cast<int64_t>(head << a.page_shift) + (slot & ((int64_t{1} << a.page_shift) - 1));
        }
    }
    uint32_t words[UNITS][BITS / 4];
    uint32_t byte[UNITS];
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        byte[n] = 0;
        if (page[n] != nullptr) {
            const int64_t at = row[n] * a.head_dim + unit[n] % chunks * 8;
            get_words(words[n], page[n] + at * BITS / 8);
            byte[n] = page[n][a.block_offset + at / kMxBlock];
        }
    }
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        if (page[n] != nullptr) {
            const bool value = unit[n] >= row_units / 2;
            uint16_t* const out = value ? a.v_out + token[n] * a.v_stride : a.k_out + token[n] * a.k_stride;
            *reinterpret_cast<uint4*>(out + (value ? unit[n] - row_units / 2 : unit[n]) * 8) =
                mx_unpack8<T, BITS>(words[n], mx_power(byte[n]));
        }
    }
}

template <typename T, int BITS, int UNITS>
__global__ __launch_bounds__(kThreads) void read_kernel(MxReadArgs a, int64_t units) {
    constexpr int kBlockUnits = UNITS * kThreads;
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * kBlockUnits; first < units;
         first += static_cast<int64_t>(gridDim.x) * kBlockUnits) {
        read_units<T, BITS, UNITS>(a, first);
    }
}

template <typename T, int BITS, int UNITS>
hipError_t launch(const MxReadArgs& a, int64_t units, hipStream_t stream) {
    constexpr int64_t kMostBlocks = int64_t{1} << 20;
    const int64_t blocks = (units + UNITS * kThreads - 1) / (UNITS * kThreads);
    hipLaunchKernelGGL((read_kernel<T, BITS, UNITS>), dim3(static_cast<unsigned>(blocks < kMostBlocks ? blocks : kMostBlocks)),
                       dim3(kThreads), 0, stream, a, units);
    return hipGetLastError();
}

template <typename T, int BITS>
hipError_t launch(const MxReadArgs& a, hipStream_t stream) {
    const int64_t units = a.tokens * 2 * a.kv_heads * (a.head_dim / 8);
    // few rows: a unit a lane, to spread them (the kernel alone, 2 heads of 128 in 8 bits: 2000
    // rows 3.4 us by one and 4.8 by four, 8192 5.8 and 6.2, 32000 13.7 and 13.1, 120000 51 and
    // 41 -- 187 MB, 4.6 TB/s)
    return units <= int64_t{1} << 20 ? launch<T, BITS, 1>(a, units, stream) : launch<T, BITS, 4>(a, units, stream);
}

}  // namespace

hipError_t launch_mx_append(Act act, const MxAppendArgs& a, hipStream_t stream) {
    const auto wide = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    // 16-byte pieces where every row, and every pair's two places, begin on one
    const bool pieces = wide(a.q) && wide(a.q_out) && wide(a.k) && wide(a.v) &&
                        (a.q_stride | a.out_stride | a.k_stride | a.v_stride) % 8 == 0 && a.rotary_dim % 16 == 0;
    if (act == Act::kBf16) {
        if (a.bits == 4) {
            return pieces ? launch<Bf16, 4, true>(a, stream) : launch<Bf16, 4, false>(a, stream);
        }
        return pieces ? launch<Bf16, 8, true>(a, stream) : launch<Bf16, 8, false>(a, stream);
    }
    if (a.bits == 4) {
        return pieces ? launch<F16, 4, true>(a, stream) : launch<F16, 4, false>(a, stream);
    }
    return pieces ? launch<F16, 8, true>(a, stream) : launch<F16, 8, false>(a, stream);
}

hipError_t launch_mx_read(Act act, const MxReadArgs& a, hipStream_t stream) {
    if (act == Act::kBf16) {
        return a.bits == 4 ? launch<Bf16, 4>(a, stream) : launch<Bf16, 8>(a, stream);
    }
    return a.bits == 4 ? launch<F16, 4>(a, stream) : launch<F16, 8>(a, stream);
}

}  // namespace kc
