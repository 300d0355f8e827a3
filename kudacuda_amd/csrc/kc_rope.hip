// Rotary positions of many rows, alone or on the way into a paged KV cache.
//
// The first rotary_dim dims of a head are pairs (x1, x2): dims i and
// i + rotary_dim / 2 (half layout) or 2 i and 2 i + 1 (interleaved).  Pair i of a
// token at position p turns by a = p * inv_freq[i]:
//     y1 = c (x1 cos a - x2 sin a),  y2 = c (x1 sin a + x2 cos a)
// with c the amplitude that scaled frequencies bring along.  The angle is reduced
// to a quarter turn in 64 bits (in 32 the product alone is off by 0.06 rad at a
// million tokens), sine and cosine of the rest are fp32 polynomials, the products
// are fp32 and each result is rounded once.
//
// Bound by the bytes of the rows.  A block owns one or four tokens: its threads
// form the tokens' cosines and sines once in LDS, then a wave takes a token's
// heads -- queries, keys, values one after the other -- 2 x 16 bytes a lane.  32768
// tokens of 16 and 2 heads of 128 (336 MB): 65 us, 5.2 TB/s; with single elements 100.
#include "kc_kernels.h"
#include "kc_rope.h"

namespace kc {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = kRopeMaxDim / 2;

// (cos, sin) of position * freq, times amplitude.
__device__ __forceinline__ float2 turn(int32_t position, double freq, float amplitude) {
    constexpr double kTwoOverPi = 0x1.45f306dc9c883p-1;
    constexpr float kHalfPi = 0x1.921fb6p+0f;
    const double t = static_cast<double>(position) * freq * kTwoOverPi;  // quarter turns
    const double n = rint(t);
    const float x = static_cast<float>(t - n) * kHalfPi;  // |x| <= pi / 4
    const int quarter = static_cast<int>(n - 4.0 * floor(n * 0.25));
    const float z = x * x;
    // Taylor polynomials: the first term left out is below 2^-29 (sin) and 2^-31 (cos)
    float s = fmaf(z, 0x1.71de3ap-19f, -0x1.a01a02p-13f);
    s = fmaf(z, s, 0x1.111112p-7f);
    s = fmaf(z, s, -0x1.555556p-3f);
    s = fmaf(x * z, s, x);
    float c = fmaf(z, -0x1.27e4fcp-22f, 0x1.a01a02p-16f);
    c = fmaf(z, c, -0x1.6c16c2p-10f);
    c = fmaf(z, c, 0x1.555556p-5f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    const float cs = (quarter & 1) != 0 ? s : c;
    const float sn = (quarter & 1) != 0 ? c : s;
    return make_float2(((quarter + 1) & 2) != 0 ? -cs * amplitude : cs * amplitude,
                       (quarter & 2) != 0 ? -sn * amplitude : sn * amplitude);
}

template <typename T, int V, int TOKENS>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
    __shared__ float2 s_cs[TOKENS][kMaxPairs];
    const int pairs = a.rotary_dim / 2;
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * TOKENS;
    for (int i = threadIdx.x; i < TOKENS * pairs; i += kThreads) {
        const int64_t token = token0 + i / pairs;
        if (token < a.tokens) {
            s_cs[i / pairs][i % pairs] = turn(a.positions[token], a.inv_freq[i % pairs], a.amplitude);
        }
    }
    __syncthreads();
    constexpr int kLanes = kThreads / TOKENS;  // of a token
    const int mine = static_cast<int>(threadIdx.x) / kLanes;
    const int64_t token = token0 + mine;
    if (token >= a.tokens) {
        return;
    }
    int64_t row = 0;  // element offset of the token's row in the pools
    if (a.slots != nullptr) {
        const int64_t slot = a.slots[token];
        if (slot < 0 || slot >= (a.num_pages << a.page_shift)) {
            return;  // padding
        }
        row = (slot >> a.page_shift) * a.page_stride + (slot & ((int64_t{1} << a.page_shift) - 1)) * a.token_stride;
    }
    const int units = a.head_dim / (2 * V);
    const int total = (a.q_heads + 2 * a.kv_heads) * units;
    for (int i = static_cast<int>(threadIdx.x) % kLanes; i < total; i += kLanes) {
        const int head = i / units;
        const int u = i % units;
        if (head < a.q_heads) {
            unit<T, V>(a, s_cs[mine], u, true, a.q + token * a.q_stride + head * a.head_dim,
                       a.q_out + token * a.out_stride + head * a.head_dim);
        } else if (head < a.q_heads + a.kv_heads) {
            const int h = head - a.q_heads;
            unit<T, V>(a, s_cs[mine], u, true, a.k + token * a.k_stride + h * a.head_dim,
                       a.k_pages + row + h * a.head_stride);
        } else {
            const int h = head - a.q_heads - a.kv_heads;
            unit<T, V>(a, s_cs[mine], u, false, a.v + token * a.v_stride + h * a.head_dim,
                       a.v_pages + row + h * a.head_stride);
        }
    }
}

template <typename T, int V>
hipError_t launch(const RopeArgs& a, hipStream_t stream) {
    // few tokens: one a block, to spread them over the chip (the kernel alone, 16 and 2
    // heads of 128: 8 tokens 4.0 us one a block and 5.4 four, 2000 7.0 and 8.0, 4000 11.6
    // and 11.0, 32768 78 and 65)
    if (a.tokens < 2048) {
        hipLaunchKernelGGL((rope_kernel<T, V, 1>), dim3(static_cast<unsigned>(a.tokens)), dim3(kThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL((rope_kernel<T, V, 4>), dim3(static_cast<unsigned>((a.tokens + 3) / 4)), dim3(kThreads), 0,
                           stream, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(Act act, const RopeArgs& a, hipStream_t stream) {
    const auto wide = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const int64_t strides = a.q_stride | a.out_stride | a.k_stride | a.v_stride | a.page_stride | a.head_stride | a.token_stride;
    // 16-byte pieces where every row, and every pair's two places, begin on one
    const bool pieces = wide(a.q) && wide(a.q_out) && wide(a.k) && wide(a.v) && wide(a.k_pages) && wide(a.v_pages) &&
                        strides % 8 == 0 && a.head_dim % 16 == 0 && a.rotary_dim % 16 == 0;
    if (act == Act::kBf16) {
        return pieces ? launch<Bf16, 8>(a, stream) : launch<Bf16, 1>(a, stream);
    }
    return pieces ? launch<F16, 8>(a, stream) : launch<F16, 1>(a, stream);
}

}  // namespace kc
