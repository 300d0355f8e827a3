// Microscaled numbers of a cache: blocks of 32 elements share a power of two.
//
// Elements are e2m1 (BITS 4: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, element 2 i in
// the low half of byte i) or e4m3 (BITS 8: up to 448), a block's byte is 127 + exponent,
// 255 for NaN.  An element times its power of two is a number of bf16, and of fp16 within
// the exponents below, so unpacking is exact: the conversions of gfx950 take the power
// along (full rate: 4.7 cycles a wave and pair, as a product).
#pragma once

#include "kc_device.h"

namespace kc {
namespace {

constexpr int kMxBlock = 32;

// The exponents of blocks that are written.  Below the lowest, elements would fall out of
// the type's numbers (bf16: far enough above its subnormals); above the highest they would
// pass its largest, and saturate instead.
template <typename T, int BITS>
struct MxRange {
    static constexpr int kLowest = -110;
    static constexpr int kHighest = BITS == 4 ? 125 : 119;
};
template <int BITS>
struct MxRange<F16, BITS> {
    static constexpr int kLowest = BITS == 4 ? -23 : -15;
    static constexpr int kHighest = BITS == 4 ? 13 : 7;
};

__device__ __forceinline__ float mx_power(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// ------------------------------------------------------------------ unpacking
// Two elements as T: pair `I` of a word (4 bits: byte I; 8 bits: half I).
template <int I>
__device__ __forceinline__ uint32_t mx_pair(Bf16, std::integral_constant<int, 4>, uint32_t word, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, power, I));
}
template <int I>
__device__ __forceinline__ uint32_t mx_pair(F16, std::integral_constant<int, 4>, uint32_t word, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, power, I));
}
template <int I>
__device__ __forceinline__ uint32_t mx_pair(Bf16, std::integral_constant<int, 8>, uint32_t word, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, power, I != 0));
}
template <int I>
__device__ __forceinline__ uint32_t mx_pair(F16, std::integral_constant<int, 8>, uint32_t word, float power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, power, I != 0));
}
// Eight elements, BITS / 4 words from `words`.
template <typename T, int BITS>
__device__ __forceinline__ uint4 mx_unpack8(const uint32_t* words, float power) {
    constexpr std::integral_constant<int, BITS> bits{};
    if constexpr (BITS == 4) {
        return make_uint4(mx_pair<0>(T{}, bits, words[0], power), mx_pair<1>(T{}, bits, words[0], power),
                          mx_pair<2>(T{}, bits, words[0], power), mx_pair<3>(T{}, bits, words[0], power));
    } else {
        return make_uint4(mx_pair<0>(T{}, bits, words[0], power), mx_pair<1>(T{}, bits, words[0], power),
                          mx_pair<0>(T{}, bits, words[1], power), mx_pair<1>(T{}, bits, words[1], power));
    }
}

// WORDS 32-bit words, aligned to their size.
template <int WORDS>
__device__ __forceinline__ void get_words(uint32_t (&w)[WORDS], const uint8_t* p) {
    static_assert(WORDS == 1 || WORDS == 2 || WORDS == 4 || WORDS == 8, "whole loads");
    if constexpr (WORDS == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (WORDS == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x;
        w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x;
            w[i + 1] = v.y;
            w[i + 2] = v.z;
            w[i + 3] = v.w;
        }
    }
}

// A page's first `bytes` bytes, of the whole wave's page: a load behind them reads nothing and
// gives zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_buffer(const uint8_t* page, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(page), 0, bytes, 0x00027000);
}
template <int WORDS>
__device__ __forceinline__ void get_words(uint32_t (&w)[WORDS], __amdgpu_buffer_rsrc_t page, int offset) {
    static_assert(WORDS == 2 || WORDS == 4 || WORDS == 8, "whole loads");
    if constexpr (WORDS == 2) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(page, offset, 0, 0);
        w[0] = v[0];
        w[1] = v[1];
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(page, offset + 4 * i, 0, 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w[i + k] = v[k];
            }
        }
    }
}

// -------------------------------------------------------------------- packing
// The byte of a block whose largest magnitude has these bits (sign off), 255 if it is no
// number: the least exponent e with magnitude < 7 * 2^e (4 bits), 464 * 2^e (8 bits), so
// that no element is off by more than half a step.
template <typename T, int BITS>
__device__ __forceinline__ uint32_t mx_byte(uint32_t magnitude) {
    constexpr uint32_t kInfinity = std::is_same<T, Bf16>::value ? 0x7f80u : 0x7c00u;
    const uint32_t f = __float_as_uint(T::load(static_cast<uint16_t>(magnitude)));
    int e = static_cast<int>(f >> 23) - 127;
    e += BITS == 4 ? ((f & 0x7fffffu) >= 0x600000u ? -1 : -2) : ((f & 0x7fffffu) >= 0x680000u ? -7 : -8);
    e = e > MxRange<T, BITS>::kLowest ? e : MxRange<T, BITS>::kLowest;
    e = e < MxRange<T, BITS>::kHighest ? e : MxRange<T, BITS>::kHighest;
    return magnitude >= kInfinity ? 255u : static_cast<uint32_t>(e + 127);
}

// Eight numbers as elements of a block with this byte (nearest, ties to even).
template <int BITS>
__device__ __forceinline__ void mx_pack8(const float (&x)[8], uint32_t byte, uint32_t (&words)[BITS / 4]) {
    const float power = __uint_as_float(byte << 23);
    if (byte == 255u) {
#pragma unroll
        for (int i = 0; i < BITS / 4; ++i) {
            words[i] = 0;
        }
        return;
    }
    if constexpr (BITS == 4) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], power, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], power, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], power, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], power, 3);
        words[0] = w;
    } else {
        typedef short shortx2 __attribute__((ext_vector_type(2)));
        const float most = 448.0f * power;  // (past the highest exponent)
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = fminf(fmaxf(x[i], -most), most);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            shortx2 w = {0, 0};
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, y[4 * i], y[4 * i + 1], power, false);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, y[4 * i + 2], y[4 * i + 3], power, true);
            words[i] = __builtin_bit_cast(uint32_t, w);
        }
    }
}

}  // namespace
}  // namespace kc
