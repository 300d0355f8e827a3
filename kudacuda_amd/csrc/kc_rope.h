// A head's row turned by its position, piece by piece (kc_rope.hip tells the layouts).
#pragma once

#include "kc_device.h"

namespace kc {
namespace {

template <typename T>
__device__ __forceinline__ void turn_pair(float2 cs, uint16_t& a, uint16_t& b) {
    const float x1 = T::load(a);
    const float x2 = T::load(b);
    a = T::store(fmaf(x1, cs.x, -(x2 * cs.y)));
    b = T::store(fmaf(x1, cs.y, x2 * cs.x));
}

// V elements at p: one 16-byte piece or one element.
template <int V>
__device__ __forceinline__ void get(uint16_t (&x)[V], const uint16_t* p) {
    if constexpr (V == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        __builtin_memcpy(x, &v, 16);
    } else {
        x[0] = p[0];
    }
}
template <int V>
__device__ __forceinline__ void put(const uint16_t (&x)[V], uint16_t* p) {
    if constexpr (V == 8) {
        uint4 v;
        __builtin_memcpy(&v, x, 16);
        *reinterpret_cast<uint4*>(p) = v;
    } else {
        p[0] = x[0];
    }
}

// Unit u of a head: two pieces of V elements, V pairs of the rotary part or 2 V
// elements behind it.
template <typename T, int V, typename Args>
__device__ __forceinline__ void unit(const Args& a, const float2* cs, int u, bool rotate, const uint16_t* src,
                                     uint16_t* dst) {
    const int pairs = a.rotary_dim / 2;
    uint16_t x[V], y[V];
    const bool turned = rotate && u * V < pairs;
    const int at = turned && !a.interleaved ? u * V : 2 * u * V;
    const int other = at + (turned && !a.interleaved ? pairs : V);
    get<V>(x, src + at);
    get<V>(y, src + other);
    if (turned) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!a.interleaved) {
                turn_pair<T>(cs[u * V + i], x[i], y[i]);
            } else if constexpr (V == 1) {
                turn_pair<T>(cs[u], x[0], y[0]);
            } else {
                uint16_t& lo = 2 * i < V ? x[2 * i % V] : y[2 * i % V];
                uint16_t& hi = 2 * i < V ? x[2 * i % V + 1] : y[2 * i % V + 1];
                turn_pair<T>(cs[u * V + i], lo, hi);
            }
        }
    }
    put<V>(x, dst + at);
    put<V>(y, dst + other);
}

}  // namespace
}  // namespace kc
