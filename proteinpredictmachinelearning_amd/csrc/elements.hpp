// Element types of the operators that take more than binary32: all arithmetic is binary32, one rounding on the way out.
#pragma once
#include "common.hpp"

namespace ppmlhip {
namespace {

template <class T> __device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }
template <class T> __device__ __forceinline__ T from_f32(float x) { return static_cast<T>(x); }

// V consecutive elements, as one access of V * sizeof(T) bytes
template <class T, int V> struct Elements { typedef T Raw __attribute__((ext_vector_type(V))); };
template <class T> struct Elements<T, 1> { typedef T Raw; };

template <class T, int V>
__device__ __forceinline__ void load_f32(const T* from, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = to_f32(*from);
    } else {
        const auto raw = *reinterpret_cast<const typename Elements<T, V>::Raw*>(from);
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = to_f32(static_cast<T>(raw[v]));
    }
}
template <class T, int V>
__device__ __forceinline__ void store_f32(T* to, const float (&x)[V]) {
    if constexpr (V == 1) {
        *to = from_f32<T>(x[0]);
    } else {
        typename Elements<T, V>::Raw raw;
#pragma unroll
        for (int v = 0; v < V; ++v) raw[v] = from_f32<T>(x[v]);
        *reinterpret_cast<typename Elements<T, V>::Raw*>(to) = raw;
    }
}

}  // namespace
}  // namespace ppmlhip
