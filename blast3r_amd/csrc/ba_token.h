// Loads, stores and 8-bit codes shared by the token operators (rotary positions, the key/value cache).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ba_hip.h"

namespace ba {

// what `dtype` says of a tensor of the token operators
enum { BA_F32 = 0, BA_F16 = 1, BA_BF16 = 2 };
// what `bits` says of a cache
enum { BA_FP8 = 0, BA_INT8 = 1 };

// V consecutive elements as floats, in loads of 16 bytes or what they are if less, and aligned to that
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (sizeof(T) * V > 16) {                     // a longer vector type would have the compiler take a wider alignment for granted
        constexpr int W = 16 / sizeof(T);
        static_assert(V % W == 0, "whole loads");
#pragma unroll
        for (int j = 0; j < V; j += W) {
            float x[W];
            load_vec<T, W>(p + j, x);
#pragma unroll
            for (int i = 0; i < W; ++i) v[j + i] = x[i];
        }
    } else if constexpr (V == 1) {
        v[0] = (float)p[0];
    } else if constexpr (V == 2) {                          // used where addresses are not aligned
        v[0] = (float)p[0];
        v[1] = (float)p[1];
    } else {
        static_assert(sizeof(vec) <= 16, "callers' addresses are aligned to 16 bytes");
        const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)x[i];
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    if constexpr (V == 1) {
        p[0] = (T)v[0];
    } else if constexpr (V == 2) {
        p[0] = (T)v[0];
        p[1] = (T)v[1];
    } else {
        static_assert(sizeof(vec) <= 16, "callers' addresses are aligned to 16 bytes");
        vec x;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (T)v[i];
        *reinterpret_cast<vec*>(p) = x;
    }
}

}  // namespace ba
