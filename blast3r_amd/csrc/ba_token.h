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

// The block of a list's entry, below 0 where it has none.  A block that other lists hold too, and that must therefore not be
// written for this one, may be marked (ba_kv_pool_grow): it is read like any other, while rows appended there are left out, as
// those of a number that is no block's.
#define KV_KEPT (1 << 30)
__device__ __forceinline__ int32_t kv_block(int32_t entry) { return entry & ~KV_KEPT; }

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

// Ragged calls whose sequences may each have all rows, as far as the host knows, can be too large for a grid of so many
// places for every one of them.  Then places are laid out by the offsets: sequence s has those from
// floor(offsets[s] * mul / div) + s * more on, up to the next one's, which is at least its rows * mul / div, rounded up
// (more = 1).  The sequence of place `w`, and which of its places that is (below 0: none of any sequence).
__device__ __forceinline__ int seq_of_place(const int32_t* offsets, int n_seqs, int64_t n_rows, int mul, int div, int more, unsigned w, int& place) {
    auto first = [&](int s) {
        const int64_t at = offsets[s];
        return (at < 0 ? 0 : at > n_rows ? n_rows : at) * mul / div + (int64_t)s * more;
    };
    int s = 0, e = n_seqs;                                   // the last s with first(s) <= w
    while (e - s > 1) {
        const int c = (s + e) >> 1;
        if (first(c) <= (int64_t)w) s = c; else e = c;
    }
    place = (int)((int64_t)w - first(s));
    return s;
}

}  // namespace ba
