// The few adjacent elements of a row that a lane takes at once, wherever the row begins (device code).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "vec16.hpp"

namespace fmoe {

// N elements (4 or 8) at p; WHOLE: or none.  Otherwise n may be less than N: what is behind them (`inside`: the memory there still is the
// tensor's) is read and made zeros.
template <bool WHOLE, int N, typename T> __device__ __forceinline__ void load_elems(const T *p, int n, bool inside, T (&e)[N]) {
    if (WHOLE ? n > 0 : n >= N || (n > 0 && inside)) {
        __builtin_memcpy(e, p, sizeof(e));
        if (!WHOLE) {
#pragma unroll
            for (int j = 1; j < N; ++j) e[j] = j < n ? e[j] : T{};
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) e[j] = !WHOLE && j < n ? p[j] : T{};
    }
}

template <int WORDS> struct Words { uint32_t w[WORDS]; };

// The first n of them, or, WHOLE, all or none: four, two and one at a time, put together by masks (the compiler keeps arrays of elements that are
// chosen by n in LDS: rows of 1302 float16, 1554 of them, then took 17 us instead of 4.5).
template <bool WHOLE, int N, typename T> __device__ __forceinline__ void store_elems(T *p, int n, const T (&e)[N]) {
    static_assert(N == 4 || N == 8, "four or eight elements");
    if (WHOLE ? n > 0 : n >= N) {
        __builtin_memcpy(p, e, sizeof(e));
    } else if (!WHOLE && n > 0) {
        constexpr int kHalf = (int)sizeof(T);          // words of four elements
        Words<N / 4 * kHalf> all;
        __builtin_memcpy(&all, e, sizeof(e));
        Words<kHalf> four;
        if constexpr (N == 8) {
            const uint32_t past4 = n & 4 ? ~0u : 0u;
            if (n & 4) __builtin_memcpy(p, &all, 4 * sizeof(T));
#pragma unroll
            for (int j = 0; j < kHalf; ++j) four.w[j] = (all.w[kHalf + j] & past4) | (all.w[j] & ~past4);
            p += n & 4;
        } else {
            four = all;
        }
        const uint32_t past2 = n & 2 ? ~0u : 0u;
        if (n & 2) __builtin_memcpy(p, &four, 2 * sizeof(T));
        const uint32_t one = ((kHalf == 1 ? four.w[0] >> 16 : four.w[kHalf / 2]) & past2) | (four.w[0] & ~past2);
        if (n & 1) __builtin_memcpy(p + (n & 2), &one, sizeof(T));
    }
}

typedef uint32_t AnyVec __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes wherever they begin
// The same for 16 bytes as they lie in memory (elements of a 16-bit type in a register each would take twice the registers); ONCE: not to
// be kept in the caches
template <bool ONCE, typename T> __device__ __forceinline__ u32x4 load_vec(const T *p, int n, bool inside) {
    constexpr int N = Vec<T>::N;
    u32x4 v = {0, 0, 0, 0};
    if (n >= N || (n > 0 && inside)) {
        v = ONCE ? __builtin_nontemporal_load((const AnyVec *)p) : *(const AnyVec *)p;
        if (n < N) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int left = n - j * N / 4;
                v[j] = left <= 0 ? 0 : sizeof(T) == 2 && left == 1 ? v[j] & 0xffffu : v[j];
            }
        }
    } else if (n > 0) {
        T e[N];
#pragma unroll
        for (int j = 0; j < N; ++j) e[j] = j < n ? p[j] : T{};
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}
template <bool ONCE, typename T> __device__ __forceinline__ void store_vec(T *p, int n, const u32x4 &v) {
    if (ONCE && n >= Vec<T>::N) {
        __builtin_nontemporal_store(v, (AnyVec *)p);
        return;
    }
    T e[Vec<T>::N];
    __builtin_memcpy(e, &v, 16);
    store_elems<false>(p, n, e);
}

}  // namespace fmoe
