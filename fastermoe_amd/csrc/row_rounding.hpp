// Rounding of a row's elements to 8-bit integers under the row's scale (device code):
//
//   s = max(fl32(max|x| / 127), 2^-126)        q = x / s to the nearest integer, ties to even, of the exact quotient
//
// The exact quotient's rounding, without a division per element: t = x * (1 / s) + 1.5 2^23, one fused multiply-add, has the integer next to x * (1 / s) in its low
// bits; that product is off by less than 2^-16, so q = t - 1.5 2^23 is the right integer or the one beside it, and r = x - q s, another multiply-add, is
// exact (a multiple of ulp(s) or of x's, below 2 s).  Only where |r| >= s / 2, once in some thousand elements, q may be off, or a tie: such pieces are looked at again.
#pragma once
#include "common.hpp"
#include "lane_elems.hpp"

namespace fmoe {
namespace {

constexpr int kLaneElems = 8;

// Eight elements as they lie in memory
template <typename T> struct Eight {
    static constexpr int kVecs = (int)sizeof(T) / 2;
    u32x4 v[kVecs];
    // the first n of them at p, zeros after those
    __device__ __forceinline__ void load(const T *p, int n) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[i] = load_vec<false>(p + i * Vec<T>::N, n - i * Vec<T>::N, false);
    }
    __device__ __forceinline__ void floats(float (&f)[kLaneElems]) const {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            float g[8];
            Vec<T>::unpack(v[i], g);
#pragma unroll
            for (int j = 0; j < Vec<T>::N; ++j) f[i * Vec<T>::N + j] = g[j];
        }
    }
};
// The magnitudes' bits are in the order of the magnitudes, infinity and then NaN above them: the largest of a lane's elements, as the bits of its type (16-bit types: in
// either half).
template <typename T> __device__ __forceinline__ uint32_t larger(uint32_t most, const Eight<T> &e) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < Eight<T>::kVecs; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
                most = max(most, e.v[i][j] & 0x7fffffffu);
            } else {
                const u16x2 a = __builtin_bit_cast(u16x2, most), b = __builtin_bit_cast(u16x2, e.v[i][j] & 0x7fff7fffu);
                most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
            }
        }
    return most;
}
// float32 bits of the largest magnitude
template <typename T> __device__ __forceinline__ uint32_t magnitude_bits(uint32_t most) {
    if constexpr (sizeof(T) == 4) {
        return most;
    } else {
        const uint16_t top = (uint16_t)max(most & 0xffffu, most >> 16);
        return __float_as_uint((float)__builtin_bit_cast(T, top));
    }
}

constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126
constexpr float kMagic = 12582912.f;   // 1.5 2^23
// eight integers, a byte each
__device__ __forceinline__ uint2 round_all(const float (&x)[kLaneElems], float inv, float s, float half) {
    float t[kLaneElems], off = 0.f;
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) {
        t[j] = fmaf(x[j], inv, kMagic);
        off = fmaxf(off, fabsf(fmaf(kMagic - t[j], s, x[j])));
    }
    if (off >= half) {
#pragma unroll
        for (int j = 0; j < kLaneElems; ++j) {
            const float q = t[j] - kMagic, r = fmaf(-q, s, x[j]), a = fabsf(r);
            if (a > half || (a == half && ((int)q & 1))) t[j] += r > 0.f ? 1.f : -1.f;
        }
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * h + 1]), __float_as_uint(t[4 * h]), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * h + 3]), __float_as_uint(t[4 * h + 2]), 0x04000c0cu);
        w[h] = lo | hi;
    }
    return make_uint2(w[0], w[1]);
}

// A row's scale, of the largest of its magnitudes' bits.  With an infinity or a NaN in the row: NaN, and zeros for integers, so that whatever is made of it is NaN.
struct RowScale {
    bool finite;
    float s, inv, half;
    __device__ __forceinline__ explicit RowScale(uint32_t most) {
        finite = most < 0x7f800000u;
        s = fmaxf(__uint_as_float(finite ? most : 0u) / 127.f, kLeastScale);
        inv = 1.f / s;
        half = 0.5f * s;
    }
    __device__ __forceinline__ float shown() const { return finite ? s : __uint_as_float(0x7fc00000u); }
    template <typename T> __device__ __forceinline__ uint2 round(const Eight<T> &piece) const {
        float f[kLaneElems];
        piece.floats(f);
        const uint2 w = round_all(f, inv, s, half);
        return finite ? w : make_uint2(0, 0);
    }
};

}  // namespace
}  // namespace fmoe
