// 16-byte loads of 16-bit elements from wherever they begin (device code).
#pragma once
#include "vec16.hpp"

namespace fmoe {
namespace {

template <typename T> __device__ __forceinline__ u32x4 load_unaligned(const T *p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
// the same of elements that begin on a dword
template <typename T> __device__ __forceinline__ u32x4 load_dwords(const T *p) {
    typedef uint32_t __attribute__((ext_vector_type(4), aligned(4))) dwords;
    return *(const dwords *)p;
}
// The last n of eight 16-bit elements, in the first one's place, zeros after them (n <= 0: zeros; 8 <= n: all)
__device__ __forceinline__ u32x4 moved_down(const u32x4 &v, int n) {
    const int s = 8 - max(0, min(n, 8));   // elements to move down
    const u32x4 a = s & 4 ? u32x4{v[2], v[3], 0u, 0u} : v;
    const u32x4 b = s & 2 ? u32x4{a[1], a[2], a[3], 0u} : a;
    const u32x4 c = s & 1 ? u32x4{__builtin_amdgcn_alignbit(b[1], b[0], 16), __builtin_amdgcn_alignbit(b[2], b[1], 16),
                                  __builtin_amdgcn_alignbit(b[3], b[2], 16), b[3] >> 16} : b;
    return n > 0 ? c : u32x4{0u, 0u, 0u, 0u};
}
// The first n of the eight elements at p, zeros after them.  8 <= n: all of them.  0 < n < 8: with `back`, the eight
// elements that end with them (the caller knows that as many precede them in their row), moved down; else one by one.
// n <= 0: nothing is read at p, but with `back` eight elements at `safe`.
template <typename T> __device__ __forceinline__ u32x4 load_part(const T *p, const T *safe, int n, bool back) {
    if (back) return moved_down(load_unaligned(n > 0 ? p - (8 - min(n, 8)) : safe), n);
    if (n >= 8) return load_unaligned(p);
    alignas(16) uint16_t e[8] = {};
    const uint16_t *src = (const uint16_t *)p;
#pragma unroll
    for (int j = 0; j < 7; ++j)
        if (j < n) e[j] = src[j];
    return __builtin_bit_cast(u32x4, e);
}

}  // namespace
}  // namespace fmoe
