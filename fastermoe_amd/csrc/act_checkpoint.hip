// The experts' rows kept in 8 bits for the backward pass (gfx950).
//
// A block of 32 elements along a row (fewer at its end) is held as e4m3 numbers under one power of two, the smallest 2^b
// (b >= -126) with max|x| <= 448 2^b over the block's finite elements:  q = e4m3(x 2^-b), to nearest, ties to even; the scale is the
// byte b + 127.  Dividing by a power of two is exact, so the numbers are off by their own rounding alone: 2^-4 of themselves, or, small
// against the block, 2^-10 2^b.  What rounds to more than the rows' type holds is held as the largest that it does (240 2^b in the one
// block that can); infinities and NaN are held as NaN, so that a forward that overflowed still shows in the gradients.  A ReLU's argument of at most 2^-10 2^b is
// held as 0, where its slope is 0: positive elements that are 2 to 5 10^5 times smaller than their block's largest get no gradient.
//
//   forward   y = act(x), q, b          backward  x~ = q 2^b   mid = act(x~)   grad_x = grad act'(x~)
//
// A lane takes eight elements of a row, four lanes a block: one 16-byte load of a 16-bit type, a maximum over the lanes of a quad, eight
// bytes out.  Rows of whole blocks are one run of such pieces (FLAT); others, of any length, are cut into pieces row by row, and a row's last one is
// stored in parts.  Bound by memory: 32768 rows of 14336 in bfloat16 with GELU forward 385 us, without y 231, backward 545 (6.1 to 6.2 TB/s;
// a large copy on the same card 5.0); 32768 of 4096 in float32 207 and 298 (5.9); 32768 of 1302 in bfloat16, whose rows begin anywhere, 44 and 58 (4.8
// and 5.2).  One piece to a lane: two or four in flight, on a half or a quarter of the workgroups, took 383 and 572 or 413 and 586 us of the first,
// and 4.8 and 7.0 of the 4.5 and 5.6 that 1554 rows of 1302 take.  A block to a thread, one element after the other, took 21600 for the first.
#include "common.hpp"
#include "gelu_terms.hpp"
#include "grouped_gemm.hpp"
#include "lane_elems.hpp"
#include "wave_piece.hpp"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kScaleElems = 32, kLaneElems = 8, kLanes = kScaleElems / kLaneElems;   // lanes that share a scale

// (GELU by gelu_terms in float32 too: off by up to 5.3 2^-24 |x|, where the library's error function is by 1.8.  That one takes 14.4 us instead of 13.3 of the forward of
// 8192 x 1024, 6.6 instead of 5.9 of 2048 x 1024 and nothing of 32768 x 4096, and in the backward, whose argument is off by 2^-4, 21.0 instead of 20.3 and 309 instead of 298.)
template <int ACT> __device__ __forceinline__ float act_value(float x) {
    if (ACT == FMOE_ACT_RELU) return x < 0.f ? 0.f : x;   // (NaN stays)
    if (ACT == FMOE_ACT_GELU) return x * gemm::gelu_terms(x).cdf;
    return x;
}
// act(x) and act'(x)
template <int ACT> __device__ __forceinline__ void act_both(float x, float &value, float &slope) {
    if (ACT == FMOE_ACT_RELU) {
        value = x < 0.f ? 0.f : x;
        slope = x > 0.f ? 1.f : x == x ? 0.f : x;
    } else if (ACT == FMOE_ACT_GELU) {
        const gemm::GeluTerms g = gemm::gelu_terms(x);
        value = x * g.cdf;
        slope = g.cdf + x * g.pdf;
    } else {
        value = x;
        slope = x == x ? 1.f : x;
    }
}

struct Bytes8 { uint8_t byte[kLaneElems]; };

// Where a lane's piece lies: its elements begin at `at` and are n (0 or less: past the row's or the rows' end), its block's scale is number
// `block`; `inside`: eight elements there are the tensor's.
struct Piece { int64_t at, block; int n; bool inside; };
// The calling lane's; a workgroup's pieces begin at `first`.
template <bool FLAT> __device__ __forceinline__ Piece piece_at(int64_t first, int64_t rows, int d, uint32_t per_row) {
    const uint32_t mine = threadIdx.x;
    if (FLAT) {
        const int64_t i = first + mine;
        return Piece{i * kLaneElems, i / kLanes, i < rows * per_row ? kLaneElems : 0, true};
    }
    const int64_t row0 = div_small(first, per_row);
    const uint32_t from = (uint32_t)(first - row0 * per_row) + mine, down = from / per_row, c = from - down * per_row;
    const int64_t row = row0 + down, at = row * d + c * kLaneElems;
    const int left = d - (int)c * kLaneElems;
    return Piece{at, row * (per_row / kLanes) + c / kLanes, row < rows ? left < kLaneElems ? left : kLaneElems : 0, at + kLaneElems <= rows * d};
}

// The scale's byte for a block whose largest finite magnitude is `most`
__device__ __forceinline__ int scale_byte(float most) {
    const int bits = (int)__float_as_uint(most), b = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);   // 448 = 1.75 2^8
    return b < 1 ? 1 : b;
}
// The byte of the block that could round past the largest number of the type: 2^16 for float16, 2^128 for the others
template <typename T> constexpr int top_byte() { return std::is_same<T, _Float16>::value ? 16 - 8 + 127 : 128 - 8 + 127; }

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}

// rows that there are: all of them, or those that the experts' segments take
__device__ __forceinline__ int64_t live_rows(const int32_t *table, int64_t rows) {
    if (!table) return rows;
    const int64_t n = table[segtab::kRows];
    return n < rows ? n : rows;
}

// The largest of the values of the lanes that share a scale
__device__ __forceinline__ float lanes_max(float v) {
    static_assert(kLanes == 4, "a quad of lanes");
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0xb1, 0xf, 0xf, true)));          // quad_perm 1 0 3 2
    return fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x4e, 0xf, 0xf, true)));       // quad_perm 2 3 0 1
}

template <typename T, int ACT, bool FLAT>
__global__ __launch_bounds__(kBlock) void ckpt_fwd_kernel(const T *x, T *y, uint8_t *__restrict__ held, uint8_t *__restrict__ scale,
                                                          const int32_t *__restrict__ table, int64_t rows, int d, int per_row) {
    rows = live_rows(table, rows);
    const int64_t first = (int64_t)blockIdx.x * kBlock;
    if (first >= rows * per_row) return;
    const Piece at = piece_at<FLAT>(first, rows, d, per_row);
    T e[kLaneElems];
    load_elems<FLAT>(x + at.at, at.n, at.inside, e);
    float f[kLaneElems], most = 0.f;
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) {
        f[j] = (float)e[j];
        most = fmaxf(most, finite_magnitude(f[j]));
    }
    const int b = scale_byte(lanes_max(most));
    if (at.n <= 0) return;
    const float inv = __uint_as_float((uint32_t)(254 - b) << 23), limit = b == top_byte<T>() ? 240.f : 448.f;
    if (held && threadIdx.x % kLanes == 0) scale[at.block] = (uint8_t)b;
    float v[kLaneElems];
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) v[j] = fmaf(f[j], 0.f, __builtin_amdgcn_fmed3f(f[j] * inv, -limit, limit));
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        q[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
        q[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], q[h], true);
    }
    if (held) store_elems<FLAT>(held + at.at, at.n, __builtin_bit_cast(Bytes8, q).byte);
    if (y) {
#pragma unroll
        for (int j = 0; j < kLaneElems; ++j) e[j] = (T)act_value<ACT>(f[j]);
        store_elems<FLAT>(y + at.at, at.n, e);
    }
}

template <typename T, int ACT, bool FLAT>
__global__ __launch_bounds__(kBlock) void ckpt_bwd_kernel(const T *grad, const uint8_t *__restrict__ held,
                                                          const uint8_t *__restrict__ scale, T *grad_x, T *__restrict__ mid,
                                                          const int32_t *__restrict__ table, int64_t rows, int d, int per_row) {
    rows = live_rows(table, rows);
    const int64_t first = (int64_t)blockIdx.x * kBlock;
    if (first >= rows * per_row) return;
    const Piece at = piece_at<FLAT>(first, rows, d, per_row);
    T g[kLaneElems], m[kLaneElems];
    uint8_t q[kLaneElems];
    load_elems<FLAT>(held + at.at, at.n, at.inside, q);
    const float s = __uint_as_float((uint32_t)(at.n > 0 ? scale[at.block] : 0) << 23);
    if (grad) load_elems<FLAT>(grad + at.at, at.n, at.inside, g);
    const uint2 w = __builtin_bit_cast(uint2, q);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)(h ? w.y : w.x), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)(h ? w.y : w.x), true);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float value, slope;
            act_both<ACT>((i < 2 ? lo[i & 1] : hi[i & 1]) * s, value, slope);
            m[4 * h + i] = (T)value;
            if (grad) g[4 * h + i] = (T)((float)g[4 * h + i] * slope);
        }
    }
    if (grad) store_elems<FLAT>(grad_x + at.at, at.n, g);
    if (mid) store_elems<FLAT>(mid + at.at, at.n, m);
}

int per_row(int64_t d) { return (int)(ceil_div(d, kScaleElems) * kLanes); }   // pieces
int64_t n_blocks(int64_t rows, int64_t d) { return ceil_div(rows * per_row(d), kBlock); }

int check(const char *who, int64_t rows, int64_t d, int dtype, int activation) {
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who,
                 dtype);
    FMOE_REQUIRE(activation == FMOE_ACT_NONE || activation == FMOE_ACT_RELU || activation == FMOE_ACT_GELU, "%s: unknown activation %d",
                 who, activation);
    FMOE_REQUIRE(rows >= 0 && d >= 0, "%s: bad sizes", who);
    if (rows > (int64_t)INT32_MAX || d > (int64_t)(1 << 28) || n_blocks(rows, d) > kMostThreads / kBlock)
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    return FMOE_OK;
}

// launch(kernel's type, activation, whether the rows are whole blocks)
template <typename T, typename F> void with_activation(int activation, bool flat, F &&f) {
    auto go = [&](auto act) {
        if (flat) f(T{}, act, std::true_type{});
        else f(T{}, act, std::false_type{});
    };
    if (activation == FMOE_ACT_RELU) go(std::integral_constant<int, FMOE_ACT_RELU>{});
    else if (activation == FMOE_ACT_GELU) go(std::integral_constant<int, FMOE_ACT_GELU>{});
    else go(std::integral_constant<int, FMOE_ACT_NONE>{});
}
template <typename F> void with_kernel(int dtype, int activation, int64_t d, F &&f) {
    const bool flat = d % kScaleElems == 0;
    if (dtype == FMOE_F32) with_activation<float>(activation, flat, f);
    else if (dtype == FMOE_BF16) with_activation<__bf16>(activation, flat, f);
    else with_activation<_Float16>(activation, flat, f);
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_act_checkpoint_forward(const void *x, void *y, void *held, void *scale, const void *segment_table, int64_t rows,
                                           int64_t row_elems, int dtype, int activation, void *stream) {
    const char *who = "fmoe_act_checkpoint_forward";
    if (int rc = check(who, rows, row_elems, dtype, activation)) return rc;
    if (rows == 0 || row_elems == 0) return FMOE_OK;
    FMOE_REQUIRE(x && !held == !scale && (held || y), "%s: NULL pointer", who);
    with_kernel(dtype, activation, row_elems, [&](auto t, auto act, auto flat) {
        using T = decltype(t);
        ckpt_fwd_kernel<T, act.value, flat.value><<<(int)n_blocks(rows, row_elems), kBlock, 0, (hipStream_t)stream>>>(
            (const T *)x, (T *)y, (uint8_t *)held, (uint8_t *)scale, (const int32_t *)segment_table, rows, (int)row_elems, per_row(row_elems));
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

extern "C" int fmoe_act_checkpoint_backward(const void *grad, const void *held, const void *scale, void *grad_x, void *mid,
                                            const void *segment_table, int64_t rows, int64_t row_elems, int dtype, int activation,
                                            void *stream) {
    const char *who = "fmoe_act_checkpoint_backward";
    if (int rc = check(who, rows, row_elems, dtype, activation)) return rc;
    if (rows == 0 || row_elems == 0) return FMOE_OK;
    FMOE_REQUIRE(held && scale && !grad == !grad_x && (grad_x || mid), "%s: NULL pointer", who);
    with_kernel(dtype, activation, row_elems, [&](auto t, auto act, auto flat) {
        using T = decltype(t);
        ckpt_bwd_kernel<T, act.value, flat.value><<<(int)n_blocks(rows, row_elems), kBlock, 0, (hipStream_t)stream>>>(
            (const T *)grad, (const uint8_t *)held, (const uint8_t *)scale, (T *)grad_x, (T *)mid, (const int32_t *)segment_table, rows,
            (int)row_elems, per_row(row_elems));
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
