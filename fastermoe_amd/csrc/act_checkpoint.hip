// The experts' rows kept in 8 bits for the backward pass (gfx950).
//
// A block of 32 elements along a row (fewer at its end) is held as e4m3 numbers under one power of two, the smallest 2^b
// (b >= -126) with max|x| <= 448 2^b over the block's finite elements:  q = e4m3(x 2^-b), to nearest, ties to even; the scale is the
// byte b + 127.  Dividing by a power of two is exact, so the numbers are off by their own rounding alone: 2^-4 of themselves, or, small
// against the block, 2^-10 2^b.  What rounds to more than the rows' type holds is held as the largest that it does (240 2^b in the one
// block that can); infinities and NaN are held as NaN, so that a forward that overflowed still shows in the gradients.
//
//   forward   y = act(x), q, b          backward  x~ = q 2^b   mid = act(x~)   grad_x = grad act'(x~)
#include "common.hpp"
#include "gelu_terms.hpp"
#include "grouped_gemm.hpp"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kScaleElems = 32;

__device__ __forceinline__ float act_value(float x, int act) {
    if (act == FMOE_ACT_RELU) return x < 0.f ? 0.f : x;   // (NaN stays)
    if (act == FMOE_ACT_GELU) return x * gemm::gelu_terms(x).cdf;
    return x;
}
__device__ __forceinline__ float act_slope(float x, int act) {
    if (act == FMOE_ACT_RELU) return x > 0.f ? 1.f : x == x ? 0.f : x;
    if (act == FMOE_ACT_GELU) {
        const gemm::GeluTerms g = gemm::gelu_terms(x);
        return g.cdf + x * g.pdf;
    }
    return x == x ? 1.f : x;
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

template <typename T>
__global__ __launch_bounds__(kBlock) void ckpt_fwd_kernel(const T *x, T *y, uint8_t *__restrict__ held, uint8_t *__restrict__ scale,
                                                          const int32_t *__restrict__ table, int64_t rows, int64_t d, int act) {
    const int64_t per_row = (d + kScaleElems - 1) / kScaleElems;
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x, row = i / per_row, c0 = (i - row * per_row) * kScaleElems;
    if (row >= live_rows(table, rows)) return;
    const int n = (int)(d - c0 < kScaleElems ? d - c0 : kScaleElems);
    const int64_t at = row * d + c0;
    float most = 0.f;
    for (int j = 0; j < n; ++j) most = fmaxf(most, finite_magnitude((float)x[at + j]));
    const int b = scale_byte(most);
    const float inv = __uint_as_float((uint32_t)(254 - b) << 23), limit = b == top_byte<T>() ? 240.f : 448.f;
    scale[i] = (uint8_t)b;
    for (int j = 0; j < n; ++j) {
        const float v = (float)x[at + j];
        const float q = fmaf(v, 0.f, __builtin_amdgcn_fmed3f(v * inv, -limit, limit));
        held[at + j] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
        if (y) y[at + j] = (T)act_value(v, act);
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void ckpt_bwd_kernel(const T *grad, const uint8_t *__restrict__ held,
                                                          const uint8_t *__restrict__ scale, T *grad_x, T *__restrict__ mid,
                                                          const int32_t *__restrict__ table, int64_t rows, int64_t d, int act) {
    const int64_t per_row = (d + kScaleElems - 1) / kScaleElems;
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x, row = i / per_row, c0 = (i - row * per_row) * kScaleElems;
    if (row >= live_rows(table, rows)) return;
    const int n = (int)(d - c0 < kScaleElems ? d - c0 : kScaleElems);
    const int64_t at = row * d + c0;
    const float s = __uint_as_float((uint32_t)scale[i] << 23);
    for (int j = 0; j < n; ++j) {
        const float v = __builtin_amdgcn_cvt_f32_fp8((int)held[at + j], 0) * s;
        if (grad_x) grad_x[at + j] = (T)((float)grad[at + j] * act_slope(v, act));
        if (mid) mid[at + j] = (T)act_value(v, act);
    }
}

int check(const char *who, int64_t rows, int64_t d, int dtype, int activation) {
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who,
                 dtype);
    FMOE_REQUIRE(activation == FMOE_ACT_NONE || activation == FMOE_ACT_RELU || activation == FMOE_ACT_GELU, "%s: unknown activation %d",
                 who, activation);
    FMOE_REQUIRE(rows >= 0 && d >= 0, "%s: bad sizes", who);
    if (rows > (int64_t)INT32_MAX || d > (int64_t)(1 << 28) || ceil_div(rows * ceil_div(d, kScaleElems), kBlock) > INT32_MAX)
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    return FMOE_OK;
}

template <typename F> void with_type(int dtype, F &&f) {
    if (dtype == FMOE_F32) f(float{});
    else if (dtype == FMOE_BF16) f(__bf16{});
    else f(_Float16{});
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_act_checkpoint_forward(const void *x, void *y, void *held, void *scale, const void *segment_table, int64_t rows,
                                           int64_t row_elems, int dtype, int activation, void *stream) {
    const char *who = "fmoe_act_checkpoint_forward";
    if (int rc = check(who, rows, row_elems, dtype, activation)) return rc;
    if (rows == 0 || row_elems == 0) return FMOE_OK;
    FMOE_REQUIRE(x && held && scale, "%s: NULL pointer", who);
    const int blocks = (int)ceil_div(rows * ceil_div(row_elems, kScaleElems), kBlock);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        ckpt_fwd_kernel<T><<<blocks, kBlock, 0, (hipStream_t)stream>>>((const T *)x, (T *)y, (uint8_t *)held, (uint8_t *)scale,
                                                                       (const int32_t *)segment_table, rows, row_elems, activation);
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
    const int blocks = (int)ceil_div(rows * ceil_div(row_elems, kScaleElems), kBlock);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        ckpt_bwd_kernel<T><<<blocks, kBlock, 0, (hipStream_t)stream>>>((const T *)grad, (const uint8_t *)held, (const uint8_t *)scale,
                                                                       (T *)grad_x, (T *)mid, (const int32_t *)segment_table, rows,
                                                                       row_elems, activation);
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
