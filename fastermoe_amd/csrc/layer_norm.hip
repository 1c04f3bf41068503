// Layer norm of token rows, alone or of their sum with a residual, and its backward (gfx950).
//
//   s = x + r (rounded to the rows' type)      m = mean(s)   v = mean((s - m)^2)   rstd = 1 / sqrt(v + eps)   h = (s - m) rstd
//   y = h w + b
//   grad_s = rstd (a - mean(a) - h mean(a h)) + grad_sum,  a = grad_y w        grad_w = sum grad_y h      grad_b = sum grad_y
//
// Statistics, sums and everything between the loads and the one rounding at a store are float32.
#include "common.hpp"

namespace fmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;

__device__ __forceinline__ float block_sum(float v, float *scratch) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    __syncthreads();
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWavesPerBlock; ++w) v += scratch[w];
    return v;
}

template <typename T, typename P>
__global__ __launch_bounds__(kBlock) void norm_fwd_kernel(const T *__restrict__ x, int64_t x_stride, const T *__restrict__ r,
                                                          int64_t r_stride, const P *__restrict__ w, const P *__restrict__ b,
                                                          T *__restrict__ sum, T *__restrict__ y, float *__restrict__ mean,
                                                          float *__restrict__ rstd, int64_t d, float eps) {
    __shared__ float scratch[kWavesPerBlock];
    const int64_t row = blockIdx.x;
    auto at = [&](int64_t c) {
        const float v = (float)x[row * x_stride + c];
        return r ? (float)(T)(v + (float)r[row * r_stride + c]) : v;
    };
    float acc = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += kBlock) acc += at(c);
    const float m = block_sum(acc, scratch) / (float)d;
    acc = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += kBlock) acc += (at(c) - m) * (at(c) - m);
    const float rs = 1.f / sqrtf(block_sum(acc, scratch) / (float)d + eps);
    for (int64_t c = threadIdx.x; c < d; c += kBlock) {
        const float v = at(c);
        if (sum) sum[row * d + c] = (T)v;
        y[row * d + c] = (T)((v - m) * rs * (w ? (float)w[c] : 1.f) + (b ? (float)b[c] : 0.f));
    }
    if (mean && threadIdx.x == 0) {
        mean[row] = m;
        rstd[row] = rs;
    }
}

template <typename T, typename P>
__global__ __launch_bounds__(kBlock) void norm_bwd_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ gs,
                                                          int64_t gs_stride, const T *__restrict__ x, int64_t x_stride,
                                                          const float *__restrict__ mean, const float *__restrict__ rstd,
                                                          const P *__restrict__ w, T *__restrict__ gx, int64_t d) {
    __shared__ float scratch[kWavesPerBlock];
    const int64_t row = blockIdx.x;
    const float m = mean[row], rs = rstd[row];
    float c1 = 0.f, c2 = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += kBlock) {
        const float a = (float)gy[row * gy_stride + c] * (w ? (float)w[c] : 1.f);
        c1 += a;
        c2 += a * ((float)x[row * x_stride + c] - m) * rs;
    }
    c1 = block_sum(c1, scratch) / (float)d;
    c2 = block_sum(c2, scratch) / (float)d;
    for (int64_t c = threadIdx.x; c < d; c += kBlock) {
        const float a = (float)gy[row * gy_stride + c] * (w ? (float)w[c] : 1.f);
        const float h = ((float)x[row * x_stride + c] - m) * rs;
        const float g = rs * (a - c1 - h * c2);
        gx[row * d + c] = (T)(gs ? g + (float)gs[row * gs_stride + c] : g);
    }
}

// Sums over a range of rows each, a column to each thread: part[range] holds grad_w's d sums and then grad_b's
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_param_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ x,
                                                            int64_t x_stride, const float *__restrict__ mean,
                                                            const float *__restrict__ rstd, float *__restrict__ part, int64_t rows,
                                                            int64_t d) {
    const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= d) return;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * per, hi = lo + per < rows ? lo + per : rows;
    float sw = 0.f, sb = 0.f;
    for (int64_t t = lo; t < hi; ++t) {
        const float g = (float)gy[t * gy_stride + c];
        sw += g * ((float)x[t * x_stride + c] - mean[t]) * rstd[t];
        sb += g;
    }
    part[(int64_t)blockIdx.y * 2 * d + c] = sw;
    part[(int64_t)blockIdx.y * 2 * d + d + c] = sb;
}

template <typename P>
__global__ __launch_bounds__(kBlock) void norm_param_sum_kernel(const float *__restrict__ part, int n_parts, P *__restrict__ gw,
                                                                P *__restrict__ gb, int64_t d) {
    const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= 2 * d) return;
    float s = 0.f;
    for (int p = 0; p < n_parts; ++p) s += part[(int64_t)p * 2 * d + c];
    P *out = c < d ? gw : gb;
    if (out) out[c < d ? c : c - d] = (P)s;
}

constexpr int kMostParts = 128;
int n_parts(int64_t rows) { return (int)(rows < 16 * kMostParts ? ceil_div(rows < 1 ? 1 : rows, 16) : kMostParts); }

int check(const char *who, int64_t rows, int64_t d, int dtype, int param_dtype) {
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who,
                 dtype);
    FMOE_REQUIRE(param_dtype == dtype || param_dtype == FMOE_F32, "%s: parameters must be of the rows' type or float32", who);
    FMOE_REQUIRE(rows >= 0 && d >= 1, "%s: bad sizes", who);
    if (rows > (int64_t)INT32_MAX || d > (int64_t)(1 << 28)) return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    return FMOE_OK;
}

// f(T{}, P{}) for the rows' and the parameters' types
template <typename F> void with_types(int dtype, int param_dtype, F &&f) {
    if (dtype == FMOE_F32) f(float{}, float{});
    else if (dtype == FMOE_BF16) { if (param_dtype == FMOE_F32) f(__bf16{}, float{}); else f(__bf16{}, __bf16{}); }
    else { if (param_dtype == FMOE_F32) f(_Float16{}, float{}); else f(_Float16{}, _Float16{}); }
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_layer_norm_forward(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                                       const void *weight, const void *bias, void *sum, void *y, float *mean, float *rstd,
                                       int64_t rows, int64_t row_elems, double eps, int dtype, int param_dtype, void *stream) {
    const char *who = "fmoe_layer_norm_forward";
    if (int rc = check(who, rows, row_elems, dtype, param_dtype)) return rc;
    FMOE_REQUIRE(x_stride >= 0 && residual_stride >= 0, "%s: negative stride", who);
    FMOE_REQUIRE(eps >= 0, "%s: eps must not be negative", who);
    if (rows == 0) return FMOE_OK;
    FMOE_REQUIRE(x && y && (sum || !residual) && !mean == !rstd, "%s: NULL pointer", who);
    hipStream_t st = (hipStream_t)stream;
    with_types(dtype, param_dtype, [&](auto t, auto p) {
        using T = decltype(t);
        using P = decltype(p);
        norm_fwd_kernel<T, P><<<(int)rows, kBlock, 0, st>>>((const T *)x, x_stride, (const T *)residual, residual_stride, (const P *)weight,
                                                            (const P *)bias, (T *)sum, (T *)y, mean, rstd, row_elems, (float)eps);
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

extern "C" int64_t fmoe_layer_norm_backward_workspace_bytes(int64_t rows, int64_t row_elems) {
    if (rows < 0 || row_elems < 1) return 0;
    return (int64_t)n_parts(rows) * 2 * row_elems * 4;
}

extern "C" int fmoe_layer_norm_backward(const void *grad_y, int64_t grad_y_stride, const void *grad_sum, int64_t grad_sum_stride,
                                        const void *x, int64_t x_stride, const float *mean, const float *rstd, const void *weight,
                                        void *grad_x, void *grad_weight, void *grad_bias, int64_t rows, int64_t row_elems, int dtype,
                                        int param_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "fmoe_layer_norm_backward";
    if (int rc = check(who, rows, row_elems, dtype, param_dtype)) return rc;
    FMOE_REQUIRE(grad_y_stride >= 0 && grad_sum_stride >= 0 && x_stride >= 0, "%s: negative stride", who);
    FMOE_REQUIRE(rows == 0 || (grad_y && x && mean && rstd), "%s: NULL pointer", who);
    const bool params = grad_weight || grad_bias;
    if (!params && (rows == 0 || !grad_x)) return FMOE_OK;
    const int parts = n_parts(rows);
    if (params && (!workspace || workspace_bytes < fmoe_layer_norm_backward_workspace_bytes(rows, row_elems)))
        return fail(FMOE_EWORKSPACE, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
                    (long long)fmoe_layer_norm_backward_workspace_bytes(rows, row_elems));
    hipStream_t st = (hipStream_t)stream;
    with_types(dtype, param_dtype, [&](auto t, auto p) {
        using T = decltype(t);
        using P = decltype(p);
        if (grad_x && rows > 0)
            norm_bwd_kernel<T, P><<<(int)rows, kBlock, 0, st>>>((const T *)grad_y, grad_y_stride, (const T *)grad_sum, grad_sum_stride,
                                                                (const T *)x, x_stride, mean, rstd, (const P *)weight, (T *)grad_x,
                                                                row_elems);
        if (params) {
            norm_param_kernel<T><<<dim3((int)ceil_div(row_elems, kBlock), parts), kBlock, 0, st>>>(
                (const T *)grad_y, grad_y_stride, (const T *)x, x_stride, mean, rstd, (float *)workspace, rows, row_elems);
            norm_param_sum_kernel<P><<<(int)ceil_div(2 * row_elems, kBlock), kBlock, 0, st>>>((const float *)workspace, parts,
                                                                                             (P *)grad_weight, (P *)grad_bias, row_elems);
        }
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
