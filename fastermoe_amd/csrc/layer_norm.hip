// Layer norm of token rows, alone or of their sum with a residual, and its backward (gfx950).
//
//   s = x + r (rounded to the rows' type)      m = mean(s)   v = mean((s - m)^2)   rstd = 1 / sqrt(v + eps)   h = (s - m) rstd
//   y = h w + b
//   grad_s = rstd (a - mean(a) - h mean(a h)) + grad_sum,  a = grad_y w        grad_w = sum grad_y h      grad_b = sum grad_y
//
// Statistics, sums and everything between the loads and the one rounding at a store are float32.
//
// A row lies in the registers of G lanes, V vectors of 16 bytes to each, between its one load and its one store: G x V is the smallest that
// holds it (held_forward, held_backward).  Longer rows than any holds are read again for every sum (long_* kernels).
#include "common.hpp"
#include "lane_elems.hpp"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;
constexpr int kBwdBlock = 1024;      // of the backward over rows in registers
constexpr int kBwdMostBlocks = 256;  // and its workgroups at most, each of which leaves sums over its rows

// ---- sums over the G lanes of a row, the same in all of them ------------------------------
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <int G> __device__ __forceinline__ float lanes_sum(float v) {   // G <= 64
    v += dpp<0xb1>(v);                    // quad_perm 1 0 3 2
    v += dpp<0x4e>(v);                    // quad_perm 2 3 0 1
    if (G > 4) v += dpp<0x141>(v);        // row_half_mirror
    if (G > 8) v += dpp<0x140>(v);        // row_mirror
    if (G == 32) v += __uint_as_float(__builtin_amdgcn_ds_swizzle(__float_as_uint(v), 0x401f));   // the lane 16 away
    if (G == 64) {
        const float lo = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 0)) + __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 16));
        const float hi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 32)) + __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 48));
        v = lo + hi;
    }
    return v;
}
// NS sums; rows of more than one wave meet in scratch [waves of the workgroup][NS], which the next call must not be handed
template <int G, int NS> __device__ __forceinline__ void row_sums(float (&v)[NS], float (*scratch)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = lanes_sum<(G < kWave ? G : kWave)>(v[i]);
    if constexpr (G > kWave) {
        constexpr int kWaves = G / kWave;
        const int wave = threadIdx.x / kWave, first = wave / kWaves * kWaves;
        if (threadIdx.x % kWave == 0) {
#pragma unroll
            for (int i = 0; i < NS; ++i) scratch[wave][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            float s = scratch[first][i];
#pragma unroll
            for (int u = 1; u < kWaves; ++u) s += scratch[first + u][i];
            v[i] = s;
        }
    }
}

// N parameters from column c on; `none` where there are no parameters
template <typename P, int N> __device__ __forceinline__ void load_params(const P *p, int c, int d, float none, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = none;
    if (!p) return;
#pragma unroll
    for (int k = 0; k < N; k += Vec<P>::N) {
        float t[8];
        Vec<P>::unpack(load_vec(p + c + k, d - c - k, false), t);
#pragma unroll
        for (int i = 0; i < Vec<P>::N && k + i < N; ++i) f[k + i] = t[i];
    }
}

// ---- forward over rows in registers ------------------------------------------------------
template <typename T, typename P, int G, int V>
__global__ __launch_bounds__(G > kBlock ? G : kBlock) void norm_fwd_kernel(const T *__restrict__ x, int64_t x_stride, const T *__restrict__ r,
                                                                           int64_t r_stride, const P *__restrict__ w, const P *__restrict__ b,
                                                                           T *__restrict__ sum, T *__restrict__ y, float *__restrict__ mean,
                                                                           float *__restrict__ rstd, int64_t rows, int d, float eps) {
    constexpr int N = Vec<T>::N, kRows = (G > kBlock ? G : kBlock) / G;
    __shared__ float scratch[2][kRows * G / kWave][1];
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const bool live = row < rows;
    u32x4 e[V], re[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * G + lane) * N, n = live ? d - c : 0;
        e[v] = load_vec(x + row * x_stride + c, n, (row - rows + 1) * x_stride + c + N <= d);
        if (r) re[v] = load_vec(r + row * r_stride + c, n, (row - rows + 1) * r_stride + c + N <= d);
    }
    float f[V][8], s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
        Vec<T>::unpack(e[v], f[v]);
        if (r) {
            float t[8];
            Vec<T>::unpack(re[v], t);
#pragma unroll
            for (int i = 0; i < N; ++i) f[v][i] += t[i];
            e[v] = Vec<T>::pack(f[v]);
            Vec<T>::unpack(e[v], f[v]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) s[0] += f[v][i];
    }
    row_sums<G>(s, scratch[0]);
    const float m = s[0] / (float)d;
    s[0] = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            f[v][i] -= m;
            s[0] += (v * G + lane) * N + i < d ? f[v][i] * f[v][i] : 0.f;
        }
    row_sums<G>(s, scratch[1]);
    const float rs = 1.f / sqrtf(s[0] / (float)d + eps);
    if (!live) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * G + lane) * N, n = d - c;
        float wf[N], bf[N], out[8];
        load_params(w, c, d, 1.f, wf);
        load_params(b, c, d, 0.f, bf);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = f[v][i] * rs * wf[i] + bf[i];
        store_vec(y + row * d + c, n, Vec<T>::pack(out));
        if (sum) store_vec(sum + row * d + c, n, e[v]);
    }
    if (mean && lane == 0) {
        mean[row] = m;
        rstd[row] = rs;
    }
}

// ---- backward over rows in registers -----------------------------------------------------
// A workgroup takes kRows rows at a time and every gridDim-th such set, with the next set's loads on their way.  The lanes keep the sums of
// grad_y h and grad_y of their columns over all of them; at the end the sets' lanes meet in LDS and part[workgroup] gets 2 d sums.
template <int V> struct RowData {
    u32x4 g[V], x[V], gs[V];
    float mean, rstd;
};
template <typename T, typename P, int G, int V>
__global__ __launch_bounds__(kBwdBlock) void norm_bwd_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ gs,
                                                             int64_t gs_stride, const T *__restrict__ x, int64_t x_stride,
                                                             const float *__restrict__ mean, const float *__restrict__ rstd,
                                                             const P *__restrict__ w, T *__restrict__ gx, float *__restrict__ part,
                                                             int64_t rows, int d) {
    constexpr int N = Vec<T>::N, kRows = kBwdBlock / G;
    constexpr bool kAhead = V == 1 || V * N <= 8;
    __shared__ float scratch[2][kBwdBlock / kWave][2];
    __shared__ float sums[kRows > 1 ? kBwdBlock * V * N : 1];
    const int lane = threadIdx.x % G, mine = threadIdx.x / G;
    auto load = [&](int64_t row, RowData<V> &a) {
        const bool live = row < rows;
        const int64_t back = row - rows + 1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * G + lane) * N, n = live ? d - c : 0;
            a.g[v] = load_vec(gy + row * gy_stride + c, n, back * gy_stride + c + N <= d);
            a.x[v] = load_vec(x + row * x_stride + c, n, back * x_stride + c + N <= d);
            if (gs) a.gs[v] = load_vec(gs + row * gs_stride + c, n, back * gs_stride + c + N <= d);
        }
        a.mean = live ? mean[row] : 0.f;
        a.rstd = live ? rstd[row] : 0.f;
    };
    float wf[V][N], sw[V][N], sb[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * G + lane) * N;
        load_params(w, c, d, 1.f, wf[v]);
#pragma unroll
        for (int i = 0; i < N; ++i) sw[v][i] = sb[v][i] = 0.f;
    }
    const int64_t step = (int64_t)gridDim.x * kRows;
    RowData<V> a, next;
    int64_t row = (int64_t)blockIdx.x * kRows + mine;
    if (kAhead) load(row, a);
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * kRows; first < rows; first += step, row += step, turn ^= 1) {
        if (kAhead) {
            if (first + step < rows) load(row + step, next);
        } else {
            load(row, a);
        }
        float c12[2] = {0.f, 0.f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float g[8], h[8];
            Vec<T>::unpack(a.g[v], g);
            Vec<T>::unpack(a.x[v], h);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                h[i] = (h[i] - a.mean) * a.rstd;
                const float t = g[i] * wf[v][i];
                c12[0] += t;
                c12[1] += t * h[i];
                sw[v][i] += g[i] * h[i];
                sb[v][i] += g[i];
            }
        }
        row_sums<G>(c12, scratch[turn]);
        if (gx && row < rows) {
            const float c1 = c12[0] / (float)d, c2 = c12[1] / (float)d;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = (v * G + lane) * N;
                float g[8], h[8], t[8];
                Vec<T>::unpack(a.g[v], g);
                Vec<T>::unpack(a.x[v], h);
                if (gs) Vec<T>::unpack(a.gs[v], t);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    h[i] = (h[i] - a.mean) * a.rstd;
                    g[i] = a.rstd * (g[i] * wf[v][i] - c1 - h[i] * c2);
                    if (gs) g[i] += t[i];
                }
                store_vec(gx + row * d + c, d - c, Vec<T>::pack(g));
            }
        }
        if (kAhead) a = next;
    }
    if (!part) return;
    float *out = part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
    for (int which = 0; which < 2; ++which, out += d) {
        if constexpr (kRows == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) store_elems<false>(out + (v * G + lane) * N, d - (v * G + lane) * N, which ? sb[v] : sw[v]);
        } else {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) sums[(mine * V + v) * G * N + i * G + lane] = which ? sb[v][i] : sw[v][i];
            __syncthreads();
            // (a column's place: its vector's number, then which of the vector's elements, then the lane)
            for (int c = threadIdx.x; c < d; c += kBwdBlock) {
                const int v = c / (G * N), at = c % (G * N), place = v * G * N + at % N * G + at / N;
                float s = 0.f;
#pragma unroll
                for (int u = 0; u < kRows; ++u) s += sums[u * V * G * N + place];
                out[c] = s;
            }
        }
    }
}

// ---- rows longer than the registers ---------------------------------------------------------
__device__ __forceinline__ float block_sum(float v, float *scratch) {
    v = lanes_sum<kWave>(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWavesPerBlock; ++w) v += scratch[w];
    return v;
}

template <typename T, typename P>
__global__ __launch_bounds__(kBlock) void long_fwd_kernel(const T *__restrict__ x, int64_t x_stride, const T *__restrict__ r,
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
__global__ __launch_bounds__(kBlock) void long_bwd_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ gs,
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
__global__ __launch_bounds__(kBlock) void long_param_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ x,
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

// grad_w and grad_b out of the parts, in their order: 32 columns to a workgroup, eight ranges of parts side by side
constexpr int kSumCols = 32, kSumRanges = kBlock / kSumCols;
template <typename P>
__global__ __launch_bounds__(kBlock) void norm_param_sum_kernel(const float *__restrict__ part, int n_parts, P *__restrict__ gw,
                                                                P *__restrict__ gb, int64_t d) {
    __shared__ float sums[kSumRanges][kSumCols];
    const int col = threadIdx.x % kSumCols, range = threadIdx.x / kSumCols;
    const int64_t c = (int64_t)blockIdx.x * kSumCols + col;
    const int per = (n_parts + kSumRanges - 1) / kSumRanges, lo = range * per, hi = lo + per < n_parts ? lo + per : n_parts;
    float s = 0.f;
    if (c < 2 * d) {
#pragma unroll 8
        for (int p = lo; p < hi; ++p) s += part[(int64_t)p * 2 * d + c];
    }
    sums[range][col] = s;
    __syncthreads();
    if (range != 0 || c >= 2 * d) return;
#pragma unroll
    for (int u = 1; u < kSumRanges; ++u) s += sums[u][col];
    P *out = c < d ? gw : gb;
    if (out) out[c < d ? c : c - d] = (P)s;
}

// How a row is held: f(lanes, vectors to each), integral constants; false where nothing holds it
template <int N, int G, int V, typename F> bool held_by(int64_t d, F &&f) {
    if (d > (int64_t)G * V * N) return false;
    f(std::integral_constant<int, G>{}, std::integral_constant<int, V>{});
    return true;
}
template <int N, typename F> bool held_forward(int64_t d, F &&f) {
    return held_by<N, 8, 1>(d, f) || held_by<N, 32, 1>(d, f) || held_by<N, 64, 1>(d, f) || held_by<N, 64, 2>(d, f) || held_by<N, 256, 1>(d, f) ||
           held_by<N, 256, 2>(d, f) || held_by<N, 1024, 1>(d, f) || held_by<N, 1024, 2>(d, f) || held_by<N, 1024, 4>(d, f);
}
template <int N, typename F> bool held_backward(int64_t d, F &&f) {
    if (held_by<N, 8, 1>(d, f) || held_by<N, 32, 1>(d, f) || held_by<N, 64, 1>(d, f) || held_by<N, 128, 1>(d, f) || held_by<N, 256, 1>(d, f) ||
        held_by<N, 512, 1>(d, f) || held_by<N, 1024, 1>(d, f) || held_by<N, 1024, 2>(d, f))
        return true;
    if constexpr (N == 4) return held_by<N, 1024, 4>(d, f);
    return false;
}

constexpr int kLongParts = 128;
int n_parts(int64_t rows) { return (int)(rows < 1 ? 1 : rows < kBwdMostBlocks ? rows : kBwdMostBlocks); }

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
        const bool held = held_forward<Vec<T>::N>(row_elems, [&](auto g, auto v) {
            constexpr int kThreads = g.value > kBlock ? g.value : kBlock;
            norm_fwd_kernel<T, P, g.value, v.value><<<(int)ceil_div(rows, kThreads / g.value), kThreads, 0, st>>>(
                (const T *)x, x_stride, (const T *)residual, residual_stride, (const P *)weight, (const P *)bias, (T *)sum, (T *)y, mean, rstd,
                rows, (int)row_elems, (float)eps);
        });
        if (!held)
            long_fwd_kernel<T, P><<<(int)rows, kBlock, 0, st>>>((const T *)x, x_stride, (const T *)residual, residual_stride,
                                                                (const P *)weight, (const P *)bias, (T *)sum, (T *)y, mean, rstd, row_elems,
                                                                (float)eps);
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
    if (params && (!workspace || workspace_bytes < fmoe_layer_norm_backward_workspace_bytes(rows, row_elems)))
        return fail(FMOE_EWORKSPACE, "%s: workspace of %lld bytes, %lld needed", who, (long long)workspace_bytes,
                    (long long)fmoe_layer_norm_backward_workspace_bytes(rows, row_elems));
    hipStream_t st = (hipStream_t)stream;
    with_types(dtype, param_dtype, [&](auto t, auto p) {
        using T = decltype(t);
        using P = decltype(p);
        int parts = 0;
        const bool held = held_backward<Vec<T>::N>(row_elems, [&](auto g, auto v) {
            const int64_t sets = ceil_div(rows < 1 ? 1 : rows, kBwdBlock / g.value);
            parts = (int)(sets < kBwdMostBlocks ? sets : kBwdMostBlocks);
            norm_bwd_kernel<T, P, g.value, v.value><<<parts, kBwdBlock, 0, st>>>(
                (const T *)grad_y, grad_y_stride, (const T *)grad_sum, grad_sum_stride, (const T *)x, x_stride, mean, rstd, (const P *)weight,
                (T *)grad_x, params ? (float *)workspace : nullptr, rows, (int)row_elems);
        });
        if (!held) {
            parts = n_parts(rows) < kLongParts ? n_parts(rows) : kLongParts;
            if (grad_x && rows > 0)
                long_bwd_kernel<T, P><<<(int)rows, kBlock, 0, st>>>((const T *)grad_y, grad_y_stride, (const T *)grad_sum, grad_sum_stride,
                                                                    (const T *)x, x_stride, mean, rstd, (const P *)weight, (T *)grad_x,
                                                                    row_elems);
            if (params)
                long_param_kernel<T><<<dim3((int)ceil_div(row_elems, kBlock), parts), kBlock, 0, st>>>(
                    (const T *)grad_y, grad_y_stride, (const T *)x, x_stride, mean, rstd, (float *)workspace, rows, row_elems);
        }
        if (params)
            norm_param_sum_kernel<P><<<(int)ceil_div(2 * row_elems, kSumCols), kBlock, 0, st>>>((const float *)workspace, parts, (P *)grad_weight,
                                                                                               (P *)grad_bias, row_elems);
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
