// Layer norm of token rows, alone or of their sum with a residual, and its backward (gfx950).
//
//   s = x + r (rounded to the rows' type)      m = mean(s)   v = mean((s - m)^2)   rstd = 1 / sqrt(v + eps)   h = (s - m) rstd
//   y = h w + b
//   grad_s = rstd (a - mean(a) - h mean(a h)) + grad_sum,  a = grad_y w        grad_w = sum grad_y h      grad_b = sum grad_y
//
// Statistics, sums and everything between the loads and the one rounding at a store are float32 or more.
//
// A row lies in the registers of G lanes, V vectors of 16 bytes to each, between its one load and its one store: G x V is the smallest that
// holds it (held_forward, held_backward), wherever it begins and whatever its length.  Rows longer than any holds, or shorter than a vector, are read again for
// every sum (long_* kernels: 1000 bfloat16 rows of 40000 take 208 us and 317).  Bound by memory (us by events, small launches eight to a graph; TB/s of what has
// to move; a large copy on the same card 5.0):
//   rows x features             forward          backward            of it without the parameters' gradients
//   16384 x 4096 bf16, residual   92 us  5.8        91 us  5.9         84 us  6.4
//   32768 x 4096 bf16             98     5.5       144     5.6        137     5.9
//   16384 x 2048 f32, residual    92     5.8        88     6.1         83     6.4
//   32768 x 1024 bf16             26     5.1        41     4.9         36     5.6
//   65536 x 900 bf16, residual    85     5.5        86     5.5
//   32768 x 500 bf16              15     4.4        22     4.4         17     5.8
//   5000 x 12000 bf16, residual   91     5.3       130     3.7        116     4.1
//   3600 x 16384 f32, residual   184     5.1       212     4.5        197     4.8
//   509 x 4096 f16, residual      6.0               13                5.1
//   64 x 4096 bf16, residual      3.8               8.9               4.1
// (The first with a row read again for every sum and the parameters' gradients in a pass of their own: 358 and 431 us.  Rows of 900 and 500 whose last
// elements were loaded and stored apart: 102 and 129, 18 and 27.)  The backward over the longest held rows does not fit its registers: 16-bit rows of 8193 to 16384
// elements spill 10 to 19 of a lane's 128 to scratch memory (44 to 80 bytes; 3.7 to 4.1 TB/s), float32 rows of 8193 to 16384 keep 160 bytes there (3.7 to 4.5), and those
// of 4097 to 8192 with a residual spill 11 of 256 (48 bytes; 3001 x 8192 79 us, 5.0 TB/s).
#include "common.hpp"
#include "lane_elems.hpp"

#include <type_traits>

namespace fmoe {
namespace {

constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;
constexpr int bwd_threads(int v) { return v >= 4 ? 512 : 1024; }   // of the backward over rows in registers: twice the registers for long float32 rows
constexpr int kBwdMostBlocks = 256;  // and its workgroups at most, each of which leaves sums over its rows
constexpr int64_t kPartBytes = 4 << 20;
constexpr int64_t kCacheBytes = 256 << 20;   // of the memory-side cache
constexpr int kFewRows = 2048;

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
// N numbers, a power of two of them: neighbours, then neighbours of those
template <int N> __device__ __forceinline__ float pairs_sum(const float (&s)[N]) {
    float t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = s[i];
#pragma unroll
    for (int n = N; n > 1; n /= 2)
#pragma unroll
        for (int i = 0; i < n / 2; ++i) t[i] = t[2 * i] + t[2 * i + 1];
    return t[0];
}
// NS sums; rows of more than one wave meet in scratch [waves of the workgroup][NS] (another scratch than the call before, whose sums may still be read)
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
            float s[kWaves];
#pragma unroll
            for (int u = 0; u < kWaves; ++u) s[u] = scratch[first + u][i];
            v[i] = pairs_sum<kWaves>(s);
        }
    }
}

// weight or bias: of the rows' type or float32; none where the pointer is null
struct Param { const void *p; bool f32; };
// N of them from column `from` on; `none` where there are none
template <typename T, int N> __device__ __forceinline__ void load_params(const Param &p, int from, float none, float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = none;
    if (!p.p) return;
    float t[8];
    if (sizeof(T) == 2 && !p.f32) {
        Vec<T>::unpack(*(const AnyVec *)((const T *)p.p + from), t);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = t[i];
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            Vec<float>::unpack(*(const AnyVec *)((const float *)p.p + from + k), t);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[k + i] = t[i];
        }
    }
}

// Where a lane's vector number v lies in a row of d >= N elements: it begins at `from` and its first `skip` elements are another lane's.  The last vector of
// a row that is not whole vectors ends with the row and overlaps the one before it, whose lane does what the sums need of the elements they
// share; what both store there is the same.  Lanes behind the row's end take its last vector and none of its elements (skip >= N).
template <int N> struct Place {
    int from, skip;
    __device__ __forceinline__ Place(int vec, int d) : from(vec * N < d - N ? vec * N : d - N), skip(vec * N - from) {}
    __device__ __forceinline__ bool own(int i) const { return i >= skip; }
};

// The lane's vector of row `row` of `rows`, of the last one where there is none.  Always a load, with neither a branch around it nor a look at what it
// brought, either of which would have everything before its use wait for it.
template <bool ONCE, typename T> __device__ __forceinline__ u32x4 load_row(const T *p, int64_t stride, int64_t row, int64_t rows, int from) {
    const AnyVec *at = (const AnyVec *)(p + (row < rows ? row : rows - 1) * stride + from);
    return ONCE ? (u32x4)__builtin_nontemporal_load(at) : (u32x4)*at;
}
template <bool ONCE, typename T> __device__ __forceinline__ void store_row(T *p, const u32x4 &v) {
    if (ONCE) __builtin_nontemporal_store(v, (AnyVec *)p);
    else *(AnyVec *)p = v;
}

// ---- forward over rows in registers ------------------------------------------------------
// Where held_forward's rule on the number of rows chooses between one vector to a lane and two in half the lanes, the sums over the two are made
// apart, and all of them are joined in pairs: the order is that of the row's vectors, 64 at a time, either way, so that a row's result has the same bits however
// many rows there are.  (Longer rows, which one layout holds, add a lane's vectors up first: apart, 4096 x 16384 bfloat16 take 70 us instead of 51.)
template <typename T, int G, int V>
__global__ __launch_bounds__(G > kBlock ? G : kBlock) void norm_fwd_kernel(const T *__restrict__ x, int64_t x_stride, const T *__restrict__ r,
                                                                           int64_t r_stride, Param w, Param b, T *__restrict__ sum,
                                                                           T *__restrict__ y, float *__restrict__ mean,
                                                                           float *__restrict__ rstd, int64_t rows, int d, float eps) {
    constexpr int N = Vec<T>::N, kRows = (G > kBlock ? G : kBlock) / G, S = V == 2 && G <= 256 ? V : 1;
    __shared__ float scratch[2][kRows * G / kWave][S];
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    u32x4 e[V], re[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Place<N> at(v * G + lane, d);
        e[v] = load_row<false>(x, x_stride, row, rows, at.from);
        if (r) re[v] = load_row<false>(r, r_stride, row, rows, at.from);
    }
    float f[V][8], s[S] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Place<N> at(v * G + lane, d);
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
        for (int i = 0; i < N; ++i) s[v % S] += at.own(i) ? f[v][i] : 0.f;
    }
    row_sums<G>(s, scratch[0]);
    const float m = pairs_sum<S>(s) / (float)d;
#pragma unroll
    for (int i = 0; i < S; ++i) s[i] = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Place<N> at(v * G + lane, d);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            f[v][i] -= m;
            const float t = at.own(i) ? f[v][i] : 0.f;
            s[v % S] = fmaf(t, t, s[v % S]);
        }
    }
    row_sums<G>(s, scratch[1]);
    const float rs = 1.f / sqrtf(pairs_sum<S>(s) / (float)d + eps);
    if (row >= rows) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Place<N> at(v * G + lane, d);
        if (at.skip >= N) continue;
        float wf[N], bf[N], out[8];
        load_params<T, N>(w, at.from, 1.f, wf);
        load_params<T, N>(b, at.from, 0.f, bf);
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = fmaf(f[v][i] * rs, wf[i], bf[i]);
        store_row<false>(y + row * d + at.from, Vec<T>::pack(out));
        if (sum) store_row<false>(sum + row * d + at.from, e[v]);
    }
    if (mean && lane == 0) {
        mean[row] = m;
        rstd[row] = rs;
    }
}

// ---- backward over rows in registers -----------------------------------------------------
// A workgroup takes kRows rows at a time and every gridDim-th such set, with the next set's loads on their way (16384 x 4096: 104 us where a
// branch or a select made the sums wait for them).  The lanes keep the sums of grad_y h and grad_y of their columns over all of them; at the end the
// lanes of one column meet in LDS and part[workgroup] gets 2 d sums.  One workgroup of 1024 to a compute unit: two of 512 leave twice the parts (4096 x 8192:
// 59 us against 68).  One vector to a lane, where the next set's registers fit beside this one's; longer rows take two and no set ahead, in float32
// four (ahead) or eight in half the lanes (2048 x 8192, residual: 60 us against 78 with two in 1024 lanes; 3600 x 16384 212 against 249 with four, and
// 191 against 156 without a residual).
template <int V> struct RowData {
    u32x4 g[V], x[V], gs[V];
    float mean, rstd;
};
template <typename T, int G, int V, bool ONCE, bool SUM>
__global__ __launch_bounds__(bwd_threads(V)) void norm_bwd_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ gs,
                                                             int64_t gs_stride, const T *__restrict__ x, int64_t x_stride,
                                                             const float *__restrict__ mean, const float *__restrict__ rstd, Param w,
                                                             T *__restrict__ gx, float *__restrict__ part, int64_t rows, int d) {
    constexpr int N = Vec<T>::N, kThreads = bwd_threads(V), kRows = kThreads / G;
    constexpr bool kAhead = V * N <= (kThreads == 512 ? 16 : 8);
    __shared__ float scratch[2][kThreads / kWave][2];
    __shared__ float sums[kRows > 1 ? kThreads * V * N : 1];
    const int lane = threadIdx.x % G, mine = threadIdx.x / G;
    auto load = [&](int64_t row, RowData<V> &a) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Place<N> at(v * G + lane, d);
            if (SUM) a.gs[v] = load_row<ONCE>(gs, gs_stride, row, rows, at.from);
            a.g[v] = load_row<ONCE>(gy, gy_stride, row, rows, at.from);
            a.x[v] = load_row<ONCE>(x, x_stride, row, rows, at.from);
        }
        const int64_t at = row < rows ? row : rows - 1;
        a.mean = mean[at];
        a.rstd = rstd[at];
    };
    float wf[V][N], sw[V][N], sb[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        load_params<T, N>(w, Place<N>(v * G + lane, d).from, 1.f, wf[v]);
#pragma unroll
        for (int i = 0; i < N; ++i) sw[v][i] = sb[v][i] = 0.f;
    }
    int turn = 0;
    // one set's rows: sums, the gradient of the rows, and what they add to the parameters'
    auto use = [&](int64_t row, RowData<V> &a) {
        const bool live = row < rows;
        float c12[2] = {0.f, 0.f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Place<N> at(v * G + lane, d);
            float g[8], h[8];
            Vec<T>::unpack(a.g[v], g);
            Vec<T>::unpack(a.x[v], h);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                g[i] = live && at.own(i) ? g[i] : 0.f;
                h[i] = (h[i] - a.mean) * a.rstd;
                const float t = g[i] * wf[v][i];
                c12[0] += t;
                c12[1] += t * h[i];
                sw[v][i] += g[i] * h[i];
                sb[v][i] += g[i];
            }
        }
        row_sums<G>(c12, scratch[turn]);
        turn ^= 1;
        if (gx && live) {
            const float c1 = c12[0] / (float)d, c2 = c12[1] / (float)d;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Place<N> at(v * G + lane, d);
                if (at.skip >= N) continue;
                float g[8], h[8], t[8];
                Vec<T>::unpack(a.g[v], g);
                Vec<T>::unpack(a.x[v], h);
                if (SUM) Vec<T>::unpack(a.gs[v], t);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    h[i] = (h[i] - a.mean) * a.rstd;
                    g[i] = a.rstd * (g[i] * wf[v][i] - c1 - h[i] * c2);
                    if (SUM) g[i] += t[i];
                }
                store_row<ONCE>(gx + row * d + at.from, Vec<T>::pack(g));
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t first = (int64_t)blockIdx.x * kRows;
    RowData<V> a;
    if constexpr (kAhead) {
        // (two sets' registers that change places, not one copied over the other, which would wait for its loads)
        RowData<V> b;
        load(first + mine, a);
        while (true) {
            load(first + step + mine, b);
            use(first + mine, a);
            first += step;
            if (first >= rows) break;
            load(first + step + mine, a);
            use(first + mine, b);
            first += step;
            if (first >= rows) break;
        }
    } else {
        for (; first < rows; first += step) {
            load(first + mine, a);
            use(first + mine, a);
        }
    }
    if (!part) return;
    float *out = part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
    for (int which = 0; which < 2; ++which, out += d) {
        if constexpr (kRows == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Place<N> at(v * G + lane, d);
                if (at.skip == 0) {
                    __builtin_memcpy(out + at.from, which ? sb[v] : sw[v], N * sizeof(float));
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (at.own(i)) out[at.from + i] = which ? sb[v][i] : sw[v][i];
                }
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) sums[(mine * V + v) * G * N + i * G + lane] = which ? sb[v][i] : sw[v][i];
            __syncthreads();
            // (a column's place: its vector's number, then which of the vector's elements, then the lane)
            for (int c = threadIdx.x; c < d; c += kThreads) {
                const int vec = c / N, place = vec / G * G * N + (c - Place<N>(vec, d).from) * G + vec % G;
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

// Sums over a range of rows each, a column to each thread: part[range] holds grad_w's d sums and then grad_b's.  One thread adds up to rows / 128 terms, 16
// million of the most rows, so it does in float64 (8 million rows of three 0.1s: float32 is off by 6e-4).
template <typename T>
__global__ __launch_bounds__(kBlock) void long_param_kernel(const T *__restrict__ gy, int64_t gy_stride, const T *__restrict__ x,
                                                            int64_t x_stride, const float *__restrict__ mean,
                                                            const float *__restrict__ rstd, float *__restrict__ part, int64_t rows,
                                                            int64_t d) {
    const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= d) return;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * per, hi = lo + per < rows ? lo + per : rows;
    double sw = 0, sb = 0;
    for (int64_t t = lo; t < hi; ++t) {
        const float g = (float)gy[t * gy_stride + c];
        sw += g * ((float)x[t * x_stride + c] - mean[t]) * rstd[t];
        sb += g;
    }
    part[(int64_t)blockIdx.y * 2 * d + c] = (float)sw;
    part[(int64_t)blockIdx.y * 2 * d + d + c] = (float)sb;
}

// grad_w and grad_b out of the parts, in their order: 32 columns to a workgroup, 16 ranges of parts side by side
constexpr int kSumCols = 32, kSumRanges = 16, kSumBlock = kSumCols * kSumRanges;
template <typename P>
__global__ __launch_bounds__(kSumBlock) void norm_param_sum_kernel(const float *__restrict__ part, int n_parts, P *__restrict__ gw,
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
    if (d < N || d > (int64_t)G * V * N) return false;
    f(std::integral_constant<int, G>{}, std::integral_constant<int, V>{});
    return true;
}
// one_each: one vector to a lane where two would do too, for rows with a residual (two loads in flight already: 16384 x 4096 bfloat16 93 us against 99) and
// launches of fewer than kFewRows rows (64 x 4096: 4.0 against 4.4); else two (32768 x 4096: 102 us against 122; 32768 x 1024: 27 against 31).
template <int N, typename F> bool held_forward(int64_t d, bool one_each, F &&f) {
    if (held_by<N, 8, 1>(d, f) || held_by<N, 32, 1>(d, f) || held_by<N, 64, 1>(d, f)) return true;
    if (one_each ? held_by<N, 128, 1>(d, f) || held_by<N, 256, 1>(d, f) || held_by<N, 512, 1>(d, f)
                 : held_by<N, 64, 2>(d, f) || held_by<N, 128, 2>(d, f) || held_by<N, 256, 2>(d, f))
        return true;
    return held_by<N, 512, 2>(d, f) || held_by<N, 1024, 2>(d, f) || held_by<N, 1024, 4>(d, f);
}
template <int N, typename F> bool held_backward(int64_t d, F &&f) {
    if (held_by<N, 8, 1>(d, f) || held_by<N, 32, 1>(d, f) || held_by<N, 64, 1>(d, f) || held_by<N, 128, 1>(d, f) || held_by<N, 256, 1>(d, f) ||
        held_by<N, 512, 1>(d, f) || held_by<N, 1024, 1>(d, f))
        return true;
    if constexpr (N == 4) return held_by<N, 512, 4>(d, f) || held_by<N, 512, 8>(d, f);
    else return held_by<N, 1024, 2>(d, f);
}

// Ranges of the rows, as a launch counts its threads, `lanes` to a row, in 32 bits: f(first row, rows)
constexpr int64_t kLaunchThreads = INT64_C(1) << 31;
template <typename F> void in_launches(int64_t rows, int lanes, F &&f) {
    const int64_t most = kLaunchThreads / lanes;
    for (int64_t at = 0; at < rows; at += most) f(at, rows - at < most ? rows - at : most);
}
template <typename T> T *behind(T *p, int64_t elems) { return p ? p + elems : p; }

constexpr int kLongParts = 128;
int n_parts(int64_t rows) { return (int)(rows < 1 ? 1 : rows < kBwdMostBlocks ? rows : kBwdMostBlocks); }

int check(const char *who, int64_t rows, int64_t d, int dtype, int param_dtype) {
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who,
                 dtype);
    FMOE_REQUIRE(param_dtype == dtype || param_dtype == FMOE_F32, "%s: parameters must be of the rows' type or float32", who);
    FMOE_REQUIRE(rows >= 0 && d >= 1, "%s: bad sizes", who);
    if (rows > (int64_t)INT32_MAX || d > (int64_t)(1 << 26)) return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
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
        const bool param_f32 = std::is_same<P, float>::value;
        const bool held = held_forward<Vec<T>::N>(row_elems, residual || rows < kFewRows, [&](auto g, auto v) {
            constexpr int kThreads = g.value > kBlock ? g.value : kBlock;
            in_launches(rows, g.value, [&](int64_t at, int64_t n) {
                norm_fwd_kernel<T, g.value, v.value><<<(int)ceil_div(n, kThreads / g.value), kThreads, 0, st>>>(
                    (const T *)x + at * x_stride, x_stride, behind((const T *)residual, at * residual_stride), residual_stride, Param{weight, param_f32},
                    Param{bias, param_f32}, behind((T *)sum, at * row_elems), (T *)y + at * row_elems, behind(mean, at), behind(rstd, at), n, (int)row_elems,
                    (float)eps);
            });
        });
        if (!held)
            in_launches(rows, kBlock, [&](int64_t at, int64_t n) {
                long_fwd_kernel<T, P><<<(int)n, kBlock, 0, st>>>((const T *)x + at * x_stride, x_stride, behind((const T *)residual, at * residual_stride),
                                                                 residual_stride, (const P *)weight, (const P *)bias, behind((T *)sum, at * row_elems),
                                                                 (T *)y + at * row_elems, behind(mean, at), behind(rstd, at), row_elems, (float)eps);
            });
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
        // (rows that the memory-side cache could not hold go past the caches: nobody reads them again, 16384 x 4096 103 us through them, 95 past;
        // smaller launches lose by it: 4096 x 8192 53 and 55; 65536 x 512 50 and 54.  Without rows there is nothing to load from, and the parameters' gradients are sums of no parts)
        int parts = 0;
        const bool held = rows == 0 || held_backward<Vec<T>::N>(row_elems, [&](auto g, auto v) {
            // (one set to a workgroup, unless the workgroups' sums would be more than kPartBytes, then two.  One and two, us, of sums of 1.0 MB (64 x 4096
            // bfloat16) 8.7 and 9.6, 1.9 MB (777 x 1302) 10.4 and 11.1, (1000 x 1024 float32) 8.4 and 9.2, 3.1 MB (200 x 4096 bfloat16) 11.2 and 11.0,
            // 6.3 MB (100 x 8192) 11.9 and 10.9, 8.0 MB (509 x 4096 float16) 14.7 and 12.1, (128 x 8192 float32) 12.3 both, 18.8 MB (300 x 8192 bfloat16) 15.6 and 14.2)
            const int64_t sets = ceil_div(rows, bwd_threads(v.value) / g.value);
            const int64_t blocks = params && sets * 8 * row_elems > kPartBytes ? ceil_div(sets, 2) : sets;
            parts = (int)(blocks < kBwdMostBlocks ? blocks : kBwdMostBlocks);
            const bool once = rows * row_elems * (int64_t)sizeof(T) * (grad_sum ? 4 : 3) > kCacheBytes;
            auto kernel = once ? (grad_sum ? norm_bwd_kernel<T, g.value, v.value, true, true> : norm_bwd_kernel<T, g.value, v.value, true, false>)
                               : (grad_sum ? norm_bwd_kernel<T, g.value, v.value, false, true> : norm_bwd_kernel<T, g.value, v.value, false, false>);
            kernel<<<parts, bwd_threads(v.value), 0, st>>>((const T *)grad_y, grad_y_stride, (const T *)grad_sum, grad_sum_stride, (const T *)x, x_stride, mean,
                                           rstd, Param{weight, std::is_same<P, float>::value}, (T *)grad_x,
                                           params ? (float *)workspace : nullptr, rows, (int)row_elems);
        });
        if (!held) {
            parts = n_parts(rows) < kLongParts ? n_parts(rows) : kLongParts;
            if (grad_x)
                in_launches(rows, kBlock, [&](int64_t at, int64_t n) {
                    long_bwd_kernel<T, P><<<(int)n, kBlock, 0, st>>>((const T *)grad_y + at * grad_y_stride, grad_y_stride,
                                                                     behind((const T *)grad_sum, at * grad_sum_stride), grad_sum_stride,
                                                                     (const T *)x + at * x_stride, x_stride, mean + at, rstd + at, (const P *)weight,
                                                                     (T *)grad_x + at * row_elems, row_elems);
                });
            if (params)
                long_param_kernel<T><<<dim3((int)ceil_div(row_elems, kBlock), parts), kBlock, 0, st>>>(
                    (const T *)grad_y, grad_y_stride, (const T *)x, x_stride, mean, rstd, (float *)workspace, rows, row_elems);
        }
        if (params)
            norm_param_sum_kernel<P><<<(int)ceil_div(2 * row_elems, kSumCols), kSumBlock, 0, st>>>((const float *)workspace, parts, (P *)grad_weight,
                                                                                               (P *)grad_bias, row_elems);
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
