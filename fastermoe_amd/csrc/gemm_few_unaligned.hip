// Grouped forward product Y[seg_e] = X[seg_e] . W_e^T + b_e, plain or gated (act(first half) times the second), for few rows per expert of 16-bit types whose feature
// sizes or pointers are off the 16-byte grid, over a device segment table (gfx950): gemm_skinny.hip's part where its loads, which begin on dwords, cannot go.
//
// A workgroup of four waves has 32 columns (gated: 16 of each half) of one expert and its rows, sixteen at a time.  The waves take the contraction in turns of 64
// elements, four of those on their way at a time (gemm_unaligned.hip has one, and a tile's slabs come one after the other: 1.2 us each, however few rows there are),
// and add up their accumulators through LDS in a fixed order.  A load takes 16 bytes from wherever they begin; the contraction's last, partial 64 elements are read as
// the eight that end with it and moved down.  Bound by the weights' way from memory, or, of small weights, by a few waits for it.
//
// Rows that begin between two dwords (half of them where the contraction is odd) are read as the five dwords that hold eight elements, and shifted into place: 16-byte loads
// from there take many times as long as from a dword (8 experts of 4095 -> 2 x 4097, one row each, 537 MB: 274 us with them, 124 now, 4.3 TB/s).  Where it is used, and what it measured: few_unaligned() in grouped_gemm.hip.
#include "gemm_skinny.hpp"
#include "segment_table.hpp"
#include "unaligned_loads.hpp"

namespace fmoe {
namespace gemm {
namespace {

constexpr int kFewWaves = 4, kFewThreads = 64 * kFewWaves, kFewLine = 64;

// Eight elements on their way.  ODD: rows may begin between two dwords, and are read as the five dwords that hold them: the last of those may lie past the row's end, in the
// dword of the row's last element.
template <bool ODD> struct Chunk {
    u32x4 v;
    uint32_t last;
};
template <typename T, bool ODD> struct Row {
    const T *p;      // ODD: the dword that holds the first element
    uint32_t shift;  // ODD: bits to the first element
    __device__ __forceinline__ explicit Row(const T *first) : p(first), shift(0) {
        if constexpr (ODD) {
            shift = ((uintptr_t)first & 2) * 8;
            p = (const T *)((uintptr_t)first & ~(uintptr_t)3);
        }
    }
    Row() = default;
    __device__ __forceinline__ void load(Chunk<ODD> &c, int k) const {
        c.v = load_dwords(p + k);
        if constexpr (ODD) c.last = *(const uint32_t *)(p + k + 6 + shift / 8);   // (no shift: the fourth again)
    }
    __device__ __forceinline__ u32x4 elements(const Chunk<ODD> &c) const {
        if constexpr (!ODD) return c.v;
        else
            return u32x4{__builtin_amdgcn_alignbit(c.v[1], c.v[0], shift), __builtin_amdgcn_alignbit(c.v[2], c.v[1], shift),
                         __builtin_amdgcn_alignbit(c.v[3], c.v[2], shift), __builtin_amdgcn_alignbit(c.last, c.v[3], shift)};
    }
    __device__ __forceinline__ const T *first() const { return p + shift / 16; }
};

template <typename T, bool HALVES, bool ODD>
__global__ __launch_bounds__(kFewThreads) void grouped_gemm_few_unaligned_kernel(const SkinnyMoreParams prm) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass only needs the launch stub
    constexpr int kCols = HALVES ? 16 : 32;
    typedef const int32_t __attribute__((address_space(4))) *DevTab;    // read-only, uniform: scalar loads
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef const i32x4 __attribute__((address_space(4))) *DevTab4;
    __shared__ f32x4 part[kFewWaves - 1][2][64];
    const DevTab dtab = (DevTab)(uintptr_t)prm.dev_tab;
    if constexpr (HALVES) {
        const int64_t there = dtab[segtab::kRows];
        if (prm.tail != nullptr && there < prm.tail_rows)
            for (int64_t i = (int64_t)blockIdx.x * kFewThreads + threadIdx.x; i < (prm.tail_rows - there) * prm.tail_elems; i += (int64_t)gridDim.x * kFewThreads)
                ((T *)prm.tail)[there * prm.tail_elems + i] = (T)0.f;
    }
    const int place = __builtin_amdgcn_readfirstlane(blockIdx.x / prm.tiles_n), tile_n = blockIdx.x - place * prm.tiles_n;
    if (place >= dtab[segtab::kTiles128]) return;
    const i32x4 entry = ((DevTab4)(dtab + prm.order_off))[place];   // {expert, first row, rows}, at most 128 rows
    const int expert = entry[0], first = entry[1], rows = entry[2];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n0 = tile_n * kCols, K = prm.k_extent, n_cols = prm.n_cols;
    const int lb = lane & 15, hq = lane >> 4;
    // A load takes 128 bytes of eight rows, this lane 16 bytes of row lane % 8 (see pair_to_steps)
    const int chunk = (hq | ((lane & 8) >> 1)) * 8, row8 = lane & 7;

    // columns past the last repeat it, as rows do; neither is stored
    const T *W = (const T *)prm.w + (int64_t)expert * (HALVES ? 2 : 1) * n_cols * K;
    Row<T, ODD> w_row[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int col = min(n0 + (HALVES ? 0 : 16 * n) + 8 * h + row8, n_cols - 1) + (HALVES && n ? n_cols : 0);
            w_row[n][h] = Row<T, ODD>(W + (int64_t)col * K);
        }
    const int n_lines = K / kFewLine, rest = K - n_lines * kFewLine;
    const int mine = n_lines > wave ? (n_lines - wave + kFewWaves - 1) / kFewWaves : 0;   // whole lines of this wave
    const bool has_rest = rest > 0 && wave == n_lines % kFewWaves, back = K >= 8;

    constexpr int kFewAhead = ODD ? 3 : 4;   // (what the registers of two waves a SIMD hold)
    struct Line { Chunk<ODD> w[2][2], x[2]; };
    for (int r0 = 0; r0 < rows; r0 += 16) {
        Row<T, ODD> x_row[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) x_row[h] = Row<T, ODD>((const T *)prm.x + (int64_t)(first + min(r0 + 8 * h + row8, rows - 1)) * K);
        f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        auto load = [&](Line &u, int i) __attribute__((always_inline)) {   // (past the wave's last line: that one again, which nothing multiplies)
            const int k = (wave + kFewWaves * min(i, mine - 1)) * kFewLine + chunk;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) w_row[n][h].load(u.w[n][h], k);
#pragma unroll
            for (int h = 0; h < 2; ++h) x_row[h].load(u.x[h], k);
        };
        auto multiply_all = [&](u32x4 (&w)[2][2], u32x4 (&x)[2]) __attribute__((always_inline)) {
            pair_to_steps(x[0], x[1]);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                pair_to_steps(w[n][0], w[n][1]);
#pragma unroll
                for (int s = 0; s < 2; ++s) Elem<T>::mma(acc[n], w[n][s], x[s]);
            }
        };
        auto multiply = [&](const Line &u) __attribute__((always_inline)) {
            u32x4 w[2][2], x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[h] = x_row[h].elements(u.x[h]);
#pragma unroll
                for (int n = 0; n < 2; ++n) w[n][h] = w_row[n][h].elements(u.w[n][h]);
            }
            multiply_all(w, x);
        };
        if (mine > 0) {
            Line u[kFewAhead];
#pragma unroll
            for (int j = 0; j < kFewAhead; ++j) {
                load(u[j], j);
                __builtin_amdgcn_sched_barrier(0);
            }
            int i = 0;
            for (; i + kFewAhead <= mine; i += kFewAhead) {
#pragma unroll
                for (int j = 0; j < kFewAhead; ++j) {
                    multiply(u[j]);
                    load(u[j], i + j + kFewAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int j = 0; j + 1 < kFewAhead; ++j)
                if (i + j < mine) multiply(u[j]);
        }
        if (has_rest) {
            const int k = n_lines * kFewLine + chunk, left = K - k;
            u32x4 w[2][2], x[2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) w[n][h] = load_part(w_row[n][h].first() + k, w_row[n][h].first(), left, back);
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = load_part(x_row[h].first() + k, x_row[h].first(), left, back);
            multiply_all(w, x);
        }
        // the waves' sums in ascending order
        __syncthreads();   // (the rows before have been added up)
        if (wave > 0) {
#pragma unroll
            for (int n = 0; n < 2; ++n) part[wave - 1][n][lane] = acc[n];
        }
        __syncthreads();
        if (wave > 0) continue;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int w = 0; w + 1 < kFewWaves; ++w) acc[n] = add_parts<T>(acc[n], part[w][n][lane]);
        // acc[n][i] is C(row lb, column 16 n + 4 hq + i), gated: of half n, column 4 hq + i
        if (r0 + lb >= rows) continue;
        const int64_t row = first + r0 + lb;
        const T *bias = prm.bias ? (const T *)prm.bias + (int64_t)expert * (HALVES ? 2 : 1) * n_cols : nullptr;
        T *y = (T *)prm.y + row * n_cols;
        float *pre = HALVES && prm.aux ? (float *)prm.aux + row * 2 * n_cols : nullptr;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (HALVES) {
                const int col = n0 + 4 * hq + i;
                if (col >= n_cols) continue;
                const float g = acc[0][i] + (bias ? (float)bias[col] : 0.f), u = acc[1][i] + (bias ? (float)bias[n_cols + col] : 0.f);
                if (pre != nullptr) {
                    pre[col] = g;
                    pre[n_cols + col] = u;
                }
                y[col] = (T)(gate_act<true>(g, prm.activation) * u);
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int col = n0 + 16 * n + 4 * hq + i;
                    if (col < n_cols) y[col] = (T)(acc[n][i] + (bias ? (float)bias[col] : 0.f));
                }
            }
        }
    }
#endif
}

template <typename T, bool HALVES> int launch(const SkinnyMoreParams &params, int64_t rows_cap, int64_t n_expert, hipStream_t stream) {
    SkinnyMoreParams prm = params;
    prm.order_off = (int32_t)segtab::map128_off(rows_cap, n_expert);
    prm.tiles_n = (int)ceil_div(prm.n_cols, HALVES ? 16 : 32);
    const int64_t grid = segtab::cap_tiles(rows_cap, n_expert, 128) * prm.tiles_n;
    if (grid > (int64_t)INT32_MAX) return fail(FMOE_ELIMIT, "grouped GEMM: grid of %lld workgroups", (long long)grid);
    const bool odd = (prm.k_extent & 1) || (((uintptr_t)prm.x | (uintptr_t)prm.w) & 2);
    if (odd) grouped_gemm_few_unaligned_kernel<T, HALVES, true><<<(unsigned)grid, kFewThreads, 0, stream>>>(prm);
    else grouped_gemm_few_unaligned_kernel<T, HALVES, false><<<(unsigned)grid, kFewThreads, 0, stream>>>(prm);
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

}  // namespace

int launch_few_unaligned(const SkinnyMoreParams &prm, int dtype, bool gated, int64_t rows_cap, int64_t n_expert, hipStream_t stream) {
    FMOE_REQUIRE(dtype == FMOE_BF16 || dtype == FMOE_F16, "grouped GEMM: dtype %d is not a 16-bit float type", dtype);
    if (dtype == FMOE_BF16) return gated ? launch<__bf16, true>(prm, rows_cap, n_expert, stream) : launch<__bf16, false>(prm, rows_cap, n_expert, stream);
    return gated ? launch<_Float16, true>(prm, rows_cap, n_expert, stream) : launch<_Float16, false>(prm, rows_cap, n_expert, stream);
}

}  // namespace gemm
}  // namespace fmoe
