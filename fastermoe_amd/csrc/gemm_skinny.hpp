// Interface of gemm_skinny.hip: the grouped forward product for few rows per expert.
#pragma once
#include "gemm_kernel.hpp"

namespace fmoe {
namespace gemm {

struct SkinnyParams {
    const void *w, *x, *bias;     // [E, n_cols, k], rows of k, [E, n_cols] or null
    void *y, *aux;                // [rows, n_cols]; aux: the pre-activation, or null
    const int32_t *dev_tab;       // segtab layout
    const int64_t *row_index;     // as GemmParams::q_row_index, with its divisor
    int64_t x_total_rows;
    uint32_t div_mul;
    int32_t div_shift;
    int32_t n_cols, k_extent, activation;
    int32_t weights_cached;       // not 0: the weights through the caches, see caches_few_row_weights() in grouped_gemm.hip
    int32_t order_off, tiles_n, extra_groups;   // set by the launch: the table's list of experts (or its map of row tiles), see launch()
};
// Gated products and such in 8-bit integers (w: [E, 2 n_cols or n_cols, k], a gate's rows first; aux [rows, 2 n_cols] float32).  A type of its own: plain
// products of a few rows feel how long a launch's arguments are (1 row, 2048 experts of 512 x 512, in a graph: 3.72 us; with these between theirs 3.82).
struct SkinnyMoreParams : SkinnyParams {
    int64_t ldw, ldx, w_expert_stride;         // 8-bit integers: row strides in pairs of them (others are dense)
    const float *w_scale, *x_scale;            // 8-bit integers: of each row of w and of x; x_scale null: x in y's type, to be rounded here
    int64_t index_div;                         // rows to be rounded: row_index's divisor, elements of a row (ldx apart)
    int32_t x_elems;
    void *tail;                                // gated, or rows to be rounded: rows of tail_elems elements behind the table's, up to tail_rows, become zeros (null: none)
    int64_t tail_rows, tail_elems;
};

// Rows that the launch in 8-bit integers rounds itself: at most this many, of at most this many elements in all (a row's rounded up to sixteen).  Each workgroup rounds all
// of its expert's rows, while its first weights are on their way.  us in a launch of their own and here, in a graph, weights from memory: 32 experts of 1024 -> 4096, 2
// rows: 6.6 / 5.2, 8 rows: 11.5 / 8.7, all 8 one expert's: 6.7 / 6.8; 8 of 4096 -> 2 x 14336, gated, 2 rows: 40.0 / 37.1; 64 of 512 -> 2 x 2048, gated, 16 rows: 13.4 /
// 10.8, all one expert's: 6.3 / 7.1; 1 row of 8192 -> 8192: 24.7 / 20.8.
constexpr int kSkinnyRoundRows = 16, kSkinnyRoundElems = 8192;

// rows_cap: the rows that the table was laid out for
int launch_skinny(const SkinnyParams &prm, int dtype, int64_t rows_cap, int64_t n_expert, hipStream_t stream);
// gated forward, 16-bit types
int launch_skinny_gated(const SkinnyMoreParams &prm, int dtype, int64_t rows_cap, int64_t n_expert, hipStream_t stream);
// rows and weights in 8-bit integers, k_extent in pairs, dtype of the results, whose columns are a multiple of four
int launch_skinny_int8(const SkinnyMoreParams &prm, int dtype, bool gated, int64_t rows_cap, int64_t n_expert, hipStream_t stream);

// Rows off the 16-byte grid, 16-bit types (gemm_few_unaligned.hip): the plain or the gated forward product
int launch_few_unaligned(const SkinnyMoreParams &prm, int dtype, bool gated, int64_t rows_cap, int64_t n_expert, hipStream_t stream);

// Two loads of 128 bytes of rows 0 to 7 and 8 to 15 (lane: row lane % 8, bit 3: half of the line) become the operands of two
// steps (lane: row lane % 16, chunk lane / 16 of the step's 64 bytes): the lanes with bit 3 set give the first load's second chunks
// for the second load's first.
__device__ __forceinline__ void pair_to_steps(u32x4 &a, u32x4 &b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = a[i], hi = b[i];   // (row_ror 8 within 16 lanes, written to the upper or to the lower eight)
        a[i] = __builtin_amdgcn_update_dpp(lo, hi, 0x128, 0xf, 0xc, false);
        b[i] = __builtin_amdgcn_update_dpp(hi, lo, 0x128, 0xf, 0x3, false);
    }
}

}  // namespace gemm
}  // namespace fmoe
