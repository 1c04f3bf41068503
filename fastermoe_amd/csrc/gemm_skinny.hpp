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
    // Gated products and such in 8-bit integers (w: [E, 2 n_cols or n_cols, k], a gate's rows first; aux [rows, 2 n_cols]):
    int64_t ldw, ldx, w_expert_stride;         // 8-bit integers: row strides in pairs of them (others are dense)
    const float *w_scale, *x_scale;            // 8-bit integers: of each row of w and of x
    void *tail;                                // gated: rows of tail_elems 16-bit elements behind the table's, up to tail_rows, become zeros (null: none)
    int64_t tail_rows, tail_elems;
    int32_t order_off, tiles_n, extra_groups;   // set by the launch: the table's list of experts (or its map of row tiles), see launch()
};

// rows_cap: the rows that the table was laid out for
int launch_skinny(const SkinnyParams &prm, int dtype, int64_t rows_cap, int64_t n_expert, hipStream_t stream);
// gated forward, 16-bit types
int launch_skinny_gated(const SkinnyParams &prm, int dtype, int64_t rows_cap, int64_t n_expert, hipStream_t stream);
// rows and weights in 8-bit integers, k_extent in pairs, dtype of the results, whose columns are a multiple of four
int launch_skinny_int8(const SkinnyParams &prm, int dtype, bool gated, int64_t rows_cap, int64_t n_expert, hipStream_t stream);

}  // namespace gemm
}  // namespace fmoe
