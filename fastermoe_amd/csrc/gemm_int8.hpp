// Interface of the experts' products in 8-bit integers.
#pragma once
#include "grouped_gemm.hpp"

namespace fmoe {

// y[r, c] = act(s_r t_c sum_k x[r, k] w[c, k] + bias[c]) of each expert's rows; gated: w has 2 n_cols rows a gate's and then its linear half's,
// y[r, c] = act(first) second.
struct Int8Params {
    const void *x;                // rows of ldx bytes, zeros from the contraction's end to whole 16 bytes
    const int8_t *w;              // rows of ldw bytes
    const float *x_scale, *w_scale;
    // x_scale null (int8_rounds_rows): x is of y's type, rows of in_feat elements ldx apart, x_rows of them, taken as fmoe_quantize_rows does; rows of y
    // behind the table's become zeros
    const int64_t *row_index;
    int64_t index_div, x_rows, in_feat;
    const void *bias;             // [E, columns] of y's type, or null
    void *y;                      // [rows, n_cols]
    int64_t ldx, ldw, w_expert_stride;   // bytes, multiples of 16
    int32_t n_cols, k_extent;     // k_extent: bytes of contraction, a multiple of 16
    int32_t gated, activation;
    const int32_t *dev_tab;       // segtab layout
    int64_t n_expert, rows_cap;
    int dtype;                    // of y
};

// The kernels of 16-bit types with pairs of integers in their elements' places (grouped_gemm.hip): the workspace, which is not needed but used to share a last round's
// tiles, and the launch.
bool int8_rounds_rows(const Int8Params &a);
int64_t int8_workspace_bytes(const Int8Params &a);
int launch_int8(const Int8Params &a, void *workspace, int64_t workspace_bytes, hipStream_t stream);

}  // namespace fmoe
