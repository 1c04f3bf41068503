// The experts' product of rows and weights in 8-bit integers, each row and each output channel under a scale of its own (gfx950):
//
//   y[r, c] = act(s_r t_c sum_k q[r, k] w[c, k] + b[c])         gated: act(the same of Wg, bg) (the same of Wu, bu)
//
// The sums are 32-bit integers and exact; one rounding makes them float32, the scales, the bias and the activation are float32, one more rounding makes the
// result.  v_mfma_i32_16x16x64_i8 takes 16 bytes of a row per lane, as the 16-bit forms do, so slabs of 128 bytes, their LDS image and its swizzle are those of
// gemm_kernel.hpp.
//
// The kernels are those of 16-bit types (gemm_kernel.hpp, gemm_ring.hpp, gemm_skinny.hip); this file holds the call.  Few rows are bound by the weights' way from memory
// (64 sequences of two experts each, 8 experts of 4096 -> 2 x 14336: 165 us, 5.7 TB/s), many by the matrix pipe and at last by the card's power (32768 rows there:
// 2.93 ms, 2620 TOP/s; of zeros 3560), between them by a last round of tiles that is partly filled (8192 rows, 16 experts of 2048 -> 2048: 56 us, 1220).
#include "gemm_int8.hpp"
#include "gated_terms.hpp"

using namespace fmoe;

namespace {
Int8Params sizes(int64_t n_expert, int64_t rows_cap, int64_t in_feat, int64_t out_feat, int gated, int dtype) {
    Int8Params prm{};
    prm.n_expert = n_expert; prm.rows_cap = rows_cap; prm.n_cols = (int)out_feat; prm.k_extent = (int)(ceil_div(in_feat, 16) * 16);
    prm.gated = gated != 0; prm.dtype = dtype; prm.in_feat = in_feat;
    return prm;
}
bool sizes_known(int64_t n_expert, int64_t rows_cap, int64_t in_feat, int64_t out_feat) {
    return n_expert >= 1 && rows_cap >= 1 && in_feat >= 1 && in_feat <= 131072 && out_feat >= 1 && out_feat <= (1 << 28);
}
// (131072 products of numbers up to 128: below 2^31; a tile's rows within 2 GiB of its first)
bool features_taken(int64_t in_feat, int64_t out_feat, int64_t w_rows, int64_t ldw, int dtype) {
    return in_feat <= 131072 && out_feat <= (1 << 28) && ldw <= (1 << 22) && w_rows * ldw < ((int64_t)1 << 31) && out_feat * dtype_bytes(dtype) <= (1 << 22);
}
}  // namespace

extern "C" int fmoe_linear_int8_supported(int64_t in_feat, int64_t out_feat, int gated, int dtype) {
    return (dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16) && in_feat >= 1 && out_feat >= 1 &&
           features_taken(in_feat, out_feat, out_feat * (gated ? 2 : 1), ceil_div(in_feat, 16) * 16, dtype);
}

extern "C" int fmoe_linear_int8(const void *x, int64_t ldx, const void *x_scale, const int64_t *row_index, int64_t index_div, int64_t x_rows, const void *w, int64_t ldw, int64_t w_expert_stride,
                                const void *w_scale, const void *bias, void *y, const void *segment_table, int64_t n_expert, int64_t rows_cap,
                                int64_t in_feat, int64_t out_feat, int gated, int activation, int dtype, void *workspace, int64_t workspace_bytes,
                                void *stream) {
    const char *who = "fmoe_linear_int8";
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who, dtype);
    FMOE_REQUIRE(is_gate_activation(activation), "%s: unknown activation %d", who, activation);
    FMOE_REQUIRE(n_expert >= 1 && rows_cap >= 0 && in_feat >= 1 && out_feat >= 1, "%s: bad sizes", who);
    const int64_t whole = ceil_div(in_feat, 16) * 16, w_rows = out_feat * (gated ? 2 : 1);
    if (n_expert > (1 << 24) || rows_cap > (int64_t)INT32_MAX - 65536 || (x_scale != nullptr && ldx > (1 << 22)) || !features_taken(in_feat, out_feat, w_rows, ldw, dtype))
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    FMOE_REQUIRE((x_scale == nullptr || (ldx >= whole && ldx % 16 == 0)) && ldw >= whole && ldw % 16 == 0 && w_expert_stride % 16 == 0 && w_expert_stride >= 0,
                 "%s: rows of 8-bit integers begin on 16 bytes, at least %lld apart", who, (long long)whole);
    if (rows_cap == 0) return FMOE_OK;
    Int8Params prm = sizes(n_expert, rows_cap, in_feat, out_feat, gated, dtype);
    FMOE_REQUIRE(x_scale != nullptr || int8_rounds_rows(prm), "%s: rows of these sizes come in 8-bit integers with x_scale", who);
    FMOE_REQUIRE(x_scale == nullptr || row_index == nullptr, "%s: row_index goes with rows that are not rounded yet", who);
    FMOE_REQUIRE(x_scale != nullptr || (index_div >= 1 && x_rows >= 0 && (row_index != nullptr || x_rows >= rows_cap)), "%s: bad rows", who);
    FMOE_REQUIRE((x || (x_scale == nullptr && x_rows == 0)) && w && w_scale && y && segment_table, "%s: NULL pointer", who);
    FMOE_REQUIRE((x_scale == nullptr || aligned16(x)) && aligned16(w) && aligned16(segment_table) && aligned16(y) && aligned16(w_scale) && (bias == nullptr || aligned16(bias)),
                 "%s: tensors begin on 16 bytes", who);
    prm.x = x; prm.w = (const int8_t *)w; prm.x_scale = (const float *)x_scale; prm.w_scale = (const float *)w_scale;
    prm.bias = bias; prm.y = y; prm.ldx = ldx; prm.ldw = ldw; prm.w_expert_stride = w_expert_stride;
    prm.row_index = row_index; prm.index_div = index_div; prm.x_rows = x_rows;
    prm.activation = activation; prm.dev_tab = (const int32_t *)segment_table;
    return launch_int8(prm, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int fmoe_linear_int8_rounds_rows(int64_t n_expert, int64_t rows_cap, int64_t in_feat, int64_t out_feat, int gated, int dtype) {
    return sizes_known(n_expert, rows_cap, in_feat, out_feat) && int8_rounds_rows(sizes(n_expert, rows_cap, in_feat, out_feat, gated, dtype));
}

extern "C" int64_t fmoe_linear_int8_workspace_bytes(int64_t n_expert, int64_t rows_cap, int64_t in_feat, int64_t out_feat, int gated, int dtype) {
    return sizes_known(n_expert, rows_cap, in_feat, out_feat) ? int8_workspace_bytes(sizes(n_expert, rows_cap, in_feat, out_feat, gated, dtype)) : 0;
}
