// The experts' product of rows and weights in 8-bit integers, each row and each output channel under a scale of its own (gfx950):
//
//   y[r, c] = act(s_r t_c sum_k q[r, k] w[c, k] + b[c])         gated: act(the same of Wg, bg) (the same of Wu, bu)
//
// The sums are 32-bit integers and exact; one rounding makes them float32, the scales, the bias and the activation are float32, one more rounding makes the
// result.  v_mfma_i32_16x16x64_i8 takes 16 bytes of a row per lane, as the 16-bit forms do, so slabs of 128 bytes, their LDS image and its swizzle are those of
// gemm_kernel.hpp.
//
// The kernels are those of 16-bit types (gemm_kernel.hpp, gemm_ring.hpp, gemm_skinny.hip); this file holds the call.
#include "gemm_int8.hpp"
#include "gated_terms.hpp"

using namespace fmoe;

extern "C" int fmoe_linear_int8(const void *x, int64_t ldx, const void *x_scale, const void *w, int64_t ldw, int64_t w_expert_stride,
                                const void *w_scale, const void *bias, void *y, const void *segment_table, int64_t n_expert, int64_t rows_cap,
                                int64_t in_feat, int64_t out_feat, int gated, int activation, int dtype, void *workspace, int64_t workspace_bytes,
                                void *stream) {
    const char *who = "fmoe_linear_int8";
    FMOE_REQUIRE(dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who, dtype);
    FMOE_REQUIRE(is_gate_activation(activation), "%s: unknown activation %d", who, activation);
    FMOE_REQUIRE(n_expert >= 1 && rows_cap >= 0 && in_feat >= 1 && out_feat >= 1, "%s: bad sizes", who);
    const int64_t whole = ceil_div(in_feat, 16) * 16, w_rows = out_feat * (gated ? 2 : 1);
    // (131072 products of numbers up to 128: below 2^31)
    if (in_feat > 131072 || n_expert > (1 << 24) || rows_cap > (int64_t)INT32_MAX - 65536 || out_feat > (1 << 28) || ldx > (1 << 22) ||
        ldw > (1 << 22) || w_rows * ldw >= ((int64_t)1 << 31))
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    FMOE_REQUIRE(ldx >= whole && ldw >= whole && ldx % 16 == 0 && ldw % 16 == 0 && w_expert_stride % 16 == 0 && w_expert_stride >= 0,
                 "%s: rows of 8-bit integers begin on 16 bytes, at least %lld apart", who, (long long)whole);
    if (rows_cap == 0) return FMOE_OK;
    FMOE_REQUIRE(x && x_scale && w && w_scale && y && segment_table, "%s: NULL pointer", who);
    FMOE_REQUIRE(aligned16(x) && aligned16(w) && aligned16(segment_table) && aligned16(y) && aligned16(w_scale) && (bias == nullptr || aligned16(bias)),
                 "%s: tensors begin on 16 bytes", who);
    Int8Params prm{};
    prm.x = (const int8_t *)x; prm.w = (const int8_t *)w; prm.x_scale = (const float *)x_scale; prm.w_scale = (const float *)w_scale;
    prm.bias = bias; prm.y = y; prm.ldx = ldx; prm.ldw = ldw; prm.w_expert_stride = w_expert_stride;
    prm.n_cols = (int)out_feat; prm.k_extent = (int)whole; prm.gated = gated != 0; prm.activation = activation;
    prm.dev_tab = (const int32_t *)segment_table; prm.n_expert = n_expert; prm.rows_cap = rows_cap; prm.dtype = dtype;
    return launch_int8(prm, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int64_t fmoe_linear_int8_workspace_bytes(int64_t n_expert, int64_t rows_cap, int64_t in_feat, int64_t out_feat, int gated, int dtype) {
    if (n_expert < 1 || rows_cap < 1 || in_feat < 1 || in_feat > 131072 || out_feat < 1 || out_feat > (1 << 28)) return 0;
    Int8Params prm{};
    prm.n_expert = n_expert; prm.rows_cap = rows_cap; prm.n_cols = (int)out_feat; prm.k_extent = (int)(ceil_div(in_feat, 16) * 16);
    prm.gated = gated != 0; prm.dtype = dtype;
    return int8_workspace_bytes(prm);
}
