// Gated experts (gfx950): per expert, over its rows,
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  m = act(g) u,  y = m W2^T + b2            (W1 = [Wg; Wu], its products [g u] = `pre`)
//   dm = dy W2,  dg = dm u act'(g),  du = dm act(g),  dx = [dg du] W1,  dW1 = [dg du]^T x,  dW2 = dy^T m
//
// This file holds the calls of the whole block and the two kernels between its products for the shapes whose product does not do their work in
// its epilogue.
#include "gated_terms.hpp"
#include "grouped_gemm.hpp"
#include "lane_elems.hpp"
#include "wave_piece.hpp"

#include <algorithm>
#include <type_traits>

namespace fmoe {
namespace {

constexpr int kBlock = 256, kLaneElems = 8;

// rows that there are: all of them, or those that the experts' segments take
__device__ __forceinline__ int64_t live_rows(const int32_t *table, int64_t rows) {
    if (!table) return rows;
    const int64_t n = table[segtab::kRows];
    return n < rows ? n : rows;
}

// A lane's eight elements of a row of h: row, first element, how many (0 or less: none).
struct Piece { int64_t row; int c, n; };
__device__ __forceinline__ Piece piece_of(int64_t rows, int h, uint32_t per_row) {
    const int64_t first = (int64_t)blockIdx.x * kBlock, row0 = div_small(first, per_row);
    const uint32_t from = (uint32_t)(first - row0 * per_row) + threadIdx.x, down = from / per_row, c = (from - down * per_row) * kLaneElems;
    return Piece{row0 + down, (int)c, row0 + down < rows ? min(kLaneElems, h - (int)c) : 0};
}

// Rows from `live` on of a result [rows, d] that a product leaves as they are: zeros, by all threads of a launch.
template <typename T> struct Tail {
    T *rows_at;      // or null
    int64_t rows;
    int d;
    __device__ __forceinline__ void clear(int64_t live) const {
        if (rows_at == nullptr || live >= rows) return;
        const int64_t n = (rows - live) * d;
        T *at = rows_at + live * d;
        for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) at[i] = (T)0.f;
    }
};

// m = act(g) u.  pre [rows, 2 h], mid [rows, h].  Bound by memory.
template <typename T>
__global__ __launch_bounds__(kBlock) void gated_act_fwd_kernel(const T *__restrict__ pre, T *__restrict__ mid, const int32_t *__restrict__ table,
                                                               int64_t rows, int h, int per_row, int act, const Tail<T> tail) {
    const int64_t all = rows * 2 * h;
    rows = live_rows(table, rows);
    tail.clear(rows);
    const Piece p = piece_of(rows, h, per_row);
    if (p.n <= 0) return;
    const int64_t at = p.row * 2 * h + p.c;
    T g[kLaneElems], u[kLaneElems];
    load_elems<false>(pre + at, p.n, at + kLaneElems <= all, g);
    load_elems<false>(pre + at + h, p.n, at + h + kLaneElems <= all, u);
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) g[j] = (T)(gate_act<sizeof(T) == 2>((float)g[j], act) * (float)u[j]);
    store_elems<false>(mid + p.row * h + p.c, p.n, g);
}

// grad_pre = [dm u act'(g), dm act(g)]
template <typename T>
__global__ __launch_bounds__(kBlock) void gated_act_bwd_kernel(const T *__restrict__ grad_mid, const T *__restrict__ pre, T *__restrict__ grad_pre,
                                                               const int32_t *__restrict__ table, int64_t rows, int h, int per_row, int act,
                                                               const Tail<T> tail) {
    const int64_t all = rows * h;
    rows = live_rows(table, rows);
    tail.clear(rows);
    const Piece p = piece_of(rows, h, per_row);
    if (p.n <= 0) return;
    const int64_t at = p.row * 2 * h + p.c, at_mid = p.row * h + p.c;
    T g[kLaneElems], u[kLaneElems], d[kLaneElems];
    load_elems<false>(pre + at, p.n, at + kLaneElems <= 2 * all, g);
    load_elems<false>(pre + at + h, p.n, at + h + kLaneElems <= 2 * all, u);
    load_elems<false>(grad_mid + at_mid, p.n, at_mid + kLaneElems <= all, d);
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) {
        const ActTerms t = gate_terms<sizeof(T) == 2>((float)g[j], act);
        const float dm = (float)d[j];
        g[j] = (T)(dm * (float)u[j] * t.slope);
        u[j] = (T)(dm * t.value);
    }
    store_elems<false>(grad_pre + at, p.n, g);
    store_elems<false>(grad_pre + at + h, p.n, u);
}

int per_row(int64_t h) { return (int)ceil_div(h, kLaneElems); }

template <typename F> void with_type(int dtype, F &&f) {
    if (dtype == FMOE_F32) f(float{});
    else if (dtype == FMOE_BF16) f(__bf16{});
    else f(_Float16{});
}

// `live` rows at most (with a table: those that it has); rows of `tail` behind them become zeros
struct Between {
    const int32_t *table;
    int64_t live, h;
    int dtype, activation;
    void *tail;
    int64_t tail_rows, tail_elems;
    hipStream_t stream;
};
int gated_act_forward(const void *pre, void *mid, const Between &b) {
    with_type(b.dtype, [&](auto t) {
        using T = decltype(t);
        gated_act_fwd_kernel<T><<<(unsigned)std::max<int64_t>(1, ceil_div(b.live * per_row(b.h), kBlock)), kBlock, 0, b.stream>>>(
            (const T *)pre, (T *)mid, b.table, b.live, (int)b.h, per_row(b.h), b.activation, Tail<T>{(T *)b.tail, b.tail_rows, (int)b.tail_elems});
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}
int gated_act_backward(const void *grad_mid, const void *pre, void *grad_pre, const Between &b) {
    with_type(b.dtype, [&](auto t) {
        using T = decltype(t);
        gated_act_bwd_kernel<T><<<(unsigned)std::max<int64_t>(1, ceil_div(b.live * per_row(b.h), kBlock)), kBlock, 0, b.stream>>>(
            (const T *)grad_mid, (const T *)pre, (T *)grad_pre, b.table, b.live, (int)b.h, per_row(b.h), b.activation,
            Tail<T>{(T *)b.tail, b.tail_rows, (int)b.tail_elems});
    });
    FMOE_LAUNCH_CHECK();
    return FMOE_OK;
}

struct Sizes {
    int64_t n_expert, rows, d, h;
    int dtype, activation;
};
int check(const char *who, const Sizes &s, const void *segment_table, const int64_t *counts_host) {
    FMOE_REQUIRE(s.dtype == FMOE_F32 || s.dtype == FMOE_BF16 || s.dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who, s.dtype);
    FMOE_REQUIRE(is_gate_activation(s.activation), "%s: unknown activation %d", who, s.activation);
    FMOE_REQUIRE(s.n_expert >= 1 && s.rows >= 0 && s.d >= 1 && s.h >= 1, "%s: bad sizes", who);
    FMOE_REQUIRE(!segment_table != !counts_host, "%s: either a segment table or the counts on the host", who);
    if (s.n_expert > (1 << 24) || s.rows > (int64_t)INT32_MAX - 65536 || s.d > (1 << 28) || s.h > (1 << 28) ||
        ceil_div(s.rows * per_row(s.h), kBlock) > kMostThreads / kBlock)
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    if (counts_host) {
        int64_t total = 0;
        for (int64_t e = 0; e < s.n_expert; ++e) {
            FMOE_REQUIRE(counts_host[e] >= 0 && counts_host[e] <= s.rows, "%s: expert_count[%lld]=%lld", who, (long long)e, (long long)counts_host[e]);
            total += counts_host[e];
        }
        FMOE_REQUIRE(total <= s.rows, "%s: the counts add up to %lld of %lld rows", who, (long long)total, (long long)s.rows);
    }
    return FMOE_OK;
}
int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
// where a call's scratch rows and its products' own workspace lie, one behind the other
struct Scratch {
    int64_t first, second, split;   // bytes
    int64_t total() const { return first + second + split; }
};
GatedArgs gated_sizes(const Sizes &s) {
    static const int32_t some = 0;
    GatedArgs a{};
    a.d = s.d; a.h = s.h; a.n_expert = s.n_expert; a.rows_cap = s.rows; a.dtype = s.dtype; a.activation = s.activation; a.dev_tab = &some;
    return a;
}
Scratch forward_scratch(const Sizes &s, bool keeps_pre, bool table) {
    const bool fused = table && gated_forward_fused(gated_sizes(s));
    return Scratch{keeps_pre || fused ? 0 : round256(s.rows * 2 * s.h * dtype_bytes(s.dtype)), 0,
                   std::max(fused ? gated_forward_workspace_bytes(gated_sizes(s))
                                  : fmoe_linear_forward_dev_workspace_bytes(s.rows, s.n_expert, s.d, 2 * s.h, s.dtype, FMOE_ACT_NONE, 0, 0),
                            fmoe_linear_forward_dev_workspace_bytes(s.rows, s.n_expert, s.h, s.d, s.dtype, FMOE_ACT_NONE, 0, 0))};
}
Scratch backward_scratch(const Sizes &s, bool table) {
    const bool fused = table && gated_dgrad_fused(gated_sizes(s));
    const int64_t row = s.rows * s.h * dtype_bytes(s.dtype);
    return Scratch{round256(2 * row), fused ? 0 : round256(row),
                   std::max(fused ? gated_dgrad_workspace_bytes(gated_sizes(s))
                                  : fmoe_linear_dgrad_dev_workspace_bytes(s.rows, s.n_expert, s.h, s.d, s.dtype, FMOE_ACT_NONE),
                            fmoe_linear_dgrad_dev_workspace_bytes(s.rows, s.n_expert, s.d, 2 * s.h, s.dtype, FMOE_ACT_NONE))};
}

// The products, over a table in device memory or over counts on the host.
struct Products {
    const int32_t *table;
    const int64_t *counts;
    int64_t n_expert, rows, total;   // total: rows that there are, or may be
    int dtype;
    void *ws;
    int64_t ws_bytes;
    hipStream_t stream;

    template <typename Args> void place(Args &a) const {
        a.dev_tab = table;
        a.dev_rows_cap = table ? rows : 0;
        a.dev_any_grid = true;
    }
    int forward(const void *x, const void *w, const void *bias, void *y, int64_t in, int64_t out, bool once) const {
        LinearForwardArgs a{x, w, bias, y, nullptr, in, out, dtype, kEpiStore, FMOE_ACT_NONE};
        place(a);
        a.dev_few_unaligned = true;
        a.dev_weights_once = once;   // (no backward that reads them again)
        a.dev_workspace = ws;
        a.dev_workspace_bytes = ws_bytes;
        return grouped_linear_forward(a, counts, n_expert, 0, total, stream);
    }
    int dgrad(const void *gy, const void *w, void *gx, int64_t in, int64_t out) const {
        LinearDgradArgs a{gy, w, gx, nullptr, in, out, dtype, kEpiStore, FMOE_ACT_NONE};
        place(a);
        a.dev_workspace = ws;
        a.dev_workspace_bytes = ws_bytes;
        return grouped_linear_dgrad(a, counts, n_expert, 0, total, stream);
    }
    int wgrad(const void *gy, const void *x, void *gw, void *gb, int64_t in, int64_t out) const {
        LinearWgradArgs a{gy, x, gw, gb, in, out, dtype};
        place(a);
        return grouped_linear_wgrad(a, counts, n_expert, 0, total, true, stream);
    }
};
Products products(const Sizes &s, const void *segment_table, const int64_t *counts, void *ws, int64_t ws_bytes, void *stream) {
    int64_t total = 0;
    for (int64_t e = 0; counts && e < s.n_expert; ++e) total += counts[e];
    return Products{(const int32_t *)segment_table, counts, s.n_expert, s.rows, segment_table ? s.rows : total, s.dtype, ws, ws_bytes, (hipStream_t)stream};
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int64_t fmoe_gated_mlp_forward_workspace_bytes(int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden, int dtype,
                                                          int activation, int keep, int table) {
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    static const int64_t one = 0;
    if (rows < 1 || n_expert < 1 || check("fmoe_gated_mlp_forward", s, &one, nullptr) != FMOE_OK) return 0;
    return forward_scratch(s, keep != 0, table != 0).total();
}

extern "C" int fmoe_gated_mlp_forward(const void *x, const void *w1, const void *b1, const void *w2, const void *b2, void *pre, void *mid, void *y,
                                      const void *segment_table, const int64_t *expert_count_host, int64_t n_expert, int64_t rows, int64_t d_model,
                                      int64_t d_hidden, int dtype, int activation, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "fmoe_gated_mlp_forward";
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    if (int rc = check(who, s, segment_table, expert_count_host)) return rc;
    if (rows == 0) return FMOE_OK;
    FMOE_REQUIRE(x && w1 && w2 && mid && y, "%s: NULL pointer", who);
    const Scratch need = forward_scratch(s, pre != nullptr, segment_table != nullptr);
    if (need.total() > 0 && (workspace == nullptr || workspace_bytes < need.total() || !aligned16(workspace)))
        return fail(FMOE_EWORKSPACE, "%s: a workspace of %lld bytes on 16 bytes is needed", who, (long long)need.total());
    char *ws = (char *)workspace;
    const Products p = products(s, segment_table, expert_count_host, ws + need.first, need.split, stream);
    const GatedArgs fused{x, w1, b1, pre, mid, y, d_model, d_hidden, n_expert, rows, dtype, activation, p.table, p.ws, p.ws_bytes};
    if (gated_forward_fused(fused)) {
        if (int rc = grouped_gated_forward(fused, p.stream)) return rc;
        return p.forward(mid, w2, b2, y, d_hidden, d_model, pre == nullptr);
    }
    void *between = pre ? pre : ws;
    if (int rc = p.forward(x, w1, b1, between, d_model, 2 * d_hidden, pre == nullptr)) return rc;
    if (int rc = gated_act_forward(between, mid, Between{p.table, p.total, d_hidden, dtype, activation, y, rows, d_model, p.stream})) return rc;
    return p.forward(mid, w2, b2, y, d_hidden, d_model, pre == nullptr);
}

extern "C" int64_t fmoe_gated_mlp_backward_workspace_bytes(int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden, int dtype,
                                                           int activation, int table) {
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    static const int64_t one = 0;
    if (rows < 1 || n_expert < 1 || check("fmoe_gated_mlp_backward", s, &one, nullptr) != FMOE_OK) return 0;
    return backward_scratch(s, table != 0).total();
}

extern "C" int fmoe_gated_mlp_backward(const void *grad_y, const void *x, const void *w1, const void *w2, const void *pre, const void *mid,
                                       void *grad_x, void *grad_w1, void *grad_b1, void *grad_w2, void *grad_b2, const void *segment_table,
                                       const int64_t *expert_count_host, int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden,
                                       int dtype, int activation, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "fmoe_gated_mlp_backward";
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    if (int rc = check(who, s, segment_table, expert_count_host)) return rc;
    FMOE_REQUIRE((!grad_b1 || grad_w1) && (!grad_b2 || grad_w2), "%s: a bias gradient comes with its weight's", who);
    FMOE_REQUIRE(rows == 0 || (grad_y && x && w1 && w2 && pre && mid), "%s: NULL pointer", who);
    const Scratch need = rows == 0 ? Scratch{0, 0, 0} : backward_scratch(s, segment_table != nullptr);
    if (need.total() > 0 && (workspace == nullptr || workspace_bytes < need.total() || !aligned16(workspace)))
        return fail(FMOE_EWORKSPACE, "%s: a workspace of %lld bytes on 16 bytes is needed", who, (long long)need.total());
    char *ws = (char *)workspace;
    const Products p = products(s, segment_table, expert_count_host, ws + need.first + need.second, need.split, stream);
    void *grad_pre = ws, *grad_mid = ws + need.first;
    const GatedArgs fused{grad_y, w2, nullptr, const_cast<void *>(pre), grad_pre, grad_x, d_model, d_hidden, n_expert, rows, dtype, activation, p.table,
                          p.ws, p.ws_bytes};
    if (rows > 0 && (grad_x || grad_w1) && gated_dgrad_fused(fused)) {
        if (int rc = grouped_gated_dgrad(fused, p.stream)) return rc;
    } else if (rows > 0 && (grad_x || grad_w1)) {
        if (int rc = p.dgrad(grad_y, w2, grad_mid, d_hidden, d_model)) return rc;
        if (int rc = gated_act_backward(grad_mid, pre, grad_pre, Between{p.table, p.total, d_hidden, dtype, activation, grad_x, rows, d_model, p.stream}))
            return rc;
    }
    if (grad_w2)
        if (int rc = p.wgrad(grad_y, mid, grad_w2, grad_b2, d_hidden, d_model)) return rc;
    if (grad_x && rows > 0)
        if (int rc = p.dgrad(grad_pre, w1, grad_x, d_model, 2 * d_hidden)) return rc;
    if (grad_w1)
        if (int rc = p.wgrad(grad_pre, x, grad_w1, grad_b1, d_model, 2 * d_hidden)) return rc;
    return FMOE_OK;
}
