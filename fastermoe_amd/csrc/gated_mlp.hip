// Gated experts (gfx950): per expert, over its rows,
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  m = act(g) u,  y = m W2^T + b2            (W1 = [Wg; Wu], its products [g u] = `pre`, float32)
//   dm = dy W2,  dg = dm u act'(g),  du = dm act(g),  dx = [dg du] W1,  dW1 = [dg du]^T x,  dW2 = dy^T m
//
// The products do the activation's work in their epilogues (gemm_kernel.hpp, gemm_ring.hpp, gemm_skinny.hip; rows off the 16-byte grid, 16-bit types:
// gemm_unaligned.hip, gemm_few_unaligned.hip).  This file holds the calls of the whole block, the activation's kernel for few rows in float32, and the kernel that moves
// float32 tensors of sizes that are no multiple of four into rows that are, and results back: the padding is zeros, whose g, u and m are zeros too.
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

// m = act(g) u for few rows in float32, whose products are the decoding kernel's.  pre [rows, 2 h], mid [rows, h].  Bound by its launch.
__global__ __launch_bounds__(kBlock) void gated_act_kernel(const float *__restrict__ pre, float *__restrict__ mid, const int32_t *__restrict__ table, int64_t rows,
                                                           int h, int per_row, int act, const Tail<float> tail) {
    const int64_t all = rows * 2 * h;
    rows = live_rows(table, rows);
    tail.clear(rows);
    const Piece p = piece_of(rows, h, per_row);
    if (p.n <= 0) return;
    const int64_t at = p.row * 2 * h + p.c;
    float g[kLaneElems], u[kLaneElems];
    load_elems<false>(pre + at, p.n, at + kLaneElems <= all, g);
    load_elems<false>(pre + at + h, p.n, at + h + kLaneElems <= all, u);
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) g[j] = gate_act<false>(g[j], act) * u[j];
    store_elems<false>(mid + p.row * h + p.c, p.n, g);
}

int per_row(int64_t h) { return (int)ceil_div(h, kLaneElems); }

// Rows of float32 from one place into another, in blocks of rows (a matrix half, or all): what of a block or a row the source has none of becomes zeros, what the
// destination has no room for is left out.
struct Move {
    const float *src;
    float *dst;
    int64_t rows;                              // of the destination
    int64_t block_src, block_dst;              // rows of a block
    int cols_src, cols_dst;
    const int32_t *table;
    int rows_of_row;                           // not 0: only rows r with r / rows_of_row below the table's rows
    int blocks_of_expert;                      // not 0: only blocks of experts with rows
};
constexpr int kMoveLoads = 8, kMoves = 6;
// all of a direction's, one after the other
struct Moves {
    Move m[kMoves];
    int n;
};
// A wave to a row, kMoveLoads of a lane's loads on their way at a time (one: 1001 -> 2 x 2003, 8 experts, 1 row, forward 70 us, 52 so, 40 with
// all moves of a direction in one launch).  Bound by memory.
__global__ __launch_bounds__(kBlock) void move_rows_kernel(const Moves all) {
    const int lane = threadIdx.x % kWave;
    int64_t row = (int64_t)blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
    const int64_t step = (int64_t)gridDim.x * (kBlock / kWave);
    for (int i = 0; i < all.n; ++i) {
        const Move &m = all.m[i];
        for (; row < m.rows; row += step) {
            if (m.rows_of_row && row / m.rows_of_row >= m.table[segtab::kRows]) continue;
            const int64_t block = row / m.block_dst, in_block = row - block * m.block_dst;
            if (m.blocks_of_expert) {
                const int64_t e = block / m.blocks_of_expert;
                if (m.table[segtab::kHeader + e] == m.table[segtab::kHeader + e + 1]) continue;
            }
            const float *src = m.src + (block * m.block_src + in_block) * m.cols_src;
            const int n = in_block < m.block_src ? m.cols_src : 0;
            float *dst = m.dst + row * m.cols_dst;
            for (int c = lane; c < m.cols_dst; c += kMoveLoads * kWave) {
                float v[kMoveLoads];
#pragma unroll
                for (int j = 0; j < kMoveLoads; ++j) v[j] = c + j * kWave < n ? __builtin_nontemporal_load(src + c + j * kWave) : 0.f;
#pragma unroll
                for (int j = 0; j < kMoveLoads; ++j)
                    if (c + j * kWave < m.cols_dst) dst[c + j * kWave] = v[j];
            }
        }
        row -= m.rows;   // (the next one's rows follow)
    }
}

struct Sizes {
    int64_t n_expert, rows, d, h;
    int dtype, activation;
};
// float32, and its rounded sizes: offsets from a tile's first row of weights, over both halves, in 31 bits; rows of at most 4 MiB
bool features_taken(int64_t d, int64_t h, int dtype) {
    return d <= (1 << 28) && h <= (1 << 28) &&
           (dtype != FMOE_F32 || ((2 * h + 264) * (d + 3) * 4 < ((int64_t)1 << 31) && 2 * (h + 3) * 4 <= (1 << 22) && ceil_div(d, 4) * 16 <= (1 << 22)));
}
int check(const char *who, const Sizes &s) {
    FMOE_REQUIRE(s.dtype == FMOE_F32 || s.dtype == FMOE_BF16 || s.dtype == FMOE_F16, "%s: dtype %d is not float32, bfloat16 or float16", who, s.dtype);
    FMOE_REQUIRE(is_gate_activation(s.activation), "%s: unknown activation %d", who, s.activation);
    FMOE_REQUIRE(s.n_expert >= 1 && s.rows >= 0 && s.d >= 1 && s.h >= 1, "%s: bad sizes", who);
    if (!features_taken(s.d, s.h, s.dtype))
        return fail(FMOE_ELIMIT, "%s: d_model=%lld d_hidden=%lld are beyond the supported range (float32: 2 GiB of an expert's weights, rows of 4 MiB)", who,
                    (long long)s.d, (long long)s.h);
    if (s.n_expert > (1 << 24) || s.rows > (int64_t)INT32_MAX - 65536 ||
        (s.dtype == FMOE_F32 && ceil_div(s.rows * per_row(s.h), kBlock) > kMostThreads / kBlock))   // (the activation's kernel)
        return fail(FMOE_ELIMIT, "%s: sizes beyond the supported range", who);
    return FMOE_OK;
}
int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
// where a call's scratch rows and its products' own workspace lie, one behind the other
struct Scratch {
    int64_t first, split;   // bytes
    int64_t total() const { return first + split; }
};
GatedArgs gated_sizes(const Sizes &s) {
    static const int32_t some = 0;
    GatedArgs a{};
    a.d = s.d; a.h = s.h; a.n_expert = s.n_expert; a.rows_cap = s.rows; a.dtype = s.dtype; a.activation = s.activation; a.dev_tab = &some;
    return a;
}
Scratch forward_scratch(const Sizes &s, bool keeps_pre) {
    const bool fused = gated_forward_fused(gated_sizes(s));
    return Scratch{keeps_pre || fused ? 0 : round256(s.rows * 2 * s.h * dtype_bytes(s.dtype)),
                   std::max(fused ? gated_forward_workspace_bytes(gated_sizes(s))
                                  : fmoe_linear_forward_dev_workspace_bytes(s.rows, s.n_expert, s.d, 2 * s.h, s.dtype, FMOE_ACT_NONE, 0, 0),
                            std::max(fmoe_linear_forward_dev_workspace_bytes(s.rows, s.n_expert, s.h, s.d, s.dtype, FMOE_ACT_NONE, 0, 0),
                                     unaligned_parts_bytes(s.rows, s.n_expert, s.d, s.h, s.dtype)))};
}
Scratch backward_scratch(const Sizes &s) {
    return Scratch{round256(2 * s.rows * s.h * dtype_bytes(s.dtype)),
                   std::max(gated_dgrad_workspace_bytes(gated_sizes(s)),
                            std::max(fmoe_linear_dgrad_dev_workspace_bytes(s.rows, s.n_expert, s.d, 2 * s.h, s.dtype, FMOE_ACT_NONE),
                                     unaligned_parts_bytes(s.rows, s.n_expert, s.d, 2 * s.h, s.dtype)))};
}

// The products over the table
struct Products {
    const int32_t *table;
    int64_t n_expert, rows;
    int dtype;
    void *ws;
    int64_t ws_bytes;
    hipStream_t stream;

    template <typename Args> void place(Args &a) const {
        a.dev_tab = table;
        a.dev_rows_cap = rows;
        a.dev_any_grid = true;
    }
    int forward(const void *x, const void *w, const void *bias, void *y, int64_t in, int64_t out, bool once) const {
        LinearForwardArgs a{x, w, bias, y, nullptr, in, out, dtype, kEpiStore, FMOE_ACT_NONE};
        place(a);
        a.dev_any_order = true;
        a.dev_weights_once = once;   // (no backward that reads them again)
        a.dev_workspace = ws;
        a.dev_workspace_bytes = ws_bytes;
        return grouped_linear_forward(a, nullptr, n_expert, 0, rows, stream);
    }
    int dgrad(const void *gy, const void *w, void *gx, int64_t in, int64_t out) const {
        LinearDgradArgs a{gy, w, gx, nullptr, in, out, dtype, kEpiStore, FMOE_ACT_NONE};
        place(a);
        a.dev_any_order = true;
        a.dev_workspace = ws;
        a.dev_workspace_bytes = ws_bytes;
        return grouped_linear_dgrad(a, nullptr, n_expert, 0, rows, stream);
    }
    int wgrad(const void *gy, const void *x, void *gw, void *gb, int64_t in, int64_t out) const {
        LinearWgradArgs a{gy, x, gw, gb, in, out, dtype};
        place(a);
        return grouped_linear_wgrad(a, nullptr, n_expert, 0, rows, true, stream);
    }
};

struct Forward {
    const void *x, *w1, *b1, *w2, *b2;
    void *pre, *mid, *y;
};
struct Backward {
    const void *grad_y, *x, *w1, *w2, *pre, *mid;
    void *grad_x, *grad_w1, *grad_b1, *grad_w2, *grad_b2;
};

int forward(const Sizes &s, const Forward &f, const int32_t *table, char *ws, hipStream_t stream) {
    const Scratch need = forward_scratch(s, f.pre != nullptr);
    const Products p{table, s.n_expert, s.rows, s.dtype, ws + need.first, need.split, stream};
    const GatedArgs fused{f.x, f.w1, f.b1, f.pre, f.mid, f.y, s.d, s.h, s.n_expert, s.rows, s.dtype, s.activation, table, p.ws, p.ws_bytes};
    const bool once = f.pre == nullptr;
    if (gated_forward_fused(fused)) {
        if (int rc = grouped_gated_forward(fused, stream)) return rc;
    } else {
        void *pre = f.pre ? f.pre : ws;
        if (int rc = p.forward(f.x, f.w1, f.b1, pre, s.d, 2 * s.h, once)) return rc;
        gated_act_kernel<<<(unsigned)std::max<int64_t>(1, ceil_div(s.rows * per_row(s.h), kBlock)), kBlock, 0, stream>>>(
            (const float *)pre, (float *)f.mid, table, s.rows, (int)s.h, per_row(s.h), s.activation, Tail<float>{(float *)f.y, s.rows, (int)s.d});
        FMOE_LAUNCH_CHECK();
    }
    return p.forward(f.mid, f.w2, f.b2, f.y, s.h, s.d, once);
}

int backward(const Sizes &s, const Backward &b, const int32_t *table, char *ws, hipStream_t stream) {
    const Scratch need = s.rows == 0 ? Scratch{0, 0} : backward_scratch(s);
    const Products p{table, s.n_expert, s.rows, s.dtype, ws + need.first, need.split, stream};
    void *grad_pre = ws;
    if (s.rows > 0 && (b.grad_x || b.grad_w1)) {
        const GatedArgs fused{b.grad_y, b.w2, nullptr, const_cast<void *>(b.pre), grad_pre, b.grad_x, s.d, s.h, s.n_expert, s.rows, s.dtype, s.activation, table,
                              p.ws, p.ws_bytes};
        if (int rc = grouped_gated_dgrad(fused, stream)) return rc;
    }
    if (b.grad_w2)
        if (int rc = p.wgrad(b.grad_y, b.mid, b.grad_w2, b.grad_b2, s.h, s.d)) return rc;
    if (b.grad_x && s.rows > 0)
        if (int rc = p.dgrad(grad_pre, b.w1, b.grad_x, s.d, 2 * s.h)) return rc;
    if (b.grad_w1)
        if (int rc = p.wgrad(grad_pre, b.x, b.grad_w1, b.grad_b1, s.d, 2 * s.h)) return rc;
    return FMOE_OK;
}

// float32 in sizes that are no multiple of four: the same with sizes that are, on copies.  (With products that check every
// element, over counts read on the host, us forward and with the backward, and like this: 1 row, 8 experts of 1001 -> 2 x 2003: 180, 493 / 40, 242; 64 rows, 33 of 443 -> 2 x
// 2368: 300, 801 / 186, 757; 1554 rows, 12 of 501 -> 2 x 1303: 257, 677 / 128, 384; 8192 rows, 8 of 1023 -> 2 x 2047: 2088, 5494 / 694, 2240.)
bool padded(const Sizes &s) { return s.dtype == FMOE_F32 && (s.d % 4 != 0 || s.h % 4 != 0); }
Sizes whole(const Sizes &s) {
    Sizes w = s;
    w.d = ceil_div(s.d, 4) * 4;
    w.h = ceil_div(s.h, 4) * 4;
    return w;
}
// What lies right as it is, in rows of a size that is a multiple of four, is used where it lies.
struct Copies {
    Sizes s, w;
    const int32_t *table;
    char *ws;          // null: only the sizes are added up
    hipStream_t stream;
    int64_t used = 0;
    Moves moves{};

    float *room(int64_t floats) {
        float *at = ws ? (float *)(ws + used) : nullptr;
        used += round256(floats * 4);
        return at;
    }
    // one matrix, or per block of rows: `blocks` of `rows` rows of `cols` elements, those of the padded sizes beside them
    struct Shape {
        int64_t blocks, rows, rows_padded, cols, cols_padded;
        int rows_of_row, blocks_of_expert;
        bool as_it_is() const { return rows == rows_padded && cols == cols_padded; }
        int64_t floats() const { return blocks * rows_padded * cols_padded; }
    };
    Shape rows_of(int halves, bool hidden) const { return {1, s.rows * halves, s.rows * halves, hidden ? s.h : s.d, hidden ? w.h : w.d, halves, 0}; }
    Shape w1() const { return {2 * s.n_expert, s.h, w.h, s.d, w.d, 0, 2}; }
    Shape b1() const { return {1, 2 * s.n_expert, 2 * s.n_expert, s.h, w.h, 0, 0}; }
    Shape w2() const { return {s.n_expert, s.d, w.d, s.h, w.h, 0, 1}; }
    Shape b2() const { return {1, s.n_expert, s.n_expert, s.d, w.d, 0, 0}; }

    void add(const Move &m) {
        if (m.rows > 0) moves.m[moves.n++] = m;
    }
    const void *in(const void *t, const Shape &at) {
        if (at.as_it_is()) return t;
        float *copy = room(at.floats());
        if (ws == nullptr || t == nullptr) return nullptr;
        add(Move{(const float *)t, copy, at.blocks * at.rows_padded, at.rows, at.rows_padded, (int)at.cols, (int)at.cols_padded, table, at.rows_of_row, at.blocks_of_expert});
        return copy;
    }
    // where a result goes first: `t` itself, or room for its padded form (wanted: or nowhere)
    void *result(void *t, const Shape &at, bool wanted = true) {
        if (at.as_it_is()) return t;
        float *copy = room(at.floats());
        return wanted ? copy : nullptr;
    }
    // `live`: only rows that there are
    void out(const void *from, void *t, const Shape &at, bool live) {
        if (t == nullptr || from == nullptr || from == t) return;
        add(Move{(const float *)from, (float *)t, at.blocks * at.rows, at.rows_padded, at.rows, (int)at.cols_padded, (int)at.cols, table, live ? at.rows_of_row : 0, 0});
    }
    int flush() {
        int64_t rows = 0;
        for (int i = 0; i < moves.n; ++i) rows += moves.m[i].rows;
        if (rows > 0) {
            move_rows_kernel<<<(unsigned)std::min<int64_t>(ceil_div(rows, kBlock / kWave), 1 << 20), kBlock, 0, stream>>>(moves);
            FMOE_LAUNCH_CHECK();
        }
        moves.n = 0;
        return FMOE_OK;
    }
};
// (ws null: the workspace's bytes in *bytes)
int padded_forward(const Sizes &s, const Forward &f, const int32_t *table, char *ws, int64_t *bytes, hipStream_t stream) {
    const Sizes w = whole(s);
    Copies c{s, w, table, ws, stream};
    Forward g{};
    g.x = c.in(f.x, c.rows_of(1, false));
    g.w1 = c.in(f.w1, c.w1()); g.b1 = c.in(f.b1, c.b1()); g.w2 = c.in(f.w2, c.w2()); g.b2 = c.in(f.b2, c.b2());
    g.mid = c.result(f.mid, c.rows_of(1, true)); g.y = c.result(f.y, c.rows_of(1, false));
    g.pre = f.pre ? c.result(f.pre, c.rows_of(2, true)) : nullptr;
    if (ws == nullptr) {
        *bytes = c.used + forward_scratch(w, f.pre != nullptr).total();
        return FMOE_OK;
    }
    if (int rc = c.flush()) return rc;
    if (int rc = forward(w, g, table, ws + c.used, stream)) return rc;
    c.out(g.y, f.y, c.rows_of(1, false), false);
    if (f.pre) {
        c.out(g.pre, f.pre, c.rows_of(2, true), true);
        c.out(g.mid, f.mid, c.rows_of(1, true), true);
    }
    return c.flush();
}
int padded_backward(const Sizes &s, const Backward &b, const int32_t *table, char *ws, int64_t *bytes, hipStream_t stream) {
    const Sizes w = whole(s);
    Copies c{s, w, table, ws, stream};
    Backward g{};
    g.grad_y = c.in(b.grad_y, c.rows_of(1, false)); g.x = c.in(b.x, c.rows_of(1, false));
    g.w1 = c.in(b.w1, c.w1()); g.w2 = c.in(b.w2, c.w2());
    g.pre = c.in(b.pre, c.rows_of(2, true)); g.mid = c.in(b.mid, c.rows_of(1, true));
    g.grad_x = c.result(b.grad_x, c.rows_of(1, false), b.grad_x != nullptr);
    g.grad_w1 = c.result(b.grad_w1, c.w1(), b.grad_w1 != nullptr); g.grad_b1 = c.result(b.grad_b1, c.b1(), b.grad_b1 != nullptr);
    g.grad_w2 = c.result(b.grad_w2, c.w2(), b.grad_w2 != nullptr); g.grad_b2 = c.result(b.grad_b2, c.b2(), b.grad_b2 != nullptr);
    if (ws == nullptr) {
        *bytes = c.used + (s.rows == 0 ? 0 : backward_scratch(w).total());
        return FMOE_OK;
    }
    if (int rc = c.flush()) return rc;
    if (int rc = backward(w, g, table, ws + c.used, stream)) return rc;
    if (s.rows > 0) c.out(g.grad_x, b.grad_x, c.rows_of(1, false), false);
    c.out(g.grad_w1, b.grad_w1, c.w1(), false); c.out(g.grad_b1, b.grad_b1, c.b1(), false);
    c.out(g.grad_w2, b.grad_w2, c.w2(), false); c.out(g.grad_b2, b.grad_b2, c.b2(), false);
    return c.flush();
}
int64_t forward_bytes(const Sizes &s, bool keep) {
    if (!padded(s)) return forward_scratch(s, keep).total();
    static char some;
    Forward f{};
    f.pre = keep ? &some : nullptr;
    int64_t bytes = 0;
    padded_forward(s, f, nullptr, nullptr, &bytes, nullptr);
    return bytes;
}
int64_t backward_bytes(const Sizes &s) {
    if (!padded(s)) return s.rows == 0 ? 0 : backward_scratch(s).total();
    int64_t bytes = 0;
    padded_backward(s, Backward{}, nullptr, nullptr, &bytes, nullptr);
    return bytes;
}

}  // namespace
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_gated_mlp_supported(int64_t d_model, int64_t d_hidden, int dtype) {
    return (dtype == FMOE_F32 || dtype == FMOE_BF16 || dtype == FMOE_F16) && d_model >= 1 && d_hidden >= 1 && features_taken(d_model, d_hidden, dtype);
}

extern "C" int64_t fmoe_gated_mlp_forward_workspace_bytes(int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden, int dtype, int activation,
                                                          int keep) {
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    if (rows < 1 || check("fmoe_gated_mlp_forward", s) != FMOE_OK) return 0;
    return forward_bytes(s, keep != 0);
}

extern "C" int fmoe_gated_mlp_forward(const void *x, const void *w1, const void *b1, const void *w2, const void *b2, void *pre, void *mid, void *y,
                                      const void *segment_table, int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden, int dtype,
                                      int activation, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "fmoe_gated_mlp_forward";
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    if (int rc = check(who, s)) return rc;
    if (rows == 0) return FMOE_OK;
    FMOE_REQUIRE(x && w1 && w2 && mid && y && segment_table, "%s: NULL pointer", who);
    FMOE_REQUIRE(aligned16(segment_table), "%s: the segment table must be 16-byte aligned", who);
    FMOE_REQUIRE(dtype != FMOE_F32 || (aligned16(x) && aligned16(w1) && aligned16(b1) && aligned16(w2) && aligned16(b2) && aligned16(pre) && aligned16(mid) &&
                                       aligned16(y)), "%s: float32 tensors begin on 16 bytes", who);
    FMOE_REQUIRE(((uintptr_t)pre & 3) == 0, "%s: pre holds float32", who);
    const int64_t need = forward_bytes(s, pre != nullptr);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(FMOE_EWORKSPACE, "%s: a workspace of %lld bytes on 16 bytes is needed", who, (long long)need);
    const Forward f{x, w1, b1, w2, b2, pre, mid, y};
    if (padded(s)) return padded_forward(s, f, (const int32_t *)segment_table, (char *)workspace, nullptr, (hipStream_t)stream);
    return forward(s, f, (const int32_t *)segment_table, (char *)workspace, (hipStream_t)stream);
}

extern "C" int64_t fmoe_gated_mlp_backward_workspace_bytes(int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden, int dtype, int activation) {
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    if (check("fmoe_gated_mlp_backward", s) != FMOE_OK) return 0;
    return backward_bytes(s);
}

extern "C" int fmoe_gated_mlp_backward(const void *grad_y, const void *x, const void *w1, const void *w2, const void *pre, const void *mid,
                                       void *grad_x, void *grad_w1, void *grad_b1, void *grad_w2, void *grad_b2, const void *segment_table,
                                       int64_t n_expert, int64_t rows, int64_t d_model, int64_t d_hidden, int dtype, int activation, void *workspace,
                                       int64_t workspace_bytes, void *stream) {
    const char *who = "fmoe_gated_mlp_backward";
    const Sizes s{n_expert, rows, d_model, d_hidden, dtype, activation};
    if (int rc = check(who, s)) return rc;
    FMOE_REQUIRE((!grad_b1 || grad_w1) && (!grad_b2 || grad_w2), "%s: a bias gradient comes with its weight's", who);
    FMOE_REQUIRE((rows == 0 || (grad_y && x && w1 && w2 && pre && mid)) && segment_table, "%s: NULL pointer", who);
    FMOE_REQUIRE(aligned16(segment_table), "%s: the segment table must be 16-byte aligned", who);
    FMOE_REQUIRE(dtype != FMOE_F32 || (aligned16(grad_y) && aligned16(x) && aligned16(w1) && aligned16(w2) && aligned16(pre) && aligned16(mid) &&
                                       aligned16(grad_x) && aligned16(grad_w1) && aligned16(grad_b1) && aligned16(grad_w2) && aligned16(grad_b2)),
                 "%s: float32 tensors begin on 16 bytes", who);
    FMOE_REQUIRE(((uintptr_t)pre & 3) == 0, "%s: pre holds float32", who);
    const int64_t need = backward_bytes(s);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(FMOE_EWORKSPACE, "%s: a workspace of %lld bytes on 16 bytes is needed", who, (long long)need);
    const Backward b{grad_y, x, w1, w2, pre, mid, grad_x, grad_w1, grad_b1, grad_w2, grad_b2};
    if (padded(s)) return padded_backward(s, b, (const int32_t *)segment_table, (char *)workspace, nullptr, (hipStream_t)stream);
    return backward(s, b, (const int32_t *)segment_table, (char *)workspace, (hipStream_t)stream);
}
