// Gated experts as an autograd node, and the experts' products in 8-bit integers, from Python's tensors to the enqueued kernels (host code).
//
// A decoding step's kernels take 12 to 20 us; from Python a call took 27 to 31 us to enqueue them.  As in block_call.cpp, what a call takes is decided here, and
// None sends it the way through Python.
#include "block_call.hpp"

#include "call_tools.hpp"

#include <torch/csrc/autograd/functions/basic_ops.h>

using namespace fmoe_call;

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the library's entry points, which Python has loaded (bind)
struct Entries {
    decltype(&fmoe_last_error) last_error;
    decltype(&fmoe_segment_table_bytes) table_bytes;
    decltype(&fmoe_gated_mlp_forward_workspace_bytes) gated_forward_bytes;
    decltype(&fmoe_gated_mlp_forward) gated_forward;
    decltype(&fmoe_gated_mlp_backward_workspace_bytes) gated_backward_bytes;
    decltype(&fmoe_gated_mlp_backward) gated_backward;
    decltype(&fmoe_quantize_rows) quantize_rows;
    decltype(&fmoe_linear_int8_workspace_bytes) int8_bytes;
    decltype(&fmoe_linear_int8) linear_int8;
    decltype(&fmoe_linear_int8_rounds_rows) int8_rounds_rows;
} entry = {};
constexpr int kEntries = 10;

void ok(int rc) { TORCH_CHECK(rc == FMOE_OK, "libfmoe_hip error ", rc, ": ", entry.last_error()); }
bool on_16_bytes(const at::Tensor &t) { return !t.defined() || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
// what a forward saved lies so, but hooks may hand back anything equal to it
at::Tensor whole(const at::Tensor &t) {
    const at::Tensor c = t.contiguous();
    return on_16_bytes(c) ? c : c.clone();
}
at::Tensor space_of(int64_t bytes, const at::Tensor &like) {
    return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

struct GatedMLP : torch::autograd::Function<GatedMLP> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &given, const at::Tensor &w1, const Maybe &of_b1, const at::Tensor &w2,
                              const Maybe &of_b2, const at::Tensor &table, int64_t activation, bool keep) {
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Tensor b1 = of_b1.value_or(at::Tensor()), b2 = of_b2.value_or(at::Tensor());
        const c10::OptionalDeviceGuard guard(given.device());
        const at::Tensor x = given.contiguous();
        const int64_t n = x.size(0), d = x.size(1), e = w1.size(0), h = w2.size(2);
        const int dtype = dtype_code(x), act = (int)activation;
        const at::Tensor y = at::empty({n, d}, x.options()), mid = at::empty({n, h}, x.options());
        const at::Tensor pre = keep ? at::empty({n, 2 * h}, x.options().dtype(at::kFloat)) : at::Tensor();
        const int64_t bytes = entry.gated_forward_bytes(e, n, d, h, dtype, act, keep);
        const at::Tensor space = space_of(bytes, x);
        ok(entry.gated_forward(pointer(x), pointer(w1), pointer(b1), pointer(w2), pointer(b2), pointer(pre), pointer(mid), pointer(y), pointer(table),
                               e, n, d, h, dtype, act, pointer(space), bytes, stream_of(x)));
        if (keep) {
            ctx->save_for_backward({x, w1, w2, pre, mid, table});
            ctx->saved_data["activation"] = activation;
            ctx->saved_data["biases"] = (int64_t)(b1.defined() ? 1 : 0) + (b2.defined() ? 2 : 0);
        }
        return y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const int64_t biases = ctx->saved_data["biases"].toInt();
        const int act = (int)ctx->saved_data["activation"].toInt();
        const bool has_b1 = biases & 1, has_b2 = biases & 2;
        // (asked by the tensors that there were)
        const bool need_x = ctx->needs_input_grad(0), need_w1 = ctx->needs_input_grad(1), need_b1 = has_b1 && ctx->needs_input_grad(2);
        const bool need_w2 = ctx->needs_input_grad(2 + has_b1), need_b2 = has_b2 && ctx->needs_input_grad(3 + has_b1);
        at::Tensor gx, gw1, gb1, gw2, gb2;
        {
            const at::NoGradGuard no_grad;
            const c10::OptionalDeviceGuard guard(saved[0].device());
            const at::Tensor x = whole(saved[0]), w1 = whole(saved[1]), w2 = whole(saved[2]), pre = whole(saved[3]), mid = whole(saved[4]);
            const at::Tensor table = whole(saved[5]), gy = whole(grads[0]);
            const int64_t n = x.size(0), d = x.size(1), e = w1.size(0), h = w2.size(2);
            auto fresh = [&](bool wanted, at::IntArrayRef sizes) { return wanted ? at::empty(sizes, x.options()) : at::Tensor(); };
            gx = fresh(need_x, {n, d});
            gw1 = fresh(need_w1 || need_b1, {e, 2 * h, d});
            gb1 = fresh(need_b1, {e, 2 * h});
            gw2 = fresh(need_w2 || need_b2, {e, d, h});
            gb2 = fresh(need_b2, {e, d});
            const int64_t bytes = entry.gated_backward_bytes(e, n, d, h, dtype_code(x), act);
            const at::Tensor space = space_of(bytes, x);
            ok(entry.gated_backward(pointer(gy), pointer(x), pointer(w1), pointer(w2), pointer(pre), pointer(mid), pointer(gx), pointer(gw1), pointer(gb1),
                                    pointer(gw2), pointer(gb2), pointer(table), e, n, d, h, dtype_code(x), act, pointer(space), bytes,
                                    stream_of(x)));
        }
        const at::Tensor none;
        variable_list out{gx, need_w1 ? gw1 : none, gb1, need_w2 ? gw2 : none, gb2};
        if (at::GradMode::is_enabled()) {   // a backward that is to be differentiated again: an error when it is
            variable_list there;
            for (at::Tensor &t : out)
                if (t.defined()) there.push_back(t.set_requires_grad(true));
            auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice through gated experts, whose backward has no derivative",
                                                                        (int64_t)there.size());
            there = (*error)(std::move(there));
            size_t i = 0;
            for (at::Tensor &t : out)
                if (t.defined()) t = there[i++];
        }
        return {out[0], out[1], out[2], out[3], out[4], none, none, none};
    }
};

bool good_table(const at::Tensor &table, const at::Tensor &x, int64_t rows, int64_t experts) {
    return on_gpu(table) && table.device() == x.device() && table.scalar_type() == at::kInt && table.is_contiguous() &&
           table.numel() * 4 == entry.table_bytes(rows, experts);
}
bool activation_taken(long a) { return a == FMOE_ACT_NONE || a == FMOE_ACT_RELU || a == FMOE_ACT_GELU || a == FMOE_ACT_SILU; }

}  // namespace

PyObject *fmoe_expert_bind(PyObject *, PyObject *args) {
    unsigned long long a[kEntries];
    if (!PyArg_ParseTuple(args, "KKKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9])) return nullptr;
    auto set = [&](auto &fn, int i) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(static_cast<uintptr_t>(a[i])); };
    set(entry.last_error, 0);
    set(entry.table_bytes, 1);
    set(entry.gated_forward_bytes, 2);
    set(entry.gated_forward, 3);
    set(entry.gated_backward_bytes, 4);
    set(entry.gated_backward, 5);
    set(entry.quantize_rows, 6);
    set(entry.int8_bytes, 7);
    set(entry.linear_int8, 8);
    set(entry.int8_rounds_rows, 9);
    Py_RETURN_NONE;
}

// gated_mlp(inp, w1, b1, w2, b2, table, activation): the block's output; None where the call does not take these tensors
PyObject *fmoe_expert_gated_mlp(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 7 || entry.gated_forward == nullptr) {
        PyErr_SetString(PyExc_TypeError, "gated_mlp: 7 arguments, after bind_expert");
        return nullptr;
    }
    std::array<at::Tensor, 6> t;
    long activation;
    if (!tensors(args, t) || !number(args[6], activation)) return nullptr;
    const auto &[x, w1, b1, w2, b2, table] = t;
    if (!on_gpu(x) || x.dim() != 2 || x.size(0) == 0 || dtype_code(x) < 0 || !activation_taken(activation) || !w1.defined() || !w2.defined()) Py_RETURN_NONE;
    for (const at::Tensor *p : {&w1, &b1, &w2, &b2})
        if (p->defined() && (!on_gpu(*p) || p->device() != x.device() || p->scalar_type() != x.scalar_type() || !p->is_contiguous())) Py_RETURN_NONE;
    if (w1.dim() != 3 || w2.dim() != 3) Py_RETURN_NONE;
    const int64_t n = x.size(0), d = x.size(1), e = w1.size(0), h = w2.size(2);
    if (e == 0 || d == 0 || h == 0 || w1.sizes() != at::IntArrayRef({e, 2 * h, d}) || w2.sizes() != at::IntArrayRef({e, d, h}) ||
        (b1.defined() && b1.sizes() != at::IntArrayRef({e, 2 * h})) || (b2.defined() && b2.sizes() != at::IntArrayRef({e, d})) ||
        !good_table(table, x, n, e))
        Py_RETURN_NONE;
    if (x.scalar_type() == at::kFloat) {   // (copied where they are not)
        if (x.is_contiguous() && !on_16_bytes(x)) Py_RETURN_NONE;
        for (const at::Tensor *p : {&w1, &b1, &w2, &b2})
            if (!on_16_bytes(*p)) Py_RETURN_NONE;
    }
    at::Tensor out;
    {
        const WithoutLock no_lock;
        bool keep = false;
        for (const at::Tensor &p : t) keep |= p.defined() && p.requires_grad();
        out = GatedMLP::apply(x, w1, maybe(b1), w2, maybe(b2), table, (int64_t)activation, keep && at::GradMode::is_enabled());
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// linear_int8(inp, weight, weight_scale, bias, table, row_index, index_div, activation, gated): the product; None where the call does not take these tensors
PyObject *fmoe_expert_linear_int8(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 9 || entry.linear_int8 == nullptr) {
        PyErr_SetString(PyExc_TypeError, "linear_int8: 9 arguments, after bind_expert");
        return nullptr;
    }
    std::array<at::Tensor, 6> t;
    long index_div, activation, gated;
    if (!tensors(args, t) || !number(args[6], index_div) || !number(args[7], activation) || !number(args[8], gated)) return nullptr;
    const auto &[x, weight, scale, bias, table, index] = t;
    if (!on_gpu(x) || x.dim() != 2 || x.size(0) == 0 || dtype_code(x) < 0 || x.stride(1) != 1 || index_div < 1 || !activation_taken(activation)) Py_RETURN_NONE;
    if (!on_gpu(weight) || weight.device() != x.device() || weight.scalar_type() != at::kChar || weight.dim() != 3 || weight.numel() == 0) Py_RETURN_NONE;
    const int64_t e = weight.size(0), rows_w = weight.size(1), d = weight.size(2), whole_d = (d + 15) / 16 * 16;
    // (rows that have to be copied, and sizes that the library refuses, go through Python)
    const int64_t by_expert = weight.stride(0), by_row = weight.stride(1);
    if (d > 131072 || by_row > (1 << 22) || (gated ? rows_w / 2 : rows_w) * x.element_size() > (1 << 22) || (by_row > 0 && rows_w * by_row >= ((int64_t)1 << 31))) Py_RETURN_NONE;
    if ((weight.stride(2) != 1 && d != 1) || by_row % 16 || by_row < whole_d || by_expert % 16 || by_expert < 0 || !on_16_bytes(weight) ||
        weight.storage_offset() + (e - 1) * by_expert + (rows_w - 1) * by_row + whole_d > (int64_t)weight.storage().nbytes())
        Py_RETURN_NONE;
    auto channels = [&](const at::Tensor &p, at::ScalarType type) {
        return on_gpu(p) && p.device() == x.device() && p.scalar_type() == type && p.is_contiguous() && on_16_bytes(p) && p.sizes() == at::IntArrayRef({e, rows_w});
    };
    if (!channels(scale, at::kFloat) || (bias.defined() && !channels(bias, x.scalar_type())) || x.size(1) != d || (gated && rows_w % 2)) Py_RETURN_NONE;
    if (index.defined() && (!on_gpu(index) || index.device() != x.device() || index.scalar_type() != at::kLong || !index.is_contiguous() || index.numel() == 0))
        Py_RETURN_NONE;
    const int64_t n = index.defined() ? index.numel() : x.size(0), out = gated ? rows_w / 2 : rows_w;
    if (!good_table(table, x, n, e)) Py_RETURN_NONE;
    at::Tensor y;
    {
        const WithoutLock no_lock;
        const at::NoGradGuard no_grad;
        const c10::OptionalDeviceGuard guard(x.device());
        const int dtype = dtype_code(x);
        y = at::empty({n, out}, x.options());
        // the rows' integers, their scales, and what the product wants, in one piece
        const bool round_first = entry.int8_rounds_rows(e, n, d, out, (int)gated, dtype) == 0;
        const int64_t q_bytes = round_first ? n * whole_d : 0, s_bytes = round_first ? (n * 4 + 15) / 16 * 16 : 0;
        const int64_t ws_bytes = entry.int8_bytes(e, n, d, out, (int)gated, dtype);
        const at::Tensor space = at::empty({q_bytes + s_bytes + ws_bytes}, x.options().dtype(at::kByte));
        char *q = (char *)pointer(space), *s = q + q_bytes, *ws = ws_bytes ? s + s_bytes : nullptr;
        const int64_t *row_index = (const int64_t *)pointer(index);
        void *stream = stream_of(x);
        if (round_first)
            ok(entry.quantize_rows(pointer(x), x.stride(0), row_index, index_div, x.size(0), q, whole_d, s, pointer(table), pointer(y), out * x.element_size(),
                                   n, d, dtype, stream));
        ok(entry.linear_int8(round_first ? q : pointer(x), round_first ? whole_d : x.stride(0), round_first ? s : nullptr, round_first ? nullptr : row_index,
                             index_div, round_first ? n : x.size(0), pointer(weight), by_row, by_expert, pointer(scale), pointer(bias), pointer(y),
                             pointer(table), e, n, d, out, (int)gated, (int)activation, dtype, ws, ws_bytes, stream));
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}
