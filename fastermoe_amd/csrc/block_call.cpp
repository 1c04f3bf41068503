// Layer norm and the gate's balance loss as autograd nodes, and rows kept in 8 bits, from Python's tensors to the enqueued kernels (host code).
//
// Their kernels take 3 to 20 us on a small training step's tensors.  As Python nodes, a forward and a backward took 138 and 90 us to enqueue,
// most of it in the backward's thread; a product and its gradient in torch itself take 46.  The calls for rows in 8 bits took 9 us each from
// Python, the kernels of a small batch 5.  What a call takes is decided here; None sends it the way through Python, which says what is wrong with its tensors.
#include "block_call.hpp"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cmath>
#include <cstdint>
#include <optional>

#include "../../include/fmoe_hip.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the library's entry points, which Python has loaded (bind)
struct Entries {
    decltype(&fmoe_last_error) last_error;
    decltype(&fmoe_layer_norm_forward) norm_forward;
    decltype(&fmoe_layer_norm_backward) norm_backward;
    decltype(&fmoe_layer_norm_backward_workspace_bytes) norm_bytes;
    decltype(&fmoe_balance_loss_forward) balance_forward;
    decltype(&fmoe_balance_loss_backward) balance_backward;
    decltype(&fmoe_balance_loss_workspace_bytes) balance_bytes;
    decltype(&fmoe_act_checkpoint_forward) checkpoint_forward;
    decltype(&fmoe_act_checkpoint_backward) checkpoint_backward;
} entry = {};

int dtype_code(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FMOE_F32;
        case at::kBFloat16: return FMOE_BF16;
        case at::kHalf: return FMOE_F16;
        default: return -1;
    }
}
void *pointer(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *floats(const at::Tensor &t) { return (float *)pointer(t); }
void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void ok(int rc) { TORCH_CHECK(rc == FMOE_OK, "libfmoe_hip error ", rc, ": ", entry.last_error()); }
at::Tensor same(const at::Tensor &t) { return at::empty(t.sizes(), t.options()); }
// rows of adjacent elements, as the kernels read them
at::Tensor as_rows(const at::Tensor &t) { return t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t; }

using Maybe = std::optional<at::Tensor>;   // (what a node takes where there may be no tensor)
Maybe maybe(const at::Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; }

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &given, const Maybe &of_residual, const Maybe &of_weight,
                                 const Maybe &of_bias, double eps, bool keep) {
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Tensor residual = of_residual.value_or(at::Tensor()), weight = of_weight.value_or(at::Tensor()), bias = of_bias.value_or(at::Tensor());
        const c10::OptionalDeviceGuard guard(given.device());
        const at::Tensor inp = as_rows(given), other = residual.defined() ? as_rows(residual) : residual;
        const int64_t n = inp.size(0), d = inp.size(1);
        const at::Tensor out = at::empty({n, d}, inp.options()), total = other.defined() ? same(out) : at::Tensor();
        at::Tensor stats;   // the rows' means, then their reciprocal deviations
        if (keep) stats = at::empty({2, n}, inp.options().dtype(at::kFloat));
        const at::Tensor &param = weight.defined() ? weight : bias;
        ok(entry.norm_forward(pointer(inp), inp.stride(0), pointer(other), other.defined() ? other.stride(0) : 0, pointer(weight), pointer(bias),
                              pointer(total), pointer(out), floats(stats), keep ? floats(stats) + n : nullptr, n, d, eps, dtype_code(inp),
                              param.defined() ? dtype_code(param) : dtype_code(inp), stream_of(inp)));
        if (keep) {
            ctx->save_for_backward({total.defined() ? total : given, stats, weight, bias});   // (a copy has no history for a second derivative)
            ctx->saved_data["eps"] = eps;
            ctx->set_materialize_grads(false);
        }
        return total.defined() ? variable_list{out, total} : variable_list{out};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &rows = saved[0], &stats = saved[1], &weight = saved[2], &bias = saved[3];
        const at::Tensor total = grads.size() > 1 ? grads[1] : at::Tensor();
        // (asked by the tensors that there were)
        const size_t has_r = grads.size() > 1, has_w = weight.defined();
        const bool need_x = ctx->needs_input_grad(0), need_r = has_r && ctx->needs_input_grad(1);
        const bool need_w = has_w && ctx->needs_input_grad(1 + has_r), need_b = bias.defined() && ctx->needs_input_grad(1 + has_r + has_w);
        at::Tensor x, w, b;
        if (!grads[0].defined()) {
            if (total.defined()) {
                x = total;
                if (need_w) w = at::zeros_like(weight);
                if (need_b) b = at::zeros_like(bias);
            }
        } else if (at::GradMode::is_enabled()) {   // (a backward that is to be differentiated again needs torch's operators)
            const at::Tensor t = rows.to(at::kFloat), g = grads[0].to(at::kFloat);
            const at::Tensor centred = t - t.mean(1, true), rstd = (centred * centred).mean(1, true).add(ctx->saved_data["eps"].toDouble()).rsqrt();
            const at::Tensor hat = centred * rstd, a = weight.defined() ? g * weight.to(at::kFloat) : g;
            x = rstd * (a - a.mean(1, true) - hat * (a * hat).mean(1, true));
            if (total.defined()) x = x + total.to(at::kFloat);
            x = x.to(rows.scalar_type());
            if (need_w) w = (g * hat).sum(0).to(weight.scalar_type());
            if (need_b) b = g.sum(0).to(bias.scalar_type());
        } else {
            const c10::OptionalDeviceGuard guard(rows.device());
            const at::Tensor gy = as_rows(grads[0]), gs = total.defined() ? as_rows(total) : total, at_rows = as_rows(rows);
            const int64_t n = rows.size(0), d = rows.size(1);
            const at::Tensor held = stats.contiguous();
            if (need_x || need_r) x = at::empty({n, d}, rows.options());
            if (need_w) w = same(weight);
            if (need_b) b = same(bias);
            const int64_t bytes = need_w || need_b ? entry.norm_bytes(n, d) : 0;
            const at::Tensor space = bytes ? at::empty({bytes}, rows.options().dtype(at::kByte)) : at::Tensor();
            const at::Tensor &param = weight.defined() ? weight : bias;
            ok(entry.norm_backward(pointer(gy), gy.stride(0), pointer(gs), gs.defined() ? gs.stride(0) : 0, pointer(at_rows), at_rows.stride(0),
                                   floats(held), floats(held) + n, pointer(weight), pointer(x), pointer(w), pointer(b), n, d, dtype_code(rows),
                                   param.defined() ? dtype_code(param) : dtype_code(rows), pointer(space), bytes, stream_of(rows)));
        }
        const at::Tensor none;
        return {need_x ? x : none, need_r ? x : none, need_w ? w : none, need_b ? b : none, none, none};
    }
};

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &given, const at::Tensor &index, const Maybe &of_mask, int64_t per_slot) {
        at::AutoDispatchBelowADInplaceOrView below;
        const at::Tensor mask = of_mask.value_or(at::Tensor());
        const c10::OptionalDeviceGuard guard(given.device());
        const at::Tensor logits = given.contiguous(), idx = index.contiguous();
        const int64_t n = logits.size(0), e = logits.size(1), bytes = entry.balance_bytes(n, e);
        const at::TensorOptions f32 = logits.options().dtype(at::kFloat);
        const at::Tensor loss = at::empty({}, f32), count = at::empty({e}, f32.dtype(at::kLong)), prob = at::empty({e}, f32);
        const at::Tensor slope = at::empty({e + 1}, f32), space = at::empty({bytes}, f32.dtype(at::kByte));
        ok(entry.balance_forward(pointer(logits), (int64_t *)pointer(idx), pointer(mask), n, e, n ? idx.numel() / n : 1, dtype_code(logits),
                                 (int)per_slot, floats(loss), (int64_t *)pointer(count), floats(prob), floats(slope), pointer(space), bytes,
                                 stream_of(logits)));
        ctx->save_for_backward({given, mask, slope});   // (as above)
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({count});
        return {loss, count, prob};
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &logits = saved[0], &mask = saved[1], &slope = saved[2], &of_loss = grads[0], &of_prob = grads[2];
        at::Tensor grad;
        if (of_loss.defined() || of_prob.defined()) {
            if (at::GradMode::is_enabled()) {   // (as above)
                const int64_t e = logits.size(1);
                at::Tensor u;
                if (of_loss.defined()) u = of_loss * slope.narrow(0, 0, e);
                if (of_prob.defined()) u = u.defined() ? u + of_prob * slope.select(0, e) : of_prob * slope.select(0, e);
                at::Tensor left_out = logits.eq(-INFINITY).all(1);
                if (mask.defined()) left_out = left_out.logical_or(mask);
                left_out = left_out.unsqueeze(1);
                const at::Tensor p = at::softmax(logits.to(at::kFloat).masked_fill(left_out, 0), 1).masked_fill(left_out, 0);
                grad = (p * (u - (p * u).sum(1, true))).to(logits.scalar_type());
            } else {
                const c10::OptionalDeviceGuard guard(logits.device());
                auto dense = [](const at::Tensor &t) { return t.defined() ? t.contiguous() : t; };
                const at::Tensor gl = dense(of_loss), gp = dense(of_prob), held = logits.contiguous(), by = slope.contiguous(), out = dense(mask);
                grad = same(held);
                ok(entry.balance_backward(pointer(held), pointer(out), floats(by), floats(gl), floats(gp), pointer(grad), logits.size(0),
                                          logits.size(1), dtype_code(logits), stream_of(logits)));
            }
        }
        return {grad, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// The interpreter's lock, given back while this lives: an allocation may wait for the device, a launch for a full queue
struct WithoutLock {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutLock() { PyEval_RestoreThread(state); }
};

// The first N arguments as tensors (undefined for None); false, with an exception set, where one is neither
template <size_t N> bool tensors(PyObject *const *args, std::array<at::Tensor, N> &t) {
    for (size_t i = 0; i < N; ++i) {
        if (args[i] == Py_None) continue;
        if (!THPVariable_Check(args[i])) {
            PyErr_SetString(PyExc_TypeError, "tensors or None");
            return false;
        }
        t[i] = THPVariable_Unpack(args[i]);
    }
    return true;
}
// The number behind them; false, with an exception set, where it is none
bool number(PyObject *arg, long &n) {
    n = PyLong_AsLong(arg);
    return n != -1 || !PyErr_Occurred();
}
// (a tensor without memory of its own, as some wrappers are, has a null pointer, which a parameter that is left out has too)
bool on_gpu(const at::Tensor &t) {
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg() && t.has_storage() &&
           (t.numel() == 0 || t.storage().data() != nullptr);
}

}  // namespace

PyObject *fmoe_block_bind(PyObject *, PyObject *args) {
    unsigned long long a[9];
    if (!PyArg_ParseTuple(args, "KKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8])) return nullptr;
    auto set = [&](auto &fn, int i) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(static_cast<uintptr_t>(a[i])); };
    set(entry.last_error, 0);
    set(entry.norm_forward, 1);
    set(entry.norm_backward, 2);
    set(entry.norm_bytes, 3);
    set(entry.balance_forward, 4);
    set(entry.balance_backward, 5);
    set(entry.balance_bytes, 6);
    set(entry.checkpoint_forward, 7);
    set(entry.checkpoint_backward, 8);
    Py_RETURN_NONE;
}

// layer_norm(inp, residual, weight, bias, eps): the result of the rows' norm, with the sum behind it where there is a residual; None where the call does
// not take these tensors
PyObject *fmoe_block_layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 5 || entry.norm_forward == nullptr) {
        PyErr_SetString(PyExc_TypeError, "layer_norm: 5 arguments, after bind_block");
        return nullptr;
    }
    std::array<at::Tensor, 4> t;
    if (!tensors(args, t)) return nullptr;
    const auto &[inp, residual, weight, bias] = t;
    const double eps = PyFloat_AsDouble(args[4]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    if (!on_gpu(inp) || inp.dim() != 2 || inp.size(1) == 0 || dtype_code(inp) < 0 || !(eps >= 0) || std::isinf(eps)) Py_RETURN_NONE;
    if (residual.defined() && (!on_gpu(residual) || residual.device() != inp.device() || residual.scalar_type() != inp.scalar_type() ||
                               residual.sizes() != inp.sizes()))
        Py_RETURN_NONE;
    for (const at::Tensor *p : {&weight, &bias})
        if (p->defined() && (!on_gpu(*p) || p->device() != inp.device() || !p->is_contiguous() || p->sizes() != at::IntArrayRef({inp.size(1)}) ||
                             (p->scalar_type() != inp.scalar_type() && p->scalar_type() != at::kFloat)))
            Py_RETURN_NONE;
    if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type()) Py_RETURN_NONE;
    variable_list out;
    {
        const WithoutLock no_lock;
        bool keep = false;
        for (const at::Tensor &p : t) keep |= p.defined() && p.requires_grad();
        out = LayerNorm::apply(inp, maybe(residual), maybe(weight), maybe(bias), eps, keep && at::GradMode::is_enabled());
    }
    if (out.size() == 1) return THPVariable_Wrap(std::move(out[0]));
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(out[0])), THPVariable_Wrap(std::move(out[1])));
    END_HANDLE_TH_ERRORS
}

// balance_loss(logits, topk_idx, mask, per_slot): (loss, counts, prob); None where the call does not take these tensors
PyObject *fmoe_block_balance_loss(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 4 || entry.balance_forward == nullptr) {
        PyErr_SetString(PyExc_TypeError, "balance_loss: 4 arguments, after bind_block");
        return nullptr;
    }
    std::array<at::Tensor, 3> t;
    if (!tensors(args, t)) return nullptr;
    const auto &[logits, idx, mask] = t;
    const long per_slot = PyLong_AsLong(args[3]);
    if (per_slot == -1 && PyErr_Occurred()) return nullptr;
    if (!on_gpu(logits) || !on_gpu(idx) || logits.dim() != 2 || dtype_code(logits) < 0 || idx.device() != logits.device() || idx.scalar_type() != at::kLong)
        Py_RETURN_NONE;
    const int64_t n = logits.size(0), e = logits.size(1);
    if (idx.dim() > 1 && idx.size(0) != n) Py_RETURN_NONE;
    if (e < 1 || e > 8192 || n > INT32_MAX / 8 || idx.numel() > INT32_MAX || idx.numel() % (n ? n : 1) != 0 || (n == 0) != (idx.numel() == 0)) Py_RETURN_NONE;
    if (mask.defined() && (!on_gpu(mask) || mask.device() != logits.device() || mask.scalar_type() != at::kBool || mask.numel() != n || !mask.is_contiguous()))
        Py_RETURN_NONE;
    variable_list out;
    {
        const WithoutLock no_lock;
        out = BalanceLoss::apply(logits, idx, maybe(mask), (int64_t)(per_slot != 0));
    }
    return Py_BuildValue("NNN", THPVariable_Wrap(std::move(out[0])), THPVariable_Wrap(std::move(out[1])), THPVariable_Wrap(std::move(out[2])));
    END_HANDLE_TH_ERRORS
}

namespace {

constexpr int64_t kScaleElems = 32;
// rows that are kept in 8 bits
bool keeps(const at::Tensor &x, long activation) {
    return on_gpu(x) && x.dim() == 2 && x.is_contiguous() && dtype_code(x) >= 0 && activation >= FMOE_ACT_NONE && activation <= FMOE_ACT_GELU;
}
bool no_or_table(const at::Tensor &t, const at::Tensor &x) {
    return !t.defined() || (on_gpu(t) && t.device() == x.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() >= 8);
}
PyObject *wrap_or_none(at::Tensor t) {
    if (t.defined()) return THPVariable_Wrap(std::move(t));
    Py_RETURN_NONE;
}

}  // namespace

// act_checkpoint_forward(x, table, activation, with_act, with_held): (y or None, held, scale or None, None); None where the call does not take these tensors
PyObject *fmoe_block_checkpoint_forward(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 5 || entry.checkpoint_forward == nullptr) {
        PyErr_SetString(PyExc_TypeError, "act_checkpoint_forward: 5 arguments, after bind_block");
        return nullptr;
    }
    std::array<at::Tensor, 2> t;
    long activation, with_act, with_held;
    if (!tensors(args, t) || !number(args[2], activation) || !number(args[3], with_act) || !number(args[4], with_held)) return nullptr;
    const auto &[x, table] = t;
    if (!keeps(x, activation) || !no_or_table(table, x)) Py_RETURN_NONE;
    at::Tensor y, held, scale;
    {
        const WithoutLock no_lock;
        const at::NoGradGuard no_grad;
        const c10::OptionalDeviceGuard guard(x.device());
        const int64_t n = x.size(0), d = x.size(1);
        if (with_held) {
            held = at::empty({n, d}, x.options().dtype(at::kFloat8_e4m3fn));
            scale = at::empty({n, (d + kScaleElems - 1) / kScaleElems}, x.options().dtype(at::kFloat8_e8m0fnu));
        }
        if (with_act) y = at::empty({n, d}, x.options());
        ok(entry.checkpoint_forward(pointer(x), pointer(y), pointer(held), pointer(scale), pointer(table), n, d, dtype_code(x), (int)activation,
                                    stream_of(x)));
    }
    return Py_BuildValue("NNN", wrap_or_none(std::move(y)), wrap_or_none(std::move(held)), wrap_or_none(std::move(scale)));
    END_HANDLE_TH_ERRORS
}

// act_checkpoint_backward(grad, held, scale, table, activation, with_mid, in_place): (grad_x, mid or None); None where the call does not take these tensors
PyObject *fmoe_block_checkpoint_backward(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 7 || entry.checkpoint_backward == nullptr) {
        PyErr_SetString(PyExc_TypeError, "act_checkpoint_backward: 7 arguments, after bind_block");
        return nullptr;
    }
    std::array<at::Tensor, 4> t;
    long activation, with_mid, in_place;
    if (!tensors(args, t) || !number(args[4], activation) || !number(args[5], with_mid) || !number(args[6], in_place)) return nullptr;
    const auto &[grad, held, scale, table] = t;
    if (!keeps(grad, activation) || !no_or_table(table, grad)) Py_RETURN_NONE;
    const int64_t n = grad.size(0), d = grad.size(1);
    auto is = [&](const at::Tensor &kept, at::ScalarType type, int64_t columns) {
        return on_gpu(kept) && kept.device() == grad.device() && kept.scalar_type() == type && kept.is_contiguous() &&
               kept.sizes() == at::IntArrayRef({n, columns});
    };
    if (!is(held, at::kFloat8_e4m3fn, d) || !is(scale, at::kFloat8_e8m0fnu, (d + kScaleElems - 1) / kScaleElems)) Py_RETURN_NONE;
    at::Tensor grad_x, mid;
    {
        const WithoutLock no_lock;
        const at::NoGradGuard no_grad;
        const c10::OptionalDeviceGuard guard(grad.device());
        grad_x = in_place ? grad : at::empty({n, d}, grad.options());
        if (with_mid) mid = at::empty({n, d}, grad.options());
        ok(entry.checkpoint_backward(pointer(grad), pointer(held), pointer(scale), pointer(grad_x), pointer(mid), pointer(table), n, d,
                                     dtype_code(grad), (int)activation, stream_of(grad)));
    }
    return Py_BuildValue("NN", THPVariable_Wrap(std::move(grad_x)), wrap_or_none(std::move(mid)));
    END_HANDLE_TH_ERRORS
}
