"""Refusals of gated experts and of experts in 8-bit integers, without a GPU: in Python, and at the C entry points, which check before they enqueue
anything."""
import pytest
import torch

from fastermoe_amd import FMoEGatedMLP, FMoEPositionwiseFF, FMoETransformerMLP, _lib, fmoe_native, functions

lib = _lib.load()
EINVAL, ELIMIT, EWORKSPACE = -1, -2, -4
P = 16   # a pointer that is never followed: the refusal comes first


def _gated_forward(x=P, w1=P, b1=P, w2=P, b2=P, pre=P, mid=P, y=P, table=P, e=2, rows=4, d=8, h=16, dt=_lib.BF16, act=_lib.ACT_SILU, ws=P, wsb=1 << 50):
    return lib.fmoe_gated_mlp_forward(x, w1, b1, w2, b2, pre, mid, y, table, e, rows, d, h, dt, act, ws, wsb, None)


def _gated_backward(gy=P, x=P, w1=P, w2=P, pre=P, mid=P, gx=P, gw1=P, gb1=P, gw2=P, gb2=P, table=P, e=2, rows=4, d=8, h=16, dt=_lib.BF16, act=_lib.ACT_SILU,
                    ws=P, wsb=1 << 50):
    return lib.fmoe_gated_mlp_backward(gy, x, w1, w2, pre, mid, gx, gw1, gb1, gw2, gb2, table, e, rows, d, h, dt, act, ws, wsb, None)


def _quantize(x=P, ldx=8, index=None, div=1, x_rows=4, q=P, ldq=16, scale=P, table=None, tail=None, tail_bytes=0, rows=4, d=8, dt=_lib.BF16):
    return lib.fmoe_quantize_rows(x, ldx, index, div, x_rows, q, ldq, scale, table, tail, tail_bytes, rows, d, dt, None)


def _linear(x=P, ldx=32, xs=P, index=None, div=1, x_rows=4, w=P, ldw=32, wes=512, ws_=P, bias=P, y=P, table=P, e=2, rows=64, d=32, out=16, gated=0,
            act=_lib.ACT_NONE, dt=_lib.BF16, ws=None, wsb=0):
    return lib.fmoe_linear_int8(x, ldx, xs, index, div, x_rows, w, ldw, wes, ws_, bias, y, table, e, rows, d, out, gated, act, dt, ws, wsb, None)


@pytest.mark.parametrize("call,arguments,code", [
    (_gated_forward, dict(dt=_lib.F64), EINVAL), (_gated_forward, dict(act=3), EINVAL), (_gated_forward, dict(act=-1), EINVAL),
    (_gated_forward, dict(act=5), EINVAL), (_gated_forward, dict(e=0), EINVAL), (_gated_forward, dict(rows=-1), EINVAL), (_gated_forward, dict(d=0), EINVAL),
    (_gated_forward, dict(h=0), EINVAL), (_gated_forward, dict(x=None), EINVAL), (_gated_forward, dict(w1=None), EINVAL),
    (_gated_forward, dict(w2=None), EINVAL), (_gated_forward, dict(mid=None), EINVAL), (_gated_forward, dict(y=None), EINVAL),
    (_gated_forward, dict(table=None), EINVAL), (_gated_forward, dict(table=20), EINVAL), (_gated_forward, dict(rows=1 << 31), ELIMIT),
    (_gated_forward, dict(d=(1 << 28) + 1), ELIMIT), (_gated_forward, dict(h=(1 << 28) + 1), ELIMIT), (_gated_forward, dict(e=(1 << 24) + 1), ELIMIT),
    (_gated_forward, dict(dt=_lib.F32, d=1 << 15, h=1 << 14), ELIMIT), (_gated_forward, dict(dt=_lib.F32, x=20), EINVAL),
    (_gated_forward, dict(dt=_lib.F32, b1=24), EINVAL), (_gated_forward, dict(dt=_lib.F32, d=7, ws=None), EWORKSPACE),
    (_gated_forward, dict(dt=_lib.F32, h=15, wsb=1000), EWORKSPACE), (_gated_forward, dict(dt=_lib.F32, h=15, ws=24), EWORKSPACE),
    (_gated_backward, dict(dt=_lib.F64), EINVAL), (_gated_backward, dict(act=9), EINVAL), (_gated_backward, dict(gw1=None), EINVAL),
    (_gated_backward, dict(gw2=None), EINVAL), (_gated_backward, dict(gy=None), EINVAL), (_gated_backward, dict(pre=None), EINVAL),
    (_gated_backward, dict(mid=None), EINVAL), (_gated_backward, dict(table=None), EINVAL), (_gated_backward, dict(ws=None), EWORKSPACE),
    (_gated_backward, dict(wsb=7), EWORKSPACE), (_gated_backward, dict(ws=20), EWORKSPACE), (_gated_backward, dict(rows=1 << 31), ELIMIT),
    (_gated_backward, dict(dt=_lib.F32, gx=20), EINVAL),
    (_quantize, dict(dt=_lib.F64), EINVAL), (_quantize, dict(rows=-1), EINVAL), (_quantize, dict(d=-1), EINVAL), (_quantize, dict(x_rows=3), EINVAL),
    (_quantize, dict(index=P, div=0), EINVAL), (_quantize, dict(tail=P), EINVAL), (_quantize, dict(ldq=8), EINVAL), (_quantize, dict(ldq=24), EINVAL),
    (_quantize, dict(d=17, ldx=17), EINVAL), (_quantize, dict(q=24), EINVAL), (_quantize, dict(x=None), EINVAL), (_quantize, dict(q=None), EINVAL),
    (_quantize, dict(scale=None), EINVAL), (_quantize, dict(d=(1 << 28) + 1), ELIMIT), (_quantize, dict(rows=1 << 31, x_rows=1 << 31), ELIMIT),
    (_linear, dict(dt=_lib.F64), EINVAL), (_linear, dict(act=3), EINVAL), (_linear, dict(e=0), EINVAL), (_linear, dict(d=0), EINVAL),
    (_linear, dict(out=0), EINVAL), (_linear, dict(d=131073, ldx=131088, ldw=131088), ELIMIT), (_linear, dict(rows=1 << 31), ELIMIT),
    (_linear, dict(ldw=1 << 23), ELIMIT), (_linear, dict(ldw=1 << 20, out=1 << 11), ELIMIT), (_linear, dict(ldx=1 << 23), ELIMIT),
    (_linear, dict(d=16, ldw=16, wes=0, out=(1 << 21) + 8), ELIMIT), (_linear, dict(d=16, ldw=16, wes=0, out=(1 << 20) + 4, dt=_lib.F32), ELIMIT),
    (_linear, dict(ldx=16), EINVAL), (_linear, dict(ldx=40), EINVAL), (_linear, dict(ldw=16), EINVAL), (_linear, dict(ldw=40), EINVAL),
    (_linear, dict(wes=500), EINVAL), (_linear, dict(wes=-512), EINVAL), (_linear, dict(x=None), EINVAL), (_linear, dict(w=None), EINVAL),
    (_linear, dict(ws_=None), EINVAL), (_linear, dict(y=None), EINVAL), (_linear, dict(table=None), EINVAL), (_linear, dict(x=20), EINVAL),
    (_linear, dict(w=20), EINVAL), (_linear, dict(bias=20), EINVAL), (_linear, dict(y=20), EINVAL), (_linear, dict(ws_=20), EINVAL),
    (_linear, dict(xs=None), EINVAL),                                              # (more rows than a product rounds itself)
    (_linear, dict(index=P), EINVAL), (_linear, dict(xs=None, rows=4, x_rows=3), EINVAL), (_linear, dict(xs=None, rows=4, index=P, div=0), EINVAL),
    (_linear, dict(xs=None, rows=4, out=18), EINVAL),                              # (columns of the kernels that do not)
])
def test_c_entries_refuse(call, arguments, code):
    assert call(**arguments) == code
    word = {"_gated_forward": "gated_mlp_forward", "_gated_backward": "gated_mlp_backward", "_quantize": "quantize_rows", "_linear": "linear_int8"}
    assert word[call.__name__].encode() in lib.fmoe_last_error()


def test_nothing_to_do_is_no_error():
    assert _gated_forward(rows=0, x=None, y=None, mid=None, ws=None, wsb=0) == 0
    assert _quantize(rows=0, x_rows=0, x=None, q=None, scale=None) == 0
    assert _linear(rows=0, x=None, y=None) == 0


def test_workspaces_and_who_rounds():
    sizes = lambda dt, keep=0, d=8, h=16: lib.fmoe_gated_mlp_forward_workspace_bytes(2, 64, d, h, dt, _lib.ACT_SILU, keep)
    assert sizes(_lib.BF16) == 0 and sizes(_lib.F64) == 0
    assert sizes(_lib.F32, d=7) >= 4 * (64 * 8 + 2 * 2 * 16 * 8 + 2 * 8 * 16)       # the padded copies
    assert sizes(_lib.F32, 1, d=7) > sizes(_lib.F32, 0, d=7) - 64 * 2 * 16 * 4 - 256
    assert lib.fmoe_gated_mlp_backward_workspace_bytes(2, 64, 8, 16, _lib.BF16, _lib.ACT_SILU) >= 64 * 32 * 2
    rounds = lambda rows, d, out=64, e=4: lib.fmoe_linear_int8_rounds_rows(e, rows, d, out, 0, _lib.BF16)
    assert rounds(1, 8192) == 1 and rounds(1, 8193) == 0 and rounds(16, 512) == 1 and rounds(16, 513) == 0 and rounds(17, 16) == 0 and rounds(2, 64, 63) == 0
    assert lib.fmoe_linear_int8_workspace_bytes(4, 0, 8, 8, 0, _lib.BF16) == 0


def test_python_refuses_tensors_of_the_host():
    x, w1, w2 = torch.zeros(3, 8), torch.zeros(2, 32, 8), torch.zeros(2, 8, 16)
    with pytest.raises((TypeError, ValueError)):
        functions.gated_mlp(x, torch.tensor([1, 2]), w1, None, w2, None, torch.nn.SiLU())
    with pytest.raises(ValueError, match="CUDA"):
        functions.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        functions.linear_int8(x, torch.tensor([1, 2]), torch.zeros(2, 16, 8, dtype=torch.int8), torch.ones(2, 16))
    with pytest.raises(ValueError, match="CUDA"):
        fmoe_native.linear_int8(x, None, torch.zeros(2, 16, 8, dtype=torch.int8), torch.ones(2, 16))
    with pytest.raises(TypeError):
        fmoe_native.quantize_rows([1.0])


@pytest.mark.parametrize("activation", [torch.nn.Tanh(), torch.nn.GELU(approximate="tanh"), torch.nn.LeakyReLU(), 3, 17])
def test_activations_that_the_block_does_not_have(activation):
    with pytest.raises((ValueError, NotImplementedError, TypeError)):
        functions.gated_mlp(torch.zeros(3, 8), torch.tensor([1, 2]), torch.zeros(2, 32, 8), None, torch.zeros(2, 8, 16), None, activation)


def test_gradients_of_8_bit_products_are_refused():
    x = torch.zeros(3, 8, requires_grad=True)
    with pytest.raises(NotImplementedError):
        functions.linear_int8(x, torch.tensor([1, 2]), torch.zeros(2, 16, 8, dtype=torch.int8), torch.ones(2, 16))


@pytest.mark.parametrize("which", ["inp", "bias", "weight_scale"])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_of_8_bit_products_are_refused(which, grad):
    """Forward mode: a dual tensor requires no gradient, and torch.no_grad leaves its tangent."""
    tensors = {"inp": torch.zeros(3, 8), "bias": torch.zeros(2, 16), "weight_scale": torch.ones(2, 16)}
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        tensors[which] = torch.autograd.forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises(NotImplementedError, match="tangents"):
            functions.linear_int8(tensors["inp"], torch.tensor([1, 2]), torch.zeros(2, 16, 8, dtype=torch.int8), tensors["weight_scale"], tensors["bias"])


def test_transforms_of_8_bit_products_are_refused():
    scale, weight = torch.ones(2, 16), torch.zeros(2, 16, 8, dtype=torch.int8)
    call = lambda x: functions.linear_int8(x, torch.tensor([1, 2]), weight, scale)
    for transformed in (lambda: torch.func.jvp(call, (torch.zeros(3, 8),), (torch.ones(3, 8),)), lambda: torch.func.vmap(call)(torch.zeros(4, 3, 8)),
                        lambda: torch.func.grad(lambda x: call(x).sum())(torch.zeros(3, 8))):
        with torch.no_grad(), pytest.raises(NotImplementedError, match="transforms"):
            transformed()


def test_tangents_that_are_nobody_elses_business():
    """A level of forward mode alone refuses nothing: what is wrong with the call is said (its tensors are the host's)."""
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="CUDA"):
        functions.linear_int8(torch.zeros(3, 8), torch.tensor([1, 2]), torch.zeros(2, 16, 8, dtype=torch.int8), torch.ones(2, 16))


def test_layers_have_the_parameters_of_their_kind():
    layer = FMoEGatedMLP(num_expert=3, d_model=8, d_hidden=20, top_k=2)
    assert layer.experts.htoh4.weight.shape == (3, 40, 8) and layer.experts.h4toh.weight.shape == (3, 8, 20)
    plain = FMoETransformerMLP(num_expert=3, d_model=8, d_hidden=20)
    assert plain.experts.htoh4.weight.shape == (3, 20, 8)
    block = FMoEPositionwiseFF(num_expert=3, d_model=8, d_hidden=20, top_k=2, gated=True)
    assert any(p.shape == (3, 40, 8) for p in block.parameters())


class _Adapter(torch.nn.Module):
    """A linear with something added, and a ``weight`` of its own."""

    def __init__(self, linear):
        super().__init__()
        self.linear = linear

    weight = property(lambda self: self.linear.weight)
    bias = property(lambda self: self.linear.bias)

    def forward(self, inp, fwd_expert_count):
        return self.linear(inp, fwd_expert_count) + 1


@pytest.mark.parametrize("kind", [FMoETransformerMLP, FMoEGatedMLP])
@pytest.mark.parametrize("name", ["htoh4", "h4toh"])
def test_replaced_linears_are_not_held_in_8_bits(kind, name):
    """What a module in a linear's place, or a hook, adds to its weight's product would be lost.  (The refusal comes before anything needs a GPU.)"""
    def adapter(experts):
        setattr(experts, name, _Adapter(getattr(experts, name)))

    def own_forward(experts):
        linear = getattr(experts, name)
        linear.forward = lambda inp, count: type(linear).forward(linear, inp, count) + 1

    def hook(experts):
        getattr(experts, name).register_forward_hook(lambda module, args, out: out + 1)

    def pre_hook(experts):
        getattr(experts, name).register_forward_pre_hook(lambda module, args: None)

    for change in (adapter, own_forward, hook, pre_hook):
        layer = kind(num_expert=3, d_model=8, d_hidden=20)
        change(layer.experts)
        before = layer.experts
        with pytest.raises(TypeError, match=name):
            layer.quantize_experts()
        assert layer.experts is before


@pytest.mark.parametrize("dt,d,h,taken", [
    (_lib.F32, 8, 16, 1), (_lib.F32, 1 << 15, 8059, 1), (_lib.F32, 1 << 15, 8060, 0), (_lib.F32, 1 << 14, 1 << 14, 0), (_lib.F32, 16, (1 << 19) - 3, 1),
    (_lib.F32, 16, (1 << 19) - 2, 0), (_lib.F32, 1 << 20, 4, 1), (_lib.F32, (1 << 20) + 1, 4, 0), (_lib.BF16, 1 << 14, 1 << 15, 1),
    (_lib.F16, 1 << 28, 1 << 28, 1), (_lib.F16, (1 << 28) + 1, 4, 0), (_lib.BF16, 4, (1 << 28) + 1, 0), (_lib.BF16, 4, 1 << 60, 0)])
def test_sizes_of_gated_experts(dt, d, h, taken):
    """What the question says is what the call does (which says next that there is no x)."""
    assert lib.fmoe_gated_mlp_supported(d, h, dt) == taken
    assert _gated_forward(x=None, dt=dt, d=d, h=h) == (EINVAL if taken else ELIMIT)
    assert _gated_backward(x=None, dt=dt, d=d, h=h) == (EINVAL if taken else ELIMIT)


def test_sizes_that_nothing_has():
    assert lib.fmoe_gated_mlp_supported(0, 8, _lib.BF16) == lib.fmoe_gated_mlp_supported(8, 0, _lib.BF16) == lib.fmoe_gated_mlp_supported(8, 8, _lib.F64) == 0
    assert lib.fmoe_linear_int8_supported(0, 8, 0, _lib.BF16) == lib.fmoe_linear_int8_supported(8, 0, 0, _lib.BF16) == 0
    assert lib.fmoe_linear_int8_supported(8, 8, 0, _lib.F64) == 0
    assert not fmoe_native.gated_mlp_supported(torch.float64) and not fmoe_native.linear_int8_supported(8, 8, False, torch.float64)


@pytest.mark.parametrize("dt,d,out,gated,taken", [
    (_lib.BF16, 32, 16, 0, 1), (_lib.BF16, 131072, 16383, 0, 1), (_lib.BF16, 131072, 16384, 0, 0), (_lib.BF16, 131072, 8192, 1, 0),
    (_lib.BF16, 131072, 8191, 1, 1), (_lib.BF16, 131073, 4, 0, 0), (_lib.F16, 16, 1 << 21, 1, 1), (_lib.F16, 16, (1 << 21) + 1, 0, 0),
    (_lib.F32, 16, 1 << 20, 0, 1), (_lib.F32, 16, (1 << 20) + 1, 0, 0)])
def test_sizes_of_8_bit_products(dt, d, out, gated, taken):
    assert lib.fmoe_linear_int8_supported(d, out, gated, dt) == taken
    whole = -(-d // 16) * 16
    assert _linear(x=None, dt=dt, d=d, ldx=whole, ldw=whole, wes=whole, out=out, gated=gated) == (EINVAL if taken else ELIMIT)


@pytest.mark.parametrize("call", [_gated_forward, _gated_backward])
@pytest.mark.parametrize("dt", [_lib.BF16, _lib.F16])
def test_pre_holds_float32_whatever_the_type(call, dt):
    """An address that 16-bit elements could have and float32 cannot."""
    assert call(pre=18, dt=dt) == EINVAL
    assert b"float32" in lib.fmoe_last_error()
