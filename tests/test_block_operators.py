"""Refusals of the layer norm, the balance loss and the rows kept in 8 bits, without a GPU: in Python, and at the C entry points, which check before
they enqueue anything."""
import pytest
import torch

from fastermoe_amd import _lib, fmoe_native, functions

lib = _lib.load()
EINVAL, ELIMIT, EWORKSPACE = -1, -2, -4
P = 16   # a pointer that is never followed: the refusal comes first


def _norm_forward(x=P, xs=8, r=None, rs=0, w=P, b=P, s=None, y=P, mean=P, rstd=P, rows=4, d=8, eps=1e-5, dt=_lib.BF16, pt=_lib.BF16):
    return lib.fmoe_layer_norm_forward(x, xs, r, rs, w, b, s, y, mean, rstd, rows, d, eps, dt, pt, None)


def _norm_backward(gy=P, gys=8, gs=None, gss=0, x=P, xs=8, mean=P, rstd=P, w=P, gx=P, gw=P, gb=P, rows=4, d=8, dt=_lib.BF16, pt=_lib.BF16, ws=P,
                   wsb=1 << 30):
    return lib.fmoe_layer_norm_backward(gy, gys, gs, gss, x, xs, mean, rstd, w, gx, gw, gb, rows, d, dt, pt, ws, wsb, None)


def _balance(logits=P, idx=P, mask=None, n=4, e=8, k=2, dt=_lib.F32, per=0, loss=P, count=P, prob=P, slope=P, ws=P, wsb=1 << 30):
    return lib.fmoe_balance_loss_forward(logits, idx, mask, n, e, k, dt, per, loss, count, prob, slope, ws, wsb, None)


def _checkpoint(x=P, y=P, held=P, scale=P, rows=4, d=8, dt=_lib.BF16, act=_lib.ACT_GELU):
    return lib.fmoe_act_checkpoint_forward(x, y, held, scale, None, rows, d, dt, act, None)


def _checkpoint_back(g=P, held=P, scale=P, gx=P, mid=P, rows=4, d=8, dt=_lib.BF16, act=_lib.ACT_GELU):
    return lib.fmoe_act_checkpoint_backward(g, held, scale, gx, mid, None, rows, d, dt, act, None)


@pytest.mark.parametrize("call,arguments,code", [
    (_norm_forward, dict(dt=_lib.F64, pt=_lib.F64), EINVAL), (_norm_forward, dict(dt=9), EINVAL),
    (_norm_forward, dict(dt=_lib.F32, pt=_lib.BF16), EINVAL), (_norm_forward, dict(dt=_lib.F16, pt=_lib.BF16), EINVAL),
    (_norm_forward, dict(rows=-1), EINVAL), (_norm_forward, dict(d=0), EINVAL), (_norm_forward, dict(xs=-1), EINVAL),
    (_norm_forward, dict(r=P, s=P, rs=-8), EINVAL), (_norm_forward, dict(eps=-1e-5), EINVAL), (_norm_forward, dict(eps=float("nan")), EINVAL),
    (_norm_forward, dict(x=None), EINVAL), (_norm_forward, dict(y=None), EINVAL), (_norm_forward, dict(r=P), EINVAL),
    (_norm_forward, dict(mean=None), EINVAL), (_norm_forward, dict(rows=1 << 31), ELIMIT), (_norm_forward, dict(d=(1 << 28) + 1), ELIMIT),
    (_norm_backward, dict(dt=_lib.F64, pt=_lib.F64), EINVAL), (_norm_backward, dict(gy=None), EINVAL), (_norm_backward, dict(x=None), EINVAL),
    (_norm_backward, dict(rstd=None), EINVAL), (_norm_backward, dict(gys=-1), EINVAL), (_norm_backward, dict(d=0), EINVAL),
    (_norm_backward, dict(ws=None), EWORKSPACE), (_norm_backward, dict(wsb=7), EWORKSPACE), (_norm_backward, dict(rows=1 << 31), ELIMIT),
    (_balance, dict(dt=_lib.F64), EINVAL), (_balance, dict(n=-1), EINVAL), (_balance, dict(e=0), EINVAL), (_balance, dict(k=0), EINVAL),
    (_balance, dict(per=2), EINVAL), (_balance, dict(logits=None), EINVAL), (_balance, dict(idx=None), EINVAL), (_balance, dict(loss=None), EINVAL),
    (_balance, dict(slope=None), EINVAL), (_balance, dict(e=8193), ELIMIT), (_balance, dict(n=1 << 30), ELIMIT),
    (_balance, dict(n=1 << 28, k=8), ELIMIT), (_balance, dict(ws=None), EWORKSPACE), (_balance, dict(wsb=3), EWORKSPACE),
    (_checkpoint, dict(dt=_lib.F64), EINVAL), (_checkpoint, dict(act=3), EINVAL), (_checkpoint, dict(act=-1), EINVAL),
    (_checkpoint, dict(rows=-1), EINVAL), (_checkpoint, dict(d=-1), EINVAL), (_checkpoint, dict(x=None), EINVAL), (_checkpoint, dict(held=None), EINVAL),
    (_checkpoint, dict(scale=None), EINVAL), (_checkpoint, dict(rows=1 << 31), ELIMIT), (_checkpoint, dict(d=(1 << 28) + 1), ELIMIT),
    (_checkpoint_back, dict(dt=_lib.F64), EINVAL), (_checkpoint_back, dict(g=None), EINVAL), (_checkpoint_back, dict(gx=None), EINVAL),
    (_checkpoint_back, dict(g=None, gx=None, mid=None), EINVAL), (_checkpoint_back, dict(held=None), EINVAL), (_checkpoint_back, dict(act=7), EINVAL),
])
def test_c_entries_refuse(call, arguments, code):
    assert call(**arguments) == code
    assert call.__name__.split("_")[1].encode() in lib.fmoe_last_error()


def test_rows_longer_than_a_launch_sums():
    assert _norm_forward(d=(1 << 26) + 1) == ELIMIT and _norm_backward(d=(1 << 26) + 1) == ELIMIT


def test_launches_of_too_many_threads():
    """2^32 and more: 16 of them for 128 elements kept in 8 bits, 64 for a token of more than 1024 experts."""
    assert _checkpoint(rows=1 << 28, d=128) == ELIMIT and _checkpoint_back(rows=1 << 28, d=100) == ELIMIT
    assert lib.fmoe_balance_loss_backward(P, None, P, P, None, P, (1 << 26) + 1, 2000, _lib.F32, None) == ELIMIT


def test_c_entries_take_nothing_to_do():
    assert _norm_forward(rows=0) == 0 and _checkpoint(rows=0) == 0 and _checkpoint(d=0) == 0 and _checkpoint_back(rows=0) == 0
    assert _norm_backward(rows=0, gw=None, gb=None, ws=None, wsb=0) == 0
    assert lib.fmoe_balance_loss_backward(P, None, P, P, None, P, 0, 8, _lib.F32, None) == 0
    assert lib.fmoe_balance_loss_backward(None, None, P, P, None, P, 4, 8, _lib.F32, None) == EINVAL
    assert lib.fmoe_layer_norm_backward_workspace_bytes(-1, 8) == 0 and lib.fmoe_balance_loss_workspace_bytes(5, 0) == 0


def test_functions_refuse_what_the_kernels_do_not_take():
    x = torch.randn(4, 8)
    for call in (lambda: functions.layer_norm(x), lambda: functions.add_layer_norm(x, x), lambda: functions.act_checkpoint(x, torch.nn.GELU()),
                 lambda: functions.balance_loss(x, torch.zeros(4, 1, dtype=torch.int64))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="per must be"):
        functions.balance_loss(x, torch.zeros(4, 1, dtype=torch.int64), per="expert")
    with pytest.raises(ValueError, match="residual"):
        functions.add_layer_norm(x, x[:2])
    with pytest.raises(NotImplementedError):
        functions.act_checkpoint(x, torch.tanh)
    with pytest.raises(ValueError):
        functions.layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError):
        functions.act_checkpoint(torch.tensor(1.0), None)


class _Wrapper(torch.Tensor):
    """A tensor that says where it is and has no memory of its own."""
    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32, device="cuda:0"):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError("nothing to see here")


def test_tensors_without_memory():
    x = _Wrapper(4, 8)
    held, scale = _Wrapper(4, 8, dtype=torch.float8_e4m3fn), _Wrapper(4, 1, dtype=torch.float8_e8m0fnu)
    for call in (lambda: fmoe_native.layer_norm_forward(x, None, None, None, 1e-5), lambda: fmoe_native._norm_params(x, _Wrapper(8), None),
                 lambda: fmoe_native.balance_loss_forward(x, x, None, False), lambda: fmoe_native._balance_args(x, _Wrapper(4, dtype=torch.bool)),
                 lambda: fmoe_native.act_checkpoint_forward(x, 0), lambda: fmoe_native.act_checkpoint_backward(x, held, scale, 0)):
        with pytest.raises(ValueError, match="memory"):
            call()


@pytest.mark.gpu
def test_parameters_without_memory(device):
    x, idx = torch.randn(4, 8, device=device), torch.zeros(4, 1, dtype=torch.int64, device=device)
    for call in (lambda: functions.layer_norm(x, _Wrapper(8)), lambda: functions.layer_norm(x, None, _Wrapper(8)),
                 lambda: fmoe_native.balance_loss_forward(x, idx, _Wrapper(4, dtype=torch.bool), False),
                 lambda: fmoe_native.act_checkpoint_forward(x, 0, table=_Wrapper(16, dtype=torch.int32))):
        with pytest.raises(ValueError, match="memory"):
            call()


@pytest.mark.gpu
def test_indices_of_tokens_the_other_way_round(device):
    x, idx = torch.randn(6, 8, device=device), torch.zeros(2, 6, dtype=torch.int64, device=device)
    for call in (lambda: functions.balance_loss(x, idx), lambda: fmoe_native.balance_loss_forward(x, idx, None, False)):
        with pytest.raises(ValueError, match="first dimension"):
            call()
    assert torch.equal(functions.balance_loss(x, idx.view(-1))[1], functions.balance_loss(x, idx.view(6, 2))[1])


@pytest.mark.gpu
def test_refusals_on_the_gpu(device):
    x = torch.randn(4, 8, device=device)
    idx = torch.zeros(4, 1, dtype=torch.int64, device=device)
    w = torch.randn(8, device=device)
    cases = [
        (TypeError, lambda: functions.layer_norm(x.double())), (TypeError, lambda: functions.layer_norm(x, w.bfloat16())),
        (TypeError, lambda: functions.layer_norm(x.half(), w.bfloat16())), (TypeError, lambda: functions.layer_norm(x.half(), w.half(), w)),
        (ValueError, lambda: functions.layer_norm(x, w[:7])), (ValueError, lambda: functions.layer_norm(x, w.cpu())),
        (ValueError, lambda: functions.layer_norm(x, torch.randn(16, device=device)[::2])), (ValueError, lambda: functions.layer_norm(x, eps=-1.0)),
        (ValueError, lambda: functions.layer_norm(x, eps=float("nan"))), (ValueError, lambda: functions.layer_norm(x[:, :0])),
        (TypeError, lambda: functions.add_layer_norm(x, x.half())), (ValueError, lambda: functions.add_layer_norm(x, x.cpu())),
        (ValueError, lambda: functions.balance_loss(x.double(), idx)), (TypeError, lambda: functions.balance_loss(x, idx.int())),
        (ValueError, lambda: functions.balance_loss(x[:0], idx)), (ValueError, lambda: functions.balance_loss(x, idx[:3])), (ValueError, lambda: functions.balance_loss(x, idx[:0])),
        (ValueError, lambda: functions.balance_loss(x, idx.cpu())), (ValueError, lambda: functions.balance_loss(x, idx, mask=idx[:3])),
        (ValueError, lambda: functions.balance_loss(x[0], idx)), (ValueError, lambda: functions.balance_loss(torch.zeros(1, 8193, device=device), idx[:1])),
        (TypeError, lambda: functions.act_checkpoint(x.double(), None)), (ValueError, lambda: functions.act_checkpoint(x, 5)),
        (TypeError, lambda: fmoe_native.act_checkpoint_backward(x, x, x, 0)),
    ]
    for n, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            print(n)
    _, held, scale = fmoe_native.act_checkpoint_forward(x, 0)
    for bad in ((held[:3].contiguous(), scale), (held, scale[:3].contiguous())):
        with pytest.raises(ValueError):
            fmoe_native.act_checkpoint_backward(x, *bad, 0)
    with pytest.raises(ValueError):
        fmoe_native.act_checkpoint_forward(x, 0, table=torch.zeros(3, dtype=torch.int32, device=device))


@pytest.mark.gpu
def test_under_inference_mode(device):
    x, r = torch.randn(30, 64, device=device), torch.randn(30, 64, device=device)
    w = torch.randn(64, device=device, requires_grad=True)
    idx = x.topk(2, dim=1).indices

    def run():
        return (functions.layer_norm(x, w), *functions.add_layer_norm(x, r, w, w), *functions.balance_loss(x, idx), functions.act_checkpoint(x, torch.nn.GELU()))

    want = run()
    with torch.inference_mode():
        got = run()
        inner = functions.layer_norm(x + 0, w)      # (of a tensor made here)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0].requires_grad and torch.equal(inner, got[0])


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(device):
    """Each call's workspace is its own: forward and backward passes that overlap give what they give alone."""
    gen = torch.Generator(device=device).manual_seed(4)
    jobs = [torch.randn(n, 512, device=device, generator=gen) for n in (4000, 3000)]

    def run(x):
        leaf, w = x.detach().requires_grad_(True), torch.ones(512, device=device, requires_grad=True)
        y = functions.layer_norm(leaf, w)
        loss, counts, prob = functions.balance_loss(leaf, idx[x.shape[0]])
        z = functions.act_checkpoint(leaf, torch.nn.GELU())
        return (y.detach(), loss.detach(), counts, z.detach()) + torch.autograd.grad([y, loss, z], [leaf, w], [x, torch.ones((), device=device), x])

    idx = {x.shape[0]: x.topk(2, dim=1).indices for x in jobs}
    want = [run(x) for x in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [None] * len(jobs)
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(jobs[i])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_rows_in_8_bits_or_their_activation():
    """Held numbers and scales come together, and something has to be wanted."""
    assert _checkpoint(y=None, held=None, scale=None) == EINVAL and _checkpoint(held=None, scale=None, rows=0) == 0
    with pytest.raises(ValueError, match="wanted"):
        fmoe_native.act_checkpoint_forward(torch.randn(4, 8), _lib.ACT_GELU, with_act=False, with_held=False)


def test_rows_without_features_of_any_leading_shape():
    """As rows of two dimensions are: the layer norm refuses them, the rows kept in 8 bits have nothing to keep."""
    assert functions._as_rows(torch.zeros(2, 3, 0)).shape == (6, 0) and functions._as_rows(torch.zeros(0, 3, 4)).shape == (0, 4)
    assert functions._as_rows(torch.zeros(5)).shape == (1, 5) and functions._as_rows(torch.zeros(0)).shape == (1, 0)


@pytest.mark.gpu
def test_rows_without_features_on_the_gpu(device):
    x = torch.zeros(2, 3, 0, device=device, requires_grad=True)
    y = functions.act_checkpoint(x, torch.nn.GELU())
    assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    with pytest.raises(ValueError, match="features"):
        functions.layer_norm(x)
