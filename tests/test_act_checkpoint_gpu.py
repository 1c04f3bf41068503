"""Rows kept in 8 bits and the backward from what was kept, against the definition in float64.

The numbers held have to be the definition's exactly: dividing by a power of two rounds nothing.  GELU's terms are off by 4e-7 (its erf formula by
0.75e-7 of the distribution function, an exponential, a reciprocal and a few products by some 2^-23 of what is at most 1/2), its slope by 1e-6."""
import math

import pytest
import torch

from fastermoe_amd import _lib, fmoe_native, functions

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU}


def two_to(b):
    """2^b in float64, exactly (``torch.ldexp`` goes through a power function in float32)."""
    return ((b.long() + 1023) << 52).view(torch.float64)


def hold(x):
    """``(held values over the scale, scale)`` in float64 of rows ``x``, block by block from the definition; NaN for what is not finite."""
    n, d = x.shape
    top = torch.finfo(x.dtype).max
    x = torch.nn.functional.pad(x.double(), (0, -d % 32)).view(n, -1, 32)
    most = torch.where(x.isfinite(), x.abs(), 0.0).amax(2, keepdim=True)
    _, b = torch.frexp(most.clamp(min=2.0 ** -140))
    b = b - 10                                          # 448 2^b is below the block's largest; two steps more are not
    for _ in range(3):
        b = torch.where(448.0 * two_to(b) < most, b + 1, b)
    b = b.clamp(min=-126)
    v = x * two_to(-b)
    _, e = torch.frexp(v.nan_to_num(0, 0, 0))
    step = two_to((e - 1).clamp(min=-6) - 3)
    q = torch.round(v / step) * step
    over = (q * two_to(b)).abs() > top
    q = torch.where(over & v.isfinite(), torch.sign(v) * 240.0, q)
    q = torch.where(x.isfinite(), q, float("nan"))
    flat = lambda t: t.reshape(n, -1)[:, :d]
    return flat(q), two_to(b).view(n, -1), flat(q * two_to(b))


def act64(v, act):
    if act == "gelu":
        return v * torch.special.ndtr(v), torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "relu":
        return torch.where(v < 0, 0.0, v), torch.where(v.isnan(), v, (v > 0).double())
    return v, torch.where(v.isnan(), v, 1.0)


def near(got, ref, slack, what):
    assert got.shape == ref.shape
    assert torch.equal(got.isnan(), ref.isnan()), what
    info = torch.finfo(got.dtype)
    limit = ref.abs().clamp(min=info.smallest_normal) * (info.eps / 2) + slack
    off = (got.double() - ref).abs()
    ok = (off <= limit) | ref.isnan() | (got.double() == ref) | ((got.double().abs() == float("inf")) & (ref.abs() > info.max * (1 - info.eps / 4)))
    assert bool(ok.all()), f"{what}: {float((off / limit)[~ok].max()):.3g} times what they may be off"


def check(x, act, dtype=None):
    dtype = x.dtype
    n, d = x.shape
    y, held, scale = fmoe_native.act_checkpoint_forward(x, CODES[act])
    q64, s64, v64 = hold(x)
    assert held.dtype == torch.float8_e4m3fn and scale.dtype == torch.float8_e8m0fnu
    got = held.float().double()
    assert torch.equal(got.isnan(), q64.isnan()) and torch.equal(got.nan_to_num(0), q64.nan_to_num(0))
    assert torch.equal(scale.float().double(), s64)
    ref, _ = act64(x.double(), act)
    near(y, ref, 4e-7 * x.double().abs() if act == "gelu" else 0.0, "y")
    g = torch.randn(n, d, device=x.device).to(dtype)
    grad, mid = fmoe_native.act_checkpoint_backward(g, held, scale, CODES[act])
    mid64, slope = act64(v64, act)
    near(mid, mid64, 4e-7 * v64.abs() if act == "gelu" else 0.0, "mid")
    near(grad, g.double() * slope, 1e-6 * g.double().abs() if act == "gelu" else 0.0, "grad")
    alone, none = fmoe_native.act_checkpoint_backward(g, held, scale, CODES[act], with_mid=False)
    assert none is None and torch.equal(alone.nan_to_num(7), grad.nan_to_num(7))
    none, held2, scale2 = fmoe_native.act_checkpoint_forward(x, CODES[act], with_act=False)
    assert none is None and torch.equal(held2.view(torch.uint8), held.view(torch.uint8)) and torch.equal(scale2.view(torch.uint8), scale.view(torch.uint8))
    over, mid2 = fmoe_native.act_checkpoint_backward(g.clone(), held, scale, CODES[act], in_place=True)
    assert torch.equal(over.nan_to_num(7), grad.nan_to_num(7)) and torch.equal(mid2.nan_to_num(7), mid.nan_to_num(7))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["gelu", "relu", "none"])
@pytest.mark.parametrize("n,d", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 8), (7, 100), (1, 4096), (64, 64), (129, 1302), (1000, 512), (33, 2048), (300, 328)])
def test_sizes(n, d, act, dtype, device):
    torch.manual_seed(n * d)
    check((torch.randn(n, d, device=device) * torch.exp(torch.randn(n, 1, device=device))).to(TYPES[dtype]), act)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_magnitude(dtype, device):
    """Blocks from the smallest numbers of the type to its largest, ties and the edges of the scale's rule among them."""
    t = TYPES[dtype]
    info = torch.finfo(t)
    top = math.log2(info.max)
    low = {"f32": -149, "bf16": -133, "f16": -24}[dtype]
    e = torch.linspace(low, top, 400, device=device, dtype=torch.float64)
    x = torch.exp2(e)[:, None] * (torch.rand(400, 64, device=device, dtype=torch.float64) * 2 - 1)
    check(x.clamp(info.min, info.max).to(t), "none")
    # 448 2^k and its neighbours as the largest of a block; every e4m3 number and every half way between two
    grid = torch.arange(0, 127, device=device, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    half = (grid[1:] + grid[:-1]) / 2
    both = torch.cat([grid, half, -half])
    block = torch.nn.functional.pad(both, (0, -both.numel() % 31)).view(-1, 31)
    rows = [torch.cat([torch.full_like(block[:, :1], m), block], 1) for m in (448.0, -448.0)]
    for k in (0, -5, 6):
        check((torch.cat(rows) * 2.0 ** k).to(t), "none")
    edge = torch.tensor([1.75, 1.7421875, 1.7578125, 1.0, 1.9921875], device=device, dtype=torch.float64)
    check((edge[:, None] * torch.linspace(-1, 1, 32, device=device, dtype=torch.float64)).to(t), "none")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["gelu", "relu", "none"])
def test_the_largest_numbers_and_what_is_not_finite(act, dtype, device):
    t = TYPES[dtype]
    info = torch.finfo(t)
    x = torch.randn(6, 96, device=device).to(t)
    x[0, 3], x[0, 40] = info.max, info.min
    x[1, :32] = info.max
    x[1, 32:64] = info.max * 0.93
    x[2, 5], x[2, 6], x[3, 70] = float("inf"), -float("inf"), float("nan")
    x[4, :32] = float("nan")
    x[5, 32:64] = 0
    x[5, 64:] = -0.0
    check(x, act)


def test_only_the_rows_there_are(device):
    """Rows behind the experts' last one are neither read into results nor written."""
    counts = torch.tensor([5, 0, 9], dtype=torch.int64, device=device)
    rows, d = 20, 100
    table = fmoe_native.segment_table(counts, rows)
    x = torch.randn(rows, d, device=device, dtype=torch.bfloat16)
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    y, grad, mid = (torch.full((rows, d), 7.0, device=device, dtype=torch.bfloat16) for _ in range(3))
    held, scale = torch.full((rows, d), 9, device=device, dtype=torch.uint8), torch.full((rows, 4), 9, device=device, dtype=torch.uint8)
    _lib.check(lib.fmoe_act_checkpoint_forward(x.data_ptr(), y.data_ptr(), held.data_ptr(), scale.data_ptr(), table.data_ptr(), rows, d,
                                               _lib.BF16, _lib.ACT_GELU, st))
    _lib.check(lib.fmoe_act_checkpoint_backward(x.data_ptr(), held.data_ptr(), scale.data_ptr(), grad.data_ptr(), mid.data_ptr(), table.data_ptr(),
                                                rows, d, _lib.BF16, _lib.ACT_GELU, st))
    want = fmoe_native.act_checkpoint_forward(x[:14], _lib.ACT_GELU)
    back = fmoe_native.act_checkpoint_backward(x[:14].contiguous(), *want[1:], _lib.ACT_GELU)
    assert torch.equal(y[:14], want[0]) and bool((y[14:] == 7).all())
    assert torch.equal(held[:14], want[1].view(torch.uint8)) and bool((held[14:] == 9).all())
    assert torch.equal(scale[:14], want[2].view(torch.uint8)) and bool((scale[14:] == 9).all())
    assert torch.equal(grad[:14], back[0]) and bool((grad[14:] == 7).all())
    assert torch.equal(mid[:14], back[1]) and bool((mid[14:] == 7).all())


def test_unaligned_tensors(device):
    """Rows that begin anywhere in memory."""
    for d in (64, 50):
        for shift in (1, 3):
            flat = torch.randn(20 * d + shift, device=device).to(torch.bfloat16)
            x = flat[shift:].view(20, d)
            y, held, scale = fmoe_native.act_checkpoint_forward(x, _lib.ACT_GELU)
            want = fmoe_native.act_checkpoint_forward(x.clone(), _lib.ACT_GELU)
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((y, held, scale), want))
            back = fmoe_native.act_checkpoint_backward(x, held, scale, _lib.ACT_GELU)
            ref = fmoe_native.act_checkpoint_backward(x.clone(), held, scale, _lib.ACT_GELU)
            assert all(torch.equal(a, b) for a, b in zip(back, ref))


@pytest.mark.parametrize("act", [torch.nn.GELU(), torch.nn.ReLU(), None])
def test_through_autograd(act, device):
    """The derivative where the numbers held are, by differences of the activation in float64."""
    x = torch.randn(4, 6, 72, device=device, requires_grad=True)
    y = functions.act_checkpoint(x, act)
    g = torch.randn_like(x)
    grad, = torch.autograd.grad(y, x, g)
    name = "none" if act is None else "gelu" if isinstance(act, torch.nn.GELU) else "relu"
    near(y.detach(), act64(x.detach().double(), name)[0], 1e-6, "y")
    v = hold(x.detach().reshape(-1, 72))[2].view_as(x)
    step = 1e-6
    slope = (act64(v + step, name)[0] - act64(v - step, name)[0]) / (2 * step)
    smooth = v.abs() > 1e-5          # (a ReLU at 0 has no two-sided derivative)
    assert torch.allclose(grad.double()[smooth], (g.double() * slope)[smooth], rtol=1e-4, atol=1e-5)
    assert torch.equal(functions.act_checkpoint(x.detach().transpose(0, 1), act), y.detach().transpose(0, 1))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(functions.act_checkpoint(x, act).sum(), x, create_graph=True)[0].sum(), x)


def test_no_rows(device):
    x = torch.empty(0, 40, device=device, requires_grad=True)
    y = functions.act_checkpoint(x, torch.nn.GELU())
    g, = torch.autograd.grad(y, x, torch.empty(0, 40, device=device))
    assert y.shape == g.shape == (0, 40)


def test_offsets_beyond_32_bits(device):
    """More than 2^31 elements: the last rows like the same rows alone."""
    n, d = 150001, 14336
    x = torch.empty(n, d, dtype=torch.bfloat16, device=device)
    x[:4].normal_()
    x[-5:].normal_()
    x[4:-5] = 0.5
    y, held, scale = fmoe_native.act_checkpoint_forward(x, _lib.ACT_RELU)
    want = fmoe_native.act_checkpoint_forward(x[-5:].clone(), _lib.ACT_RELU)
    assert torch.equal(y[-5:], want[0]) and torch.equal(held[-5:].view(torch.uint8), want[1].view(torch.uint8))
    assert torch.equal(scale[-5:].view(torch.uint8), want[2].view(torch.uint8))
    grad, mid = fmoe_native.act_checkpoint_backward(x, held, scale, _lib.ACT_RELU)
    back = fmoe_native.act_checkpoint_backward(x[-5:].clone(), *want[1:], _lib.ACT_RELU)
    assert torch.equal(grad[-5:], back[0]) and torch.equal(mid[-5:], back[1])


def test_another_stream_and_a_graph(device):
    x, g = (torch.randn(200, 320, device=device, dtype=torch.bfloat16) for _ in range(2))

    def step():
        leaf = x.detach().requires_grad_(True)
        y = functions.act_checkpoint(leaf, torch.nn.GELU())
        return y.detach(), torch.autograd.grad(y, leaf, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(warm, step()))
    del warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(torch.randn(200, 320, device=device))
        g.copy_(torch.randn(200, 320, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k


def test_called_from_python_the_same(device, monkeypatch):
    """Without the extension module: the same bits."""
    x, g = (torch.randn(40, 100, device=device, dtype=torch.float16) for _ in range(2))

    def run():
        y, held, scale = fmoe_native.act_checkpoint_forward(x, _lib.ACT_GELU)
        return (y, held.view(torch.uint8), scale.view(torch.uint8)) + fmoe_native.act_checkpoint_backward(g, held, scale, _lib.ACT_GELU)

    native = run()
    monkeypatch.setattr(_lib, "_layer_call", None)
    assert all(torch.equal(a, b) for a, b in zip(native, run()))
    for act in CODES:
        check(x, act)


def _otherwise(t):
    """An equal tensor whose elements lie in another order."""
    if t.dim() < 2 or t.shape[0] < 2:
        return t
    return t.view(torch.uint8).t().contiguous().t().view(t.dtype) if t.element_size() == 1 else t.transpose(0, 1).contiguous().transpose(0, 1)


def test_saved_tensors_may_come_back_otherwise(device):
    """Saved-tensor hooks hand back what is held in another order."""
    x = torch.randn(33, 96, device=device, requires_grad=True)
    dy = torch.randn(33, 96, device=device)
    want, = torch.autograd.grad(functions.act_checkpoint(x, torch.nn.GELU()), x, dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _otherwise):
        y = functions.act_checkpoint(x, torch.nn.GELU())
    got, = torch.autograd.grad(y, x, dy)
    assert torch.equal(got, want)


def test_experts_saved_tensors_may_come_back_otherwise(device):
    """The same of the experts' node over rows that are counted on the host."""
    from fastermoe_amd.functions import MOEExpertMLPCheckpointed
    torch.manual_seed(2)
    x = torch.randn(40, 64, device=device)
    counts = torch.tensor([13, 0, 27])
    params = [torch.randn(s, device=device) * 0.1 for s in ((3, 96, 64), (3, 96), (3, 64, 96), (3, 64))]
    dy = torch.randn(40, 64, device=device)

    def run(hook):
        leaves = [t.detach().requires_grad_(True) for t in (x, *params)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
            out = MOEExpertMLPCheckpointed.apply(leaves[0], counts, *leaves[1:], _lib.ACT_GELU)
        return torch.autograd.grad(out, leaves, dy)

    assert all(torch.equal(a, b) for a, b in zip(run(lambda t: t), run(lambda t: _otherwise(t) if t.is_cuda else t)))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("act", ["gelu", "relu", "none"])
@pytest.mark.parametrize("d", [96, 50])
def test_nothing_is_held_where_nothing_is_differentiated(d, act, native, device, monkeypatch):
    """One allocation, the result's, whose bits are those of a call that is differentiated."""
    if not native:
        monkeypatch.setattr(_lib, "_layer_call", None)
    x = torch.randn(70, d, device=device)
    want = functions.act_checkpoint(x.clone().requires_grad_(True), CODES[act]).detach()

    def count(call):
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        out = call()
        return out, torch.cuda.memory_stats()["allocation.all.allocated"] - before

    with torch.no_grad():
        out, n = count(lambda: functions.act_checkpoint(x.requires_grad_(True), CODES[act]))
    assert n == 1 and torch.equal(out, want)
    out, n = count(lambda: functions.act_checkpoint(x.detach(), CODES[act]))
    assert n == 1 and torch.equal(out, want) and not out.requires_grad
    with torch.inference_mode():
        out, n = count(lambda: functions.act_checkpoint(x, CODES[act]))
    assert n == 1 and torch.equal(out, want)


def test_the_node_by_itself(device):
    """``ActCheckpoint.apply`` with and without the last argument."""
    x = torch.randn(20, 64, device=device, requires_grad=True)
    want, = torch.autograd.grad(functions.act_checkpoint(x, CODES["gelu"]).sum(), x)
    for more in ((), (True,)):
        got, = torch.autograd.grad(functions.ActCheckpoint.apply(x, CODES["gelu"], *more).sum(), x)
        assert torch.equal(got, want)
