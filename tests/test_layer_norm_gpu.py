"""Layer norm of token rows, of their sum with a residual, and the gradients against the definition in float64.

A result may be off by half a step of its type and by what float32 does on the way: every value passes through sums of ``d`` terms,
of which a lane adds ``d / 64`` one after the other before some sixteen more steps, so each is off by at most
``c = (16 + d / 64) 2^-24`` of the magnitudes that it was made of."""
import pytest
import torch

from fastermoe_amd import _lib, functions

pytestmark = pytest.mark.gpu
ULP32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half_step(ref, dtype):
    info = torch.finfo(dtype)
    return ref.abs().clamp(min=info.smallest_normal) * (info.eps / 2)


def _check(got, ref, slack, what):
    assert got.shape == ref.shape, what
    d = (got.double() - ref).abs()
    limit = _half_step(ref, got.dtype) + slack
    bad = ~(d <= limit)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} are off, by {float((d / limit).nan_to_num(float('inf')).max()):.2f} times what they may"


def _reference(s, w, b, eps):
    """What the gradients and the bounds need, in float64."""
    d = s.shape[1]
    mean = s.mean(1, keepdim=True)
    rstd = ((s - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (s - mean) * rstd
    reach = s.abs().amax(1, keepdim=True) * rstd    # what is rounded where the mean is taken off
    c = (16 + d / 64) * ULP32
    one = torch.ones(d, dtype=torch.float64, device=s.device)
    w = one if w is None else w.detach().double()
    b = 0 * one if b is None else b.detach().double()
    return mean, rstd, h, reach, c, w, b


def _check_forward(y, s, w, b, eps, what=""):
    mean, rstd, h, reach, c, w, b = _reference(s, w, b, eps)
    _check(y, h * w + b, c * ((h.abs() + reach) * w.abs() + b.abs()), what + "y")


def _check_backward(grads, s, w, b, eps, dy, ds, what=""):
    mean, rstd, h, reach, c, w64, _ = _reference(s, w, b, eps)
    a = dy * w64
    gx = rstd * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True)) + ds
    hr = h.abs() + reach
    slack = 2 * c * (rstd * (a.abs() + a.abs().mean(1, keepdim=True) + hr * (a.abs() * hr).mean(1, keepdim=True)) + ds.abs())
    _check(grads[0], gx, slack, what + "grad_x")
    n = s.shape[0]
    chain = (160 + n / 64) * ULP32      # the sums over the rows
    if w is not None:
        _check(grads[1], (dy * h).sum(0), c * (dy.abs() * hr).sum(0) + chain * (dy * h).abs().sum(0), what + "grad_w")
    if b is not None:
        _check(grads[2], dy.sum(0), chain * dy.abs().sum(0), what + "grad_b")


def _run(n, d, dtype, residual, params, eps=1e-5, gap=0, seed=0, offset=0.0, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device=device, generator=gen)
    dtype = TYPES[dtype]
    x = (normal(n, d + gap) * torch.exp(normal(n, 1)) + offset).to(dtype)[:, :d].detach().requires_grad_(True)
    r = normal(n, d).to(dtype).requires_grad_(True) if residual else None
    w = b = None
    if params != "none":
        ptype = torch.float32 if params == "f32" else dtype
        w = (1 + 0.3 * normal(d)).to(ptype).requires_grad_(True)
        b = (0.2 * normal(d)).to(ptype).requires_grad_(True)
    dy, ds = normal(n, d).to(dtype), normal(n, d).to(dtype)
    leaves = [t for t in (x, r, w, b) if t is not None]
    if residual:
        y, s = functions.add_layer_norm(x, r, w, b, eps)
        want = (x.detach().float() + r.detach().float()).to(dtype)
        assert torch.equal(s, want)
        grads = dict(zip([id(t) for t in leaves], torch.autograd.grad([y, s], leaves, [dy, ds])))
        assert torch.equal(grads[id(x)], grads[id(r)])
        total, ds = s.detach().double(), ds.double()
    else:
        y = functions.layer_norm(x, w, b, eps)
        grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
        total, ds = x.detach().double(), torch.zeros(n, d, dtype=torch.float64, device=device)
    assert y.dtype == dtype and y.is_contiguous()
    _check_forward(y.detach(), total, w, b, eps)
    _check_backward([grads[id(x)], grads.get(id(w)), grads.get(id(b))], total, w, b, eps, dy.double(), ds)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 2), (1, 1024), (7, 37), (64, 64), (509, 500), (65, 1302), (33, 4096), (5, 8192), (3, 16400),
                                 (2, 40001), (1030, 512), (4099, 96)])
def test_sizes(n, d, residual, dtype, device):
    _run(n, d, dtype, residual, "same")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("params", ["none", "f32"])
def test_parameters(params, dtype, device):
    _run(130, 515, dtype, True, params)
    _run(130, 1024, dtype, False, params)


@pytest.mark.parametrize("gap", [1, 8, 10])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_a_wider_tensor(gap, dtype, device):
    _run(77, 1024, dtype, True, "same", gap=gap)
    _run(77, 51, dtype, False, "same", gap=gap)


def test_rows_far_from_zero(device):
    _run(40, 2048, "f32", False, "same", offset=300.0)
    _run(40, 2048, "bf16", True, "same", offset=50.0)


def test_one_parameter_alone_and_gradients_that_are_not_wanted(device):
    x = torch.randn(20, 72, device=device)
    dy = torch.randn(20, 72, device=device)
    for has in ("weight", "bias"):
        p = torch.randn(72, device=device, requires_grad=True)
        w, b = (p, None) if has == "weight" else (None, p)
        y = functions.layer_norm(x, w, b)
        _check_forward(y.detach(), x.double(), w, b, 1e-5, has + " ")
        g, = torch.autograd.grad(y, p, dy)
        h = _reference(x.double(), None, None, 1e-5)[2]
        assert torch.allclose(g.double(), (dy.double() * h).sum(0) if has == "weight" else dy.double().sum(0), rtol=1e-4, atol=1e-5)
    x.requires_grad_(True)
    w = torch.randn(72, device=device)   # (not differentiated)
    g, = torch.autograd.grad(functions.layer_norm(x, w), x, dy)
    _check_backward([g, None, None], x.detach().double(), None, None, 1e-5, (dy * w).double(), torch.zeros_like(x).double())


def test_gradients_against_differences(device):
    """Directional derivatives in float64 of the definition, by central differences, against the kernels' gradients."""
    torch.manual_seed(5)
    x, r, w, b, dy, ds = (torch.randn(*s, device=device, dtype=torch.float64) for s in ((6, 40), (6, 40), (40,), (40,), (6, 40), (6, 40)))

    def value(x, r, w, b):
        s = x + r
        h = (s - s.mean(1, keepdim=True)) * (s.var(1, correction=0, keepdim=True) + 1e-5).rsqrt()
        return ((h * w + b) * dy).sum() + (s * ds).sum()

    leaves = [t.float().requires_grad_(True) for t in (x, r, w, b)]
    y, s = functions.add_layer_norm(*leaves)
    grads = torch.autograd.grad([y, s], leaves, [dy.float(), ds.float()])
    at = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        v = torch.randn_like(at[i])
        step = 1e-5
        up, down = (value(*[t + (k * step * v if j == i else 0) for j, t in enumerate(at)]) for k in (1, -1))
        want = float((up - down) / (2 * step))
        got = float((g.double() * v).sum())
        assert abs(got - want) <= 1e-4 * float((g.double() * v).abs().sum()), i


def test_constant_and_zero_rows(device):
    """Nothing to normalise: the deviation is 0, the rows become the bias, and eps alone scales the gradient."""
    w, b = torch.randn(96, device=device), torch.randn(96, device=device)
    for value in (0.0, 2.5):
        x = torch.full((4, 96), value, device=device, requires_grad=True)
        y = functions.layer_norm(x, w, b, 1e-5)
        assert torch.equal(y.detach(), b.expand(4, 96))
        dy = torch.randn(4, 96, device=device)
        g, = torch.autograd.grad(y, x, dy)
        a = (dy * w).double()
        _check(g, (a - a.mean(1, keepdim=True)) * 1e-5 ** -0.5, 20 * ULP32 * 1e-5 ** -0.5 * (a.abs() + a.abs().mean(1, keepdim=True)), "grad")


def test_nan_and_infinity_stay_in_their_rows(device):
    x = torch.randn(5, 300, device=device, dtype=torch.bfloat16)
    clean = functions.layer_norm(x)
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    y = functions.layer_norm(x)
    assert bool(y[[1, 3]].isnan().any(1).all()) and torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


def test_no_rows_and_leading_shapes(device):
    w = torch.ones(24, device=device, requires_grad=True)
    x = torch.empty(0, 24, device=device, requires_grad=True)
    y = functions.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.empty(0, 24, device=device))
    assert y.shape == (0, 24) and gx.shape == (0, 24) and torch.equal(gw, torch.zeros_like(w))
    x = torch.randn(3, 5, 24, device=device)
    assert torch.equal(functions.layer_norm(x, w), functions.layer_norm(x.view(15, 24), w).view(3, 5, 24))
    assert torch.equal(functions.layer_norm(x[0, 0], w), functions.layer_norm(x.view(15, 24), w)[0])
    t = x.transpose(0, 1)      # rows in another order
    assert torch.equal(functions.layer_norm(t, w), functions.layer_norm(t.contiguous(), w))
    wide = torch.randn(24, 15, device=device).t()   # adjacent rows, elements apart
    assert torch.equal(functions.layer_norm(wide, w), functions.layer_norm(wide.contiguous(), w))


def test_expanded_rows_and_gradients(device):
    """A residual that is one row for all tokens, and a gradient that is one number for all elements."""
    x = torch.randn(50, 128, device=device, requires_grad=True)
    one = torch.randn(1, 128, device=device, requires_grad=True)
    y, s = functions.add_layer_norm(x, one.expand(50, 128))
    gx, g1 = torch.autograd.grad([y, s], [x, one], [torch.ones((), device=device).expand(50, 128), torch.randn(1, 128, device=device).expand(50, 128)])
    copy = one.detach().expand(50, 128).contiguous()
    y2, s2 = functions.add_layer_norm(x.detach(), copy)
    assert torch.equal(y.detach(), y2) and torch.equal(s.detach(), s2)
    assert torch.allclose(g1, gx.sum(0, keepdim=True), rtol=1e-4, atol=1e-5)


def test_gradients_through_one_result_only(device):
    x, r = (torch.randn(9, 64, device=device, requires_grad=True) for _ in range(2))
    w = torch.randn(64, device=device, requires_grad=True)
    y, s = functions.add_layer_norm(x, r, w)
    g = torch.randn(9, 64, device=device)
    gx, gr, gw = torch.autograd.grad(s, [x, r, w], g, retain_graph=True)
    assert torch.equal(gx, g) and torch.equal(gr, g) and torch.equal(gw, torch.zeros_like(w))
    gx, gw = torch.autograd.grad(y, [x, w], g)
    _check_backward([gx, gw, None], s.detach().double(), w, None, 1e-5, g.double(), torch.zeros_like(g).double())


def test_same_bits_every_time_and_by_row(device):
    """A row's results do not depend on the other rows, and the sums over the rows are made in one order."""
    x = torch.randn(3000, 768, device=device, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(768, device=device, dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(3000, 768, device=device, dtype=torch.bfloat16)
    run = lambda: (lambda y: (y,) + torch.autograd.grad(y, [x, w], dy))(functions.layer_norm(x, w))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
    assert torch.equal(functions.layer_norm(x[17:18], w), first[0][17:18])


def test_offsets_beyond_32_bits(device):
    """Rows of a tensor of more than 2^31 elements, far apart."""
    d, n = 64, 40
    stride = (1 << 31) // (n // 2)
    buf = torch.empty((n - 1) * stride + d, dtype=torch.bfloat16, device=device)
    x = buf.as_strided((n, d), (stride, 1))
    x.copy_(torch.randn(n, d, device=device))
    copy = x.contiguous()
    x.requires_grad_(True)
    y = functions.layer_norm(x)
    assert torch.equal(y.detach(), functions.layer_norm(copy))
    dy = torch.randn(n, d, device=device, dtype=torch.bfloat16)
    g, = torch.autograd.grad(y, x, dy)
    copy.requires_grad_(True)
    assert torch.equal(g, torch.autograd.grad(functions.layer_norm(copy), copy, dy)[0])


def test_another_stream_and_a_graph(device):
    """Captured, replayed with other rows between eager work, and every replay against the eager result."""
    n, d = 300, 640
    x, r, dy = (torch.randn(n, d, device=device, dtype=torch.bfloat16) for _ in range(3))
    w, b = (torch.randn(d, device=device, dtype=torch.float32) for _ in range(2))

    def step(x, r, dy, w, b):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w, b)]
        y, s = functions.add_layer_norm(*leaves)
        return (y.detach(), s.detach()) + torch.autograd.grad([y, s], leaves, [dy, dy])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(x, r, dy, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b_) for a, b_ in zip(warm, step(x, r, dy, w, b)))
    del warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x, r, dy, w, b)
    for k in range(4):
        for t in (x, r, dy):
            t.copy_(torch.randn(n, d, device=device))
        w.copy_(torch.randn(d, device=device))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(held, step(x, r, dy, w, b)):
            assert torch.equal(a, e), k


def test_checkpointed_and_module_parameters(device):
    """Inside an activation checkpoint, with an nn.LayerNorm's parameters, against the module in float64."""
    from torch.utils.checkpoint import checkpoint
    norm = torch.nn.LayerNorm(256).to(device)
    x = torch.randn(31, 256, device=device, requires_grad=True)
    dy = torch.randn(31, 256, device=device)
    y = checkpoint(lambda t: functions.layer_norm(t, norm.weight, norm.bias, norm.eps), x, use_reentrant=False)
    got = torch.autograd.grad(y, [x, norm.weight, norm.bias], dy)
    ref = torch.nn.LayerNorm(256).to(device).double()
    x64 = x.detach().double().requires_grad_(True)
    want = torch.autograd.grad(ref(x64), [x64, ref.weight, ref.bias], dy.double())
    for g, e in zip(got, want):
        assert torch.allclose(g.double(), e, rtol=1e-5, atol=1e-5)


def _twice(function, leaves, weights):
    """Gradients of a sum of squares of the gradients."""
    outs = function(*leaves)
    outs = outs if isinstance(outs, tuple) else (outs,)
    first = torch.autograd.grad(outs, leaves, weights[:len(outs)], create_graph=True)
    return torch.autograd.grad(sum(g.double().square().sum() for g in first), leaves, materialize_grads=True)


@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives(native, device, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_layer_call", None)
    torch.manual_seed(1)
    leaves = [torch.randn(*s, device=device) for s in ((5, 24), (5, 24), (24,), (24,))]
    dy, ds = torch.randn(5, 24, device=device), torch.randn(5, 24, device=device)
    got = _twice(functions.add_layer_norm, [t.clone().requires_grad_(True) for t in leaves], [dy, ds])

    def plain(x, r, w, b):
        s = x + r
        return (s - s.mean(1, keepdim=True)) * (s.var(1, correction=0, keepdim=True) + 1e-5).rsqrt() * w + b, s

    want = _twice(plain, [t.double().requires_grad_(True) for t in leaves], [dy.double(), ds.double()])
    for g, e in zip(got, want):
        assert torch.allclose(g.double(), e, rtol=1e-3, atol=1e-3 * float(e.abs().max()) + 1e-12)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_both_nodes_give_the_same_bits(dtype, device, monkeypatch):
    """The node in native code and the Python one."""
    t = TYPES[dtype]
    x, r, dy, ds = (torch.randn(70, 200, device=device).to(t) for _ in range(4))
    w, b = torch.randn(200, device=device), torch.randn(200, device=device)

    def run():
        leaves = [v.detach().requires_grad_(True) for v in (x, r, w, b)]
        y, s = functions.add_layer_norm(*leaves)
        z = functions.layer_norm(leaves[0], None, leaves[3] if dtype == "f32" else None)
        return (y.detach(), s.detach(), z.detach()) + torch.autograd.grad([y, s, z], leaves, [dy, ds, dy])

    native = run()
    assert type(functions.layer_norm(x.requires_grad_(True)).grad_fn).__name__ != "LayerNormBackward"
    monkeypatch.setattr(_lib, "_layer_call", None)
    assert type(functions.layer_norm(x).grad_fn).__name__ == "LayerNormBackward"
    assert all(torch.equal(a, e) for a, e in zip(native, run()))


def test_saved_tensors_may_come_back_otherwise(device):
    """Saved-tensor hooks hand back equal tensors that lie elsewhere, and in another order."""
    x = torch.randn(33, 48, device=device, requires_grad=True)
    w = torch.randn(48, device=device, requires_grad=True)
    dy = torch.randn(33, 48, device=device)
    want = torch.autograd.grad(functions.layer_norm(x, w), [x, w], dy)
    back = lambda t: t.t().contiguous().t() if t.dim() == 2 else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: back(t.to(device))):
        y = functions.layer_norm(x, w)
    got = torch.autograd.grad(y, [x, w], dy)
    assert all(torch.equal(a, e) for a, e in zip(want, got))


@pytest.mark.parametrize("shape,rows", [("shorter than a vector", (1 << 23) + 1001), ("one vector", (1 << 28) + 1001)])
def test_more_rows_than_one_launch_counts(device, shape, rows):
    """2^31 threads and more, 256 or 8 to a row: every row is normalised, those behind the first launch's as the same few alone."""
    d = 4 if shape == "shorter than a vector" else 8
    few = torch.randn(64, d, device=device).bfloat16()
    w = torch.randn(d, device=device)
    want = functions.layer_norm(few, w)
    if d == 4:
        x = few.repeat(-(-rows // 64), 1)[:rows].requires_grad_(True)
        y = functions.layer_norm(x, w)
        assert torch.equal(y.detach(), want.repeat(-(-rows // 64), 1)[:rows])
        g = torch.randn(64, d, device=device).bfloat16()
        alone = few.clone().requires_grad_(True)
        g_alone, = torch.autograd.grad(functions.layer_norm(alone, w), alone, g)
        g_x, = torch.autograd.grad(y, x, g.repeat(-(-rows // 64), 1)[:rows])
        assert torch.equal(g_x, g_alone.repeat(-(-rows // 64), 1)[:rows])
    else:
        y = functions.layer_norm(few[:1].expand(rows, d), w)     # (4.3 GB of results, every row the same)
        assert bool((y == want[:1]).all())


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("order", ["transposed", "sliced", "expanded"])
@pytest.mark.parametrize("residual", [False, True])
def test_second_derivatives_of_rows_in_any_order(residual, order, native, device, monkeypatch):
    """Rows that the kernels read a copy of, or where they lie: the gradient's gradient reaches them all the same."""
    if not native:
        monkeypatch.setattr(_lib, "_layer_call", None)
    torch.manual_seed(8)
    shape, view = {"transposed": ((24, 5), lambda t: t.t()), "sliced": ((5, 30), lambda t: t[:, 3:27]), "expanded": ((1, 24), lambda t: t.expand(5, 24))}[order]
    leaves = [torch.randn(s, device=device) for s in ([shape, shape] if residual else [shape]) + [(24,), (24,)]]
    dy, ds = torch.randn(5, 24, device=device), torch.randn(5, 24, device=device)

    def own(x, *rest):
        return functions.add_layer_norm(view(x), view(rest[0]), *rest[1:]) if residual else functions.layer_norm(view(x), *rest)

    def plain(x, *rest):
        s = view(x) + view(rest[0]) if residual else view(x)
        w, b = rest[-2:]
        y = (s - s.mean(1, keepdim=True)) * (s.var(1, correction=0, keepdim=True) + 1e-5).rsqrt() * w + b
        return (y, s) if residual else y

    got = _twice(own, [t.clone().requires_grad_(True) for t in leaves], [dy, ds])
    want = _twice(plain, [t.double().requires_grad_(True) for t in leaves], [dy.double(), ds.double()])
    for g, e in zip(got, want):
        assert torch.allclose(g.double(), e, rtol=1e-3, atol=1e-3 * float(e.abs().max()) + 1e-12)


@pytest.mark.parametrize("dtype,d", [("f32", 260), ("f32", 300), ("f32", 512), ("f32", 777), ("f32", 1024), ("f32", 2048), ("bf16", 1024), ("f16", 4096)])
def test_rows_do_not_depend_on_how_many_there_are(dtype, d, device):
    """One row, a few and thousands, alone or as a sum with a residual: the same bits, in float32 too, which shows the order of the sums, and in the
    gradients of the rows."""
    x, dy = (torch.randn(6000, d, device=device).to(TYPES[dtype]) for _ in range(2))
    w, b = torch.randn(d, device=device), torch.randn(d, device=device)

    def run(rows):
        leaf = x[rows].detach().requires_grad_(True)
        y = functions.layer_norm(leaf, w, b)
        return y.detach(), torch.autograd.grad(y, leaf, dy[rows])[0]

    every = run(slice(None))
    for rows in (slice(0, 1), slice(17, 60), slice(1, 2048), slice(4000, 6000)):
        assert all(torch.equal(a, e[rows]) for a, e in zip(run(rows), every)), rows
    y, s = functions.add_layer_norm(x, torch.zeros_like(x), w, b)
    assert torch.equal(s, x) and torch.equal(y, every[0])


def test_parameter_gradients_over_many_short_rows(device):
    """8 million rows shorter than a vector, whose gradients have one sign: a float32 sum of 65 thousand terms one after the other would be off by
    hundreds of steps.  A term passes through at most 8 float32 roundings (three in the normalised element, its product, a part's sum and those that join
    the parts' 128: at most 24 more), each of 2^-24 of it."""
    rows, d = (1 << 23) + 3, 3
    x = torch.randn(rows, d, device=device, generator=torch.Generator(device=device).manual_seed(3))
    w, b = torch.ones(d, device=device, requires_grad=True), torch.zeros(d, device=device, requires_grad=True)
    dy = torch.full((rows, d), 0.1, device=device)
    # (the sign of every normalised element, so that grad_w's terms have one sign too)
    mean, rstd, h = _reference(x.double(), None, None, 1e-5)[:3]
    for g, name in ((dy, "grad_b"), (torch.where(h < 0, -dy, dy), "grad_w")):
        gw, gb = torch.autograd.grad(functions.layer_norm(x, w, b), [w, b], g)
        if name == "grad_b":
            want = g.double().sum(0)
            assert bool(((gb.double() - want).abs() <= 32 * ULP32 * want).all()), ((gb.double() - want) / want).tolist()
        else:
            # (an element's own error: what the mean's rounding is to it, with the magnitudes that it was taken off)
            want, reach = (g.double() * h).sum(0), (g.double().abs() * (x.double().abs() + mean.abs()) * rstd).sum(0)
            assert bool(((gw.double() - want).abs() <= 32 * ULP32 * (want + reach)).all()), ((gw.double() - want) / want).tolist()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,d,dtype", [(9001, 768, "bf16"), (9001, 768, "f32"), (1001, 4096, "f16"), (1001, 4096, "f32"), (70001, 40, "bf16"), (4099, 2052, "f32")])
def test_several_sets_of_rows_to_a_workgroup(n, d, dtype, residual, device):
    """Backward passes whose workgroups walk over several sets of rows, the last one not full."""
    _run(n, d, dtype, residual, "same")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,d", [(5, 8200), (300, 8200), (7, 12000), (515, 12000), (3, 16384), (300, 16384), (3, 16381), (9, 20000), (2, 32768)])
def test_long_rows(n, d, residual, dtype, device):
    """Rows that take the most registers, alone and several to a workgroup."""
    _run(n, d, dtype, residual, "same")


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,d,dtype", [(11003, 4096, "bf16"), (6001, 4096, "f32"), (3001, 8192, "f32"), (1501, 16384, "f32"), (4001, 12000, "bf16"), (60001, 768, "f16"),
                                       (30001, 1500, "bf16")])
def test_rows_past_the_caches(n, d, dtype, residual, device):
    """More than 256 MiB to read and write in the backward, which goes past the caches then."""
    _run(n, d, dtype, residual, "f32" if dtype == "f16" else "same")
