"""Gated experts (functions.gated_mlp, FMoEGatedMLP) against their formulas in float64.

Tolerances.  A rounding to a type is off by at most u = eps / 2 of the value; such errors are independent of each other, of mean about 0 and at most u,
so of standard deviation u / sqrt(3) at most.  A sum of products whose terms t_k are each off by a_k at most is then off by at most
4 sqrt(sum a_k^2) (seven standard deviations), and its own float32 roundings by at most 16 2^-24 sqrt(n) sqrt(sum t_k^2) for n terms
(n roundings of partial sums, each of a few times sqrt(sum t_k^2)).  ``_reference`` carries those amplitudes along the formulas:
act(g) u is rounded once; the backward takes g and u as their type holds them, and rounds dm, then dm u act'(g) and dm act(g), once each.
The activations are off by at most 2^-21 |g|, their slopes by 2^-21 (1 + |g|)."""
import math

import pytest
import torch

from fastermoe_amd import FMoEGatedMLP, FMoEPositionwiseFF, fmoe_native, functions
from fastermoe_amd.gates.utils import limit_by_capacity  # noqa: F401  (the layer's gates import)

pytestmark = pytest.mark.gpu

ACTS = {"silu": (torch.nn.SiLU(), torch.nn.functional.silu), "gelu": (torch.nn.GELU(), torch.nn.functional.gelu),
        "relu": (torch.nn.ReLU(), torch.relu), "none": (None, lambda t: t)}
F32 = 2.0 ** -24


def _counts(kind, rows, experts, seed=0):
    gen = torch.Generator().manual_seed(seed)
    if kind == "one":          # all rows are the last expert's
        return [0] * (experts - 1) + [rows]
    if kind == "tail":         # rows behind the last expert's
        rows = rows * 3 // 4
    share = torch.rand(experts, generator=gen) ** (3 if kind == "skewed" else 1)
    if kind == "skewed" and experts > 2:
        share[1] = 0
    counts = (share / share.sum() * rows).long()
    counts[0] += rows - int(counts.sum())
    return counts.tolist()


def _dot(a, b, amp_a=None):
    """``a @ b`` and the amplitude of its error, ``amp_a`` that of ``a``'s elements."""
    n = a.shape[1]
    q = ((a * a) @ (b * b)).sqrt()
    err = 16 * F32 * math.sqrt(max(n, 1)) * q
    if amp_a is not None:
        err = err + 4 * ((amp_a * amp_a) @ (b * b)).sqrt()
    return a @ b, err


def _reference(x, counts, w1, b1, w2, b2, act, gy=None):
    """{name: (value, tolerance)} in float64."""
    u = torch.finfo(x.dtype).eps / 2
    fn = ACTS[act][1]
    x64, w1, w2 = x.double(), w1.double(), w2.double()
    h = w2.shape[2]
    zeros = lambda t: [torch.zeros_like(t, dtype=torch.float64), torch.zeros_like(t, dtype=torch.float64)]
    out = {"y": zeros(x)}
    if gy is not None:
        out.update(x=zeros(x), w1=zeros(w1), w2=zeros(w2), b1=zeros(w1[:, :, 0]), b2=zeros(w2[:, :, 0]))

    def slope(g):
        g = g.detach().requires_grad_(True)
        return torch.autograd.grad(fn(g).sum(), g)[0] if act != "none" else torch.ones_like(g)

    def put(name, at, value, amp):
        out[name][0][at] = value
        out[name][1][at] = amp + u * value.abs() * 1.01 + 1e-30 + (2.0 ** -24 if x.dtype == torch.float16 else 0)   # (float16 below 2^-14)
    lo = 0
    for e, c in enumerate(counts):
        if c == 0:
            continue
        at = slice(lo, lo + c)
        lo += c
        xe = x64[at]
        pre, pre_amp = _dot(xe, w1[e].t())
        if b1 is not None:
            pre = pre + b1[e].double()
            pre_amp = pre_amp + 2 * F32 * pre.abs()
        g, v, ga, va = pre[:, :h], pre[:, h:], pre_amp[:, :h], pre_amp[:, h:]
        a, s = fn(g), slope(g)
        a_amp = 1.2 * ga + 2.0 ** -21 * g.abs()
        mid = a * v
        mid_amp = a_amp * v.abs() + a.abs() * va + (u + 4 * F32) * mid.abs() + (2.0 ** -24 if x.dtype == torch.float16 else 0)
        y, amp = _dot(mid, w2[e].t(), mid_amp)
        if b2 is not None:
            y = y + b2[e].double()
        put("y", at, y, amp + 2 * F32 * y.abs())
        if gy is None:
            continue
        dy = gy[at].double()
        dm, dm_amp = _dot(dy, w2[e])
        dm_amp = dm_amp + u * dm.abs()
        step = u * g.abs() + ga     # how far the kept gate is from g
        s_amp = torch.maximum((slope(g + step) - s).abs(), (slope(g - step) - s).abs()) + 2.0 ** -21 * (1 + g.abs())
        a_held = torch.maximum((fn(g + step) - a).abs(), (fn(g - step) - a).abs()) + 2.0 ** -21 * g.abs()
        dg, du = dm * v * s, dm * a
        small = 2.0 ** -24 if x.dtype == torch.float16 else 0
        dg_amp = dm_amp * (v * s).abs() + (dm * s).abs() * (u * v.abs() + va) + (dm * v).abs() * s_amp + (u + 4 * F32) * dg.abs() + small * (1 + (v * s).abs())
        du_amp = dm_amp * a.abs() + dm.abs() * a_held + (u + 4 * F32) * du.abs() + small * (1 + a.abs())
        dpre, dpre_amp = torch.cat([dg, du], 1), torch.cat([dg_amp, du_amp], 1)
        put("x", at, *_dot(dpre, w1[e], dpre_amp))
        put("w1", e, *(t.t() for t in _dot_t(xe, dpre, dpre_amp)))
        put("w2", e, *_dot_t(dy, mid, mid_amp))
        ones = torch.ones(c, 1, dtype=torch.float64, device=x.device)
        put("b1", e, *(t[0] for t in _dot_t(ones, dpre, dpre_amp)))
        put("b2", e, *(t[0] for t in _dot_t(ones, dy, torch.zeros_like(dy))))
    return out


def _dot_t(a, b, amp_b):
    """``a^T @ b`` and the amplitude of its error, ``amp_b`` that of ``b``'s elements."""
    value, err = _dot(b.t(), a, amp_b.t())
    return value.t(), err.t()


def _close(name, got, want):
    value, tol = want
    err = (got.double() - value).abs()
    worst = (err / tol.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert (err <= tol).all(), f"{name}: {worst:.2f} tolerances off, {int((err > tol).sum())} of {err.numel()}, at {(err / tol.clamp(min=1e-300)).argmax().item()}"


def _tensors(rows, d, h, experts, dtype, bias, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda scale, *shape: (scale * torch.randn(shape, device="cuda", generator=gen)).to(dtype)
    return (new(1.0, rows, d), new(1 / math.sqrt(d), experts, 2 * h, d), new(0.2, experts, 2 * h) if bias else None,
            new(1 / math.sqrt(h), experts, d, h), new(0.2, experts, d) if bias else None, new(1.0, rows, d))


def _check(rows, d, h, experts, dtype, act, bias, kind, seed=0, where="device"):
    x, w1, b1, w2, b2, gy = _tensors(rows, d, h, experts, dtype, bias, seed)
    counts = _counts(kind, rows, experts, seed)
    want = _reference(x, counts, w1, b1, w2, b2, act, gy)
    cnt = torch.tensor(counts)
    if where == "device":
        cnt = cnt.cuda()
    with torch.no_grad():
        y = functions.gated_mlp(x, cnt, w1, b1, w2, b2, ACTS[act][0])
    _close("y without gradients", y, want["y"])
    leaves = {n: t.requires_grad_(True) for n, t in (("x", x), ("w1", w1), ("b1", b1), ("w2", w2), ("b2", b2)) if t is not None}
    y = functions.gated_mlp(x, cnt, w1, b1, w2, b2, ACTS[act][0])
    _close("y", y.detach(), want["y"])
    for name, grad in zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)):
        _close("grad " + name, grad, want[name])


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", list(ACTS))
def test_small(dtype, act):
    _check(37, 64, 96, 3, dtype, act, True, "even")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,d,h,experts,kind", [
    (1, 8, 8, 1, "even"), (1, 1024, 512, 4, "one"), (2, 512, 1024, 32, "skewed"), (5, 1, 1, 2, "even"), (7, 3, 5, 2, "tail"), (130, 36, 44, 3, "skewed"),
    (129, 65, 33, 2, "even"), (300, 130, 250, 12, "tail"), (64, 256, 128, 64, "even"), (257, 72, 8, 2, "one"), (1000, 320, 192, 5, "skewed")])
def test_sizes(dtype, rows, d, h, experts, kind):
    _check(rows, d, h, experts, dtype, "silu", rows % 2 == 0, kind, seed=rows)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "none"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_large_enough_to_fill_the_card(dtype, act):
    """512 tiles of 256 x 256 and more in every product, contractions that end inside a slab, columns that end inside a tile, tail rows."""
    _check(8200, 1032, 2072, 4, dtype, act, act in ("silu", "relu"), "tail" if act == "gelu" else "skewed")


@pytest.mark.parametrize("dtype,tile", [(t, s) for t in (torch.bfloat16, torch.float16) for s in ("256x256", "128x256", "128x128", "128x128+", "64x128")]
                         + [(torch.float32, s) for s in ("128x128", "128x128+", "64x64")], ids=str)
@pytest.mark.parametrize("rows,d,h,kind", [(700, 200, 328, "skewed"), (300, 5120, 136, "tail"), (150, 72, 5128, "even")])
def test_every_tile(monkeypatch, dtype, tile, rows, d, h, kind):
    """Columns and contractions that end inside a tile and a slab; long contractions, whose last round of tiles is shared (forward; data gradient)."""
    monkeypatch.setenv("FMOE_GEMM_TILE", tile)
    for act in (ACTS if rows == 700 else ("silu",)):
        _check(rows, d, h, 3, dtype, act, rows != 300, kind, seed=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,d,h,experts", [(1, 70, 63, 2), (70, 65, 64, 1), (140, 64, 65, 2), (300, 33, 130, 3), (6000, 131, 1301, 2)])
def test_every_column_off_the_grid(dtype, rows, d, h, experts):
    """Rows that begin anywhere, tiles of both heights, every activation."""
    for act in ACTS:
        _check(rows, d, h, experts, dtype, act, act != "none", "tail" if act == "relu" else "skewed", seed=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,d,h,experts,kind", [(1, 1, 3, 1, "even"), (1, 7, 9, 2, "one"), (2, 63, 65, 3, "even"), (5, 130, 333, 4, "skewed"), (16, 257, 66, 1, "even"),
                                                   (17, 515, 129, 2, "one"), (40, 1030, 70, 3, "tail"), (47, 449, 1001, 3, "skewed"), (9, 2049, 34, 600, "even"),
                                                   (150, 1302, 500, 12, "skewed"), (3, 8, 1, 1, "even"), (192, 2500, 11, 12, "skewed")])
def test_few_rows_off_the_grid(dtype, rows, d, h, experts, kind):
    for act in ("silu", "none"):
        _check(rows, d, h, experts, dtype, act, act == "silu", kind, seed=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,d,h,experts,kind", [(300, 701, 2503, 3, "skewed"), (1100, 650, 1302, 5, "tail"), (40, 130, 2049, 2, "even"), (1, 33, 5007, 1, "even"),
                                                   (700, 1283, 4, 40, "skewed"), (193, 1299, 643, 6, "one"), (260, 1281, 1283, 2, "tail")])
def test_contractions_in_parts(dtype, rows, d, h, experts, kind):
    """Off the grid, few tiles: contractions of ten slabs of 64 and more in two to eight parts, the last ones shorter."""
    for act in ("silu", "relu"):
        _check(rows, d, h, experts, dtype, act, act == "silu", kind, seed=rows)


@pytest.mark.parametrize("rows,d,h", [(9, 50, 64), (9, 64, 50), (300, 67, 96), (300, 96, 67), (300, 1, 8), (300, 8, 1)])
def test_float32_with_one_size_off_the_grid(rows, d, h):
    for act in ("silu", "gelu"):
        _check(rows, d, h, 3, torch.float32, act, act == "gelu", "tail" if act == "gelu" else "skewed", seed=rows)


@pytest.mark.parametrize("off", range(1, 8))
def test_few_rows_from_anywhere(off):
    """Tensors of sizes on the grid that begin off it."""
    gen = torch.Generator(device="cuda").manual_seed(off)
    make = lambda *shape, at: torch.randn(math.prod(shape) + 8, device="cuda", generator=gen).to(torch.bfloat16)[at:at + math.prod(shape)].view(shape)
    x, w1, w2 = make(6, 192, at=off), make(3, 256, 192, at=off // 2), make(3, 192, 128, at=0)
    counts = [1, 3, 2]
    y = functions.gated_mlp(x, torch.tensor(counts, device="cuda"), w1, None, w2, None, torch.nn.SiLU())
    value, tol = _reference(x, counts, w1, None, w2, None, "silu")["y"]
    assert ((y.double() - value).abs() <= tol).all()


@pytest.mark.parametrize("rows", [13, 16, 47, 48, 49])
def test_few_rows(rows):
    _check(rows, 512, 1024, 3, torch.bfloat16, "silu", True, "skewed", seed=rows)
    _check(rows, 512, 1024, 3, torch.float16, "gelu", False, "tail", seed=rows)


def test_large_float32():
    _check(4100, 512, 1024, 8, torch.float32, "silu", True, "skewed")


@pytest.mark.parametrize("dtype,d,h", [(torch.bfloat16, 64, 96), (torch.bfloat16, 50, 31), (torch.float32, 50, 31), (torch.float32, 64, 96)], ids=str)
def test_counts_on_the_host(dtype, d, h):
    _check(77, d, h, 4, dtype, "silu", True, "tail", where="host")


def test_decode_rows_of_large_experts():
    for rows in (1, 2, 16, 33, 128):
        _check(rows, 1024, 2816, 8, torch.bfloat16, "silu", rows == 16, "skewed", seed=rows)


def test_no_rows():
    x, w1, b1, w2, b2, _ = _tensors(0, 16, 24, 3, torch.bfloat16, True)
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = functions.gated_mlp(x, torch.zeros(3, dtype=torch.int64, device="cuda"), w1, b1, w2, b2, ACTS["silu"][0])
    assert y.shape == (0, 16)
    for t, g in zip(leaves, torch.autograd.grad(y, leaves, torch.empty_like(y))):
        assert g.shape == t.shape and not g.any()


def test_rows_behind_the_counted_ones_are_zeros_and_never_read():
    x, w1, b1, w2, b2, gy = _tensors(40, 32, 48, 3, torch.bfloat16, True)
    x[25:], gy[25:] = float("nan"), float("inf")
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = functions.gated_mlp(x, torch.tensor([20, 0, 5], device="cuda"), w1, b1, w2, b2, ACTS["silu"][0])
    grads = torch.autograd.grad(y, leaves, gy)
    assert not y[25:].any() and not grads[0][25:].any()
    assert all(torch.isfinite(t).all() for t in (y, *grads))
    assert not any(g[1].any() for g in grads[1:])   # (the expert without rows)


def test_infinities_and_nan_show():
    x, w1, _, w2, _, gy = _tensors(9, 32, 48, 1, torch.bfloat16, False)
    x[3, 5], x[7, 0] = float("inf"), float("nan")
    x.requires_grad_(True)
    y = functions.gated_mlp(x, torch.tensor([9], device="cuda"), w1, None, w2, None, ACTS["silu"][0])
    bad = ~torch.isfinite(y).all(dim=1)
    assert bad.tolist() == [i in (3, 7) for i in range(9)]


@pytest.mark.parametrize("dtype,act", [(torch.float32, "silu"), (torch.float32, "gelu")])
def test_gradients_against_differences(dtype, act):
    """(f(t + ev) - f(t - ev)) / 2e against <grad, v>, f a weighted sum of the outputs in float64.  e = 2^-6: the third derivatives take 2^-12 of the slope's
    size times a constant of a few, the outputs' roundings (2^-22 of sums of 10^3 terms of size 1) 2^-22 sqrt(10^3) / 2^-6."""
    x, w1, b1, w2, b2, gy = _tensors(24, 20, 28, 2, dtype, True)
    cnt = torch.tensor([10, 14], device="cuda")
    leaves = [x, w1, b1, w2, b2]
    y = functions.gated_mlp(*(t if i else t for i, t in enumerate([x.requires_grad_(True)])), cnt, *(t.requires_grad_(True) for t in leaves[1:]), ACTS[act][0])
    grads = torch.autograd.grad(y, leaves, gy)
    gen = torch.Generator(device="cuda").manual_seed(9)
    eps = 2.0 ** -6

    def f(ts):
        with torch.no_grad():
            return (functions.gated_mlp(ts[0], cnt, *ts[1:], ACTS[act][0]).double() * gy.double()).sum().item()
    for i, (t, g) in enumerate(zip(leaves, grads)):
        v = torch.randn(t.shape, device="cuda", generator=gen)
        v = v / v.norm()
        moved = lambda s: [u.detach() + s * eps * v if j == i else u.detach() for j, u in enumerate(leaves)]
        got, want = (f(moved(1)) - f(moved(-1))) / (2 * eps), (g.double() * v.double()).sum().item()
        assert abs(got - want) <= 2.0 ** -9 * g.norm().item() + 2.0 ** -10, (i, got, want)


def test_strided_rows_and_gradients():
    x, w1, b1, w2, b2, gy = _tensors(30, 48, 40, 2, torch.bfloat16, True)
    cnt = torch.tensor([11, 19], device="cuda")
    wide = torch.zeros(30, 96, dtype=x.dtype, device="cuda")
    wide[:, 40:88] = x
    a = wide[:, 40:88].requires_grad_(True)
    b = x.clone().requires_grad_(True)
    ya, yb = (functions.gated_mlp(t, cnt, w1, b1, w2, b2, ACTS["gelu"][0]) for t in (a, b))
    assert torch.equal(ya, yb)
    ga, = torch.autograd.grad(ya, a, gy.t().contiguous().t())
    gb, = torch.autograd.grad(yb, b, gy)
    assert torch.equal(ga, gb)


def test_single_gradients():
    x, w1, b1, w2, b2, gy = _tensors(30, 48, 40, 2, torch.bfloat16, True)
    cnt = torch.tensor([11, 19], device="cuda")
    all_of = [x, w1, b1, w2, b2]
    for t in all_of:
        t.requires_grad_(True)
    want = torch.autograd.grad(functions.gated_mlp(x, cnt, w1, b1, w2, b2, ACTS["silu"][0]), all_of, gy)
    for i in range(5):
        ts = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate(all_of)]
        y = functions.gated_mlp(ts[0], cnt, *ts[1:], ACTS["silu"][0])
        y.backward(gy)
        for j, t in enumerate(ts):
            assert (t.grad is None) == (j != i)
        assert torch.equal(ts[i].grad, want[i])


def test_same_bits_again_and_on_another_stream():
    x, w1, b1, w2, b2, gy = _tensors(700, 256, 512, 8, torch.bfloat16, True)
    cnt = torch.tensor(_counts("skewed", 700, 8), device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]

    def run():
        y = functions.gated_mlp(x, cnt, w1, b1, w2, b2, ACTS["silu"][0])
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    third = run()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_forward_replays():
    x, w1, b1, w2, b2, _ = _tensors(64, 256, 512, 8, torch.bfloat16, True)
    cnt = torch.tensor(_counts("even", 64, 8), device="cuda")

    def run():
        with torch.no_grad():
            return functions.gated_mlp(x, cnt, w1, b1, w2, b2, ACTS["silu"][0])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        cnt.copy_(cnt.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run())


def test_second_derivatives_are_refused():
    x, w1, _, w2, _, gy = _tensors(6, 16, 8, 1, torch.float32, False)
    x.requires_grad_(True)
    y = functions.gated_mlp(x, torch.tensor([6], device="cuda"), w1, None, w2, None, ACTS["silu"][0])
    g, = torch.autograd.grad(y, x, gy.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def _layer_reference(layer, x, act):
    """The layer's output and gradients from float64 products, with the gate's own choice."""
    with torch.no_grad():
        idx, score = layer.gate(x)
    ex = layer.experts
    params = [p.detach().double().requires_grad_(True) for p in (ex.htoh4.weight, ex.htoh4.bias, ex.h4toh.weight, ex.h4toh.bias)]
    w1, b1, w2, b2 = params
    x64 = x.detach().double().requires_grad_(True)
    out = torch.zeros_like(x64)
    h = w2.shape[2]
    for e in range(w1.shape[0]):
        for k in range(idx.shape[1]):
            at = (idx[:, k] == e).nonzero().reshape(-1)
            if at.numel():
                pre = x64[at] @ w1[e].t() + b1[e]
                y = (ACTS[act][1](pre[:, :h]) * pre[:, h:]) @ w2[e].t() + b2[e]
                out = out.index_add(0, at, y * score[at, k].double()[:, None])
    return out, x64, params


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d,h", [(64, 96), (50, 33)])
@pytest.mark.parametrize("fuse", [False, True])
def test_layer(dtype, d, h, fuse):
    """The norms of the errors: each of the four roundings on the way (a quarter of that more for the sums) is at most u of its value."""
    torch.manual_seed(3)
    layer = FMoEGatedMLP(num_expert=6, d_model=d, d_hidden=h, top_k=2).to(dtype).cuda()
    with torch.no_grad():
        for p in layer.experts.parameters():
            p.copy_(torch.randn(p.shape) * (0.1 if p.dim() == 2 else p.shape[2] ** -0.5))
    layer.enable_fuse = fuse
    x = torch.randn(4, 40, d, device="cuda").to(dtype).requires_grad_(True)
    flat = x.detach().reshape(-1, d)
    ref, x64, params = _layer_reference(layer, flat, "silu")
    # (the gate's own gradient left out: its scores are constants to the reference)
    with torch.no_grad():
        chosen = layer.gate(flat)
    layer.gate.forward = lambda inp: chosen
    y = layer(x)
    assert y.shape == x.shape
    gy = torch.randn_like(y)
    y.backward(gy)
    want = torch.autograd.grad(ref, [x64, *params], gy.reshape(-1, d).double())
    u = torch.finfo(dtype).eps / 2
    rel = lambda a, b: ((a.double().reshape(b.shape) - b).norm() / b.norm()).item()
    assert rel(y.detach(), ref.detach()) <= (4 * u if dtype != torch.float32 else 64 * u)
    ex = layer.experts
    for name, got, w in zip(("x", "w1", "b1", "w2", "b2"), (x.grad, ex.htoh4.weight.grad, ex.htoh4.bias.grad, ex.h4toh.weight.grad, ex.h4toh.bias.grad),
                            want):
        assert rel(got, w) <= (8 * u if dtype != torch.float32 else 64 * u), name


def test_layer_with_another_activation_runs_module_by_module():
    torch.manual_seed(3)
    layer = FMoEGatedMLP(num_expert=3, d_model=16, d_hidden=24, top_k=1, activation=torch.nn.Tanh()).cuda()
    x = torch.randn(20, 16, device="cuda", requires_grad=True)
    ex = layer.experts
    with torch.no_grad():
        idx, score = layer.gate(x)
    y = layer(x)
    y.sum().backward()
    assert ex.htoh4.weight.grad is not None and torch.isfinite(x.grad).all()
    for t in range(20):
        e = int(idx[t, 0])
        pre = ex.htoh4.weight[e] @ x[t] + ex.htoh4.bias[e]
        want = (ex.h4toh.weight[e] @ (torch.tanh(pre[:24]) * pre[24:]) + ex.h4toh.bias[e]) * score[t, 0]
        assert torch.allclose(y[t], want, rtol=1e-4, atol=1e-5)


def test_block_with_gated_experts():
    torch.manual_seed(1)
    block = FMoEPositionwiseFF(num_expert=4, d_model=32, d_hidden=48, top_k=2, pre_lnorm=True, gated=True).cuda()
    x = torch.randn(3, 7, 32, device="cuda", requires_grad=True)
    y = block(x)
    y.square().mean().backward()
    assert y.shape == x.shape and all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())


def test_activations_in_8_bits_are_refused():
    layer = FMoEGatedMLP(num_expert=2, d_model=16, d_hidden=16).cuda()
    layer.act_checkpoint = True
    with pytest.raises(NotImplementedError):
        layer(torch.randn(4, 16, device="cuda", requires_grad=True))


def test_wrong_tensors_are_refused():
    x, w1, b1, w2, b2, _ = _tensors(8, 16, 24, 2, torch.bfloat16, True)
    cnt = torch.tensor([3, 5], device="cuda")
    call = lambda **kw: functions.gated_mlp(*(kw.get(k, v) for k, v in (("x", x), ("cnt", cnt), ("w1", w1), ("b1", b1), ("w2", w2), ("b2", b2),
                                                                          ("act", torch.nn.SiLU()))), table=kw.get("table"))
    call()
    for error, kw in [(ValueError, {"w1": w1[:, :-1].contiguous()}), (ValueError, {"w2": w2[:1]}), (ValueError, {"b1": b1[:, :-1].contiguous()}),
                      (TypeError, {"w1": w1.float()}), (TypeError, {"x": x.double(), "w1": w1.double(), "w2": w2.double(), "b1": None, "b2": None}),
                      (ValueError, {"cnt": cnt[:1]}), (TypeError, {"cnt": cnt.int()}), (ValueError, {"cnt": torch.tensor([8, 1])}),
                      (ValueError, {"cnt": torch.tensor([-1, 3])}), (TypeError, {"cnt": None}), (ValueError, {"w1": w1.cpu()}),
                      (NotImplementedError, {"act": torch.nn.Tanh()}), (ValueError, {"act": 3}), (ValueError, {"x": x[0]}),
                      (ValueError, {"table": fmoe_native.segment_table(cnt, 300)}), (ValueError, {"w2": w2.transpose(1, 2).contiguous().transpose(1, 2)})]:
        with pytest.raises(error):
            call(**kw)
