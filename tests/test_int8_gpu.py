"""Experts in 8-bit integers (functions.quantize_rows, functions.linear_int8, FMoETransformerMLP.quantize_experts) against their formulas in float64.

The integers and scales have to be the same.  A product's sum is exact; float32 rounds the sum, the product of the scales, the sum with the bias, the
activation (off by 2^-21 of its argument at most) and the gate's product, the result's type rounds once more, by u = eps / 2 at most."""
import math

import pytest
import torch

from fastermoe_amd import FMoEGatedMLP, FMoETransformerMLP, fmoe_native, functions

pytestmark = pytest.mark.gpu

ACTS = {"silu": (torch.nn.SiLU(), torch.nn.functional.silu), "gelu": (torch.nn.GELU(), torch.nn.functional.gelu),
        "relu": (torch.nn.ReLU(), torch.relu), "none": (None, lambda t: t)}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
LEAST = 2.0 ** -126


def _quantized(x):
    """(q, scale) by the definition."""
    x64 = x.double()
    # (in float64, whose quotient is the float32 one once rounded; a float32 tensor over a Python number is multiplied by the number's reciprocal)
    scale = (x64.abs().amax(dim=-1) / 127.0).float().clamp(min=LEAST) if x.shape[-1] else torch.full(x.shape[:-1], LEAST, device=x.device)
    bad = ~torch.isfinite(x64).all(dim=-1)
    q = torch.round(x64 / scale.double()[..., None])
    q[bad] = 0
    scale = scale.clone()
    scale[bad] = float("nan")
    return q, scale


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 16), (2, 500), (9, 512), (4, 513), (7, 1024), (3, 1030), (2, 2048), (5, 2500), (3, 4096), (2, 8192),
                                    (3, 16384), (2, 16390), (1, 40001), (4099, 64), (1000, 777), (2050, 1000), (4100, 1500), (4100, 2000), (2100, 4000)])
def test_rows(dtype, rows, d):
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + d)
    x = (torch.randn(rows, d, device="cuda", generator=gen) * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=gen))).to(dtype)
    q, scale = functions.quantize_rows(x)
    want_q, want_scale = _quantized(x)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and q.shape == x.shape
    assert torch.equal(scale, want_scale)
    assert torch.equal(q.double(), want_q)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


def test_ties_and_borders():
    """Quotients of exactly a half, and next to one: scale 2^-3 (a largest magnitude of 127 / 8), every multiple of half a step and its neighbours."""
    half = torch.arange(-254, 255, device="cuda").float() / 16
    near = torch.cat([half, torch.nextafter(half, half + 1), torch.nextafter(half, half - 1)]).clamp(-127 / 8, 127 / 8)
    q, scale = functions.quantize_rows(near[None])
    assert scale.item() == 0.125
    assert torch.equal(q[0].double(), torch.round(near.double() * 8))
    # the same for a scale that is no power of two
    s = torch.tensor(0.3, device="cuda")
    steps = (torch.arange(-127, 127, device="cuda").double() + 0.5) * s.double()
    x = torch.cat([steps.float(), torch.nextafter(steps.float(), steps.float() + 1), torch.nextafter(steps.float(), steps.float() - 1), (127 * s.double()).float()[None]])
    q, scale = functions.quantize_rows(x[None])
    want_q, want_scale = _quantized(x[None])
    assert torch.equal(scale, want_scale) and torch.equal(q.double(), want_q)


def test_extreme_rows():
    x = torch.zeros(8, 40, device="cuda")
    x[1, 3] = 1e-45                      # the least number there is
    x[2, 5], x[2, 6] = 3.4e38, -3.4e38
    x[3, 0] = float("inf")
    x[4, 1] = float("nan")
    x[5] = 1.0
    x[6, :2] = torch.tensor([1e-38, -3e-39])
    x[7, 0] = -float("inf")
    q, scale = functions.quantize_rows(x)
    want_q, want_scale = _quantized(x)
    assert torch.equal(torch.isnan(scale), torch.isnan(want_scale)) and torch.isnan(scale).tolist() == [False] * 3 + [True, True, False, False, True]
    ok = ~torch.isnan(scale)
    assert torch.equal(scale[ok], want_scale[ok]) and torch.equal(q.double(), want_q)
    assert (q[5] == 127).all()


def test_rows_of_any_leading_shape_and_stride():
    x = torch.randn(3, 4, 50, device="cuda").bfloat16()
    q, scale = functions.quantize_rows(x)
    q2, scale2 = functions.quantize_rows(x.reshape(12, 50))
    assert q.shape == x.shape and scale.shape == (3, 4)
    assert torch.equal(q.reshape(12, 50), q2) and torch.equal(scale.reshape(-1), scale2)
    wide = torch.randn(20, 100, device="cuda").bfloat16()
    q, scale = functions.quantize_rows(wide[:, 13:60])
    q2, scale2 = functions.quantize_rows(wide[:, 13:60].contiguous())
    assert torch.equal(q, q2) and torch.equal(scale, scale2)
    q, scale = functions.quantize_rows(wide.t())
    q2, scale2 = functions.quantize_rows(wide.t().contiguous())
    assert torch.equal(q, q2) and torch.equal(scale, scale2)
    q, scale = functions.quantize_rows(x[0, 0])
    assert q.shape == (50,) and scale.shape == () and torch.equal(q, functions.quantize_rows(x[0])[0][0])
    q, scale = functions.quantize_rows(torch.empty(0, 5, device="cuda"))
    assert q.shape == (0, 5) and scale.shape == (0,)


def _counts(kind, rows, experts, seed=0):
    if kind == "one":
        return [0] * (experts - 1) + [rows]
    if kind == "tail":
        rows = rows * 3 // 4
    gen = torch.Generator().manual_seed(seed)
    share = torch.rand(experts, generator=gen) ** (3 if kind == "skewed" else 1)
    if kind == "skewed" and experts > 2:
        share[1] = 0
    counts = (share / share.sum() * rows).long()
    counts[0] += rows - int(counts.sum())
    return counts.tolist()


def _tensors(rows, d, out, experts, dtype, bias, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, d, device="cuda", generator=gen) * torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=gen))).to(dtype)
    q, scale = functions.quantize_rows(torch.randn(experts, out, d, device="cuda", generator=gen) / math.sqrt(d))
    return x, q, scale, (0.3 * torch.randn(experts, out, device="cuda", generator=gen)).to(dtype) if bias else None


def _reference(x, counts, weight, scale, bias, act, gated, at=None):
    """(value, tolerance) in float64."""
    u, f = torch.finfo(x.dtype).eps / 2, 2.0 ** -24
    q, s = _quantized(x if at is None else x[at])
    s = s.double()[:, None]
    out = weight.shape[1] // (2 if gated else 1)
    value = torch.zeros(q.shape[0], out, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(value)
    lo = 0
    for e, c in enumerate(counts):
        part = slice(lo, lo + c)
        lo += c
        if not c:
            continue
        pre = (q[part] @ weight[e].double().t()) * s[part] * scale[e].double()
        amp = 3 * f * pre.abs()
        if bias is not None:
            pre = pre + bias[e].double()
        amp = amp + f * pre.abs()
        g, ga = pre[:, :out], amp[:, :out]
        a = ACTS[act][1](g)
        y, ya = a, 1.2 * ga + (2.0 ** -21 * g.abs() if act != "none" else 0)
        if gated:
            y = a * pre[:, out:]
            ya = ya * pre[:, out:].abs() + a.abs() * amp[:, out:] + f * y.abs()
        value[part] = y
        tol[part] = ya * 1.01 + u * y.abs() * 1.01 + 1e-37 + (2.0 ** -25 if x.dtype == torch.float16 else 0)   # (float16 below 2^-14)
    return value, tol


def _close(got, want):
    value, tol = want
    err = (got.double() - value).abs()
    assert (err <= tol).all(), f"{(err / tol.clamp(min=1e-300)).max().item():.2f} tolerances off, {int((err > tol).sum())} of {err.numel()}"


def _check(rows, d, out, experts, dtype, act, gated, bias, kind, seed=0, host=False):
    x, weight, scale, b = _tensors(rows, d, out * (2 if gated else 1), experts, dtype, bias, seed)
    counts = _counts(kind, rows, experts, seed)
    cnt = torch.tensor(counts) if host else torch.tensor(counts, device="cuda")
    y = functions.linear_int8(x, cnt, weight, scale, b, ACTS[act][0], gated=gated)
    assert y.dtype == x.dtype and y.shape == (rows, out)
    _close(y, _reference(x, counts, weight, scale, b, act, gated))
    return y


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("gated", [False, True])
def test_small(dtype, act, gated):
    _check(37, 80, 96, 3, dtype, act, gated, True, "even")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,d,out,experts,kind", [
    (1, 1, 1, 1, "even"), (1, 1024, 512, 4, "one"), (2, 512, 1000, 32, "skewed"), (5, 17, 3, 2, "even"), (7, 3, 5, 2, "tail"), (130, 36, 44, 3, "skewed"),
    (129, 130, 65, 2, "even"), (300, 250, 130, 12, "tail"), (64, 256, 128, 64, "even"), (257, 72, 8, 2, "one"), (1000, 320, 200, 5, "skewed"),
    (33, 2000, 72, 2, "even"), (12, 128, 40, 2000, "skewed")])
def test_sizes(dtype, rows, d, out, experts, kind, gated):
    _check(rows, d, out, experts, dtype, "silu" if gated else "none", gated, rows % 2 == 0, kind, seed=rows)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["silu", "none", "relu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_large_enough_to_fill_the_card(dtype, act, gated):
    """512 tiles of 256 x 256 and more, contractions that end inside a slab, columns that end inside a tile, tail rows."""
    _check(8200, 1040, 4120, 4, dtype, act, gated, act in ("silu", "relu"), "tail" if act == "gelu" else "skewed")


@pytest.mark.parametrize("tile", ["256x256", "128x256", "128x128", "128x128+", "64x128"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,d,out,kind", [(700, 400, 328, "skewed"), (300, 10250, 136, "tail"), (150, 150, 5128, "even")])
def test_every_tile(monkeypatch, tile, gated, rows, d, out, kind):
    monkeypatch.setenv("FMOE_GEMM_TILE", tile)
    for act in (ACTS if rows == 700 else ("silu",)):
        for dtype in (torch.bfloat16, torch.float16):
            _check(rows, d, out, 3, dtype, act, gated, rows != 300, kind, seed=rows)


@pytest.mark.parametrize("tile", ["256x256", "128x256", "128x128", "128x128+", "64x128"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("out", [320, 331, 332, 334])
def test_every_tile_and_columns_of_any_number(monkeypatch, tile, gated, out):
    """Results in rows of whole 16-byte pieces, of whole groups of four columns, and of neither."""
    monkeypatch.setenv("FMOE_GEMM_TILE", tile)
    for dtype in DTYPES:
        _check(430, 270, out, 3, dtype, "gelu" if out % 4 else "none", gated, out != 334, "skewed", seed=out)


@pytest.mark.parametrize("gated", [False, True])
def test_few_rows_of_float32(gated):
    for rows in (1, 3, 16, 40, 64):
        for out in (132, 130):
            _check(rows, 300, out, 4, torch.float32, "silu", gated, rows != 16, "tail", seed=rows)


def test_largest_sums():
    """Every product 127 * 127, as many as there may be."""
    d = 131072
    x = torch.ones(3, d, device="cuda")
    weight, scale = functions.quantize_rows(torch.ones(1, 8, d, device="cuda"))
    weight[:, 1::2] = -127
    y = functions.linear_int8(x, torch.tensor([3], device="cuda"), weight, scale)
    want = torch.tensor([1.0, -1.0] * 4, device="cuda").double() * 127 * 127 * d * scale[0, 0].double() ** 2
    assert ((y.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("gated", [False, True])
def test_longest_rows_of_results(gated):
    """4 MiB to a row; wider ones are refused."""
    out = 1 << 21
    for rows in (3, 200):
        x, weight, scale, b = _tensors(rows, 16, out * (2 if gated else 1), 1, torch.bfloat16, True)
        y = functions.linear_int8(x, torch.tensor([rows], device="cuda"), weight, scale, b, gated=gated)
        some = weight[:, -70:] if not gated else torch.cat([weight[:, out - 70:out], weight[:, -70:]], dim=1)
        of = scale[:, -70:] if not gated else torch.cat([scale[:, out - 70:out], scale[:, -70:]], dim=1)
        bias = b[:, -70:] if not gated else torch.cat([b[:, out - 70:out], b[:, -70:]], dim=1)
        _close(y[:, -70:], _reference(x, [rows], some, of, bias, "none", gated))
        del y
    with pytest.raises(fmoe_native._lib.FmoeHipError):
        functions.linear_int8(x, torch.tensor([rows], device="cuda"), weight.new_zeros(1, (2 if gated else 1) * (out + 16), 16), torch.ones(1, (2 if gated else 1) * (out + 16), device="cuda"), gated=gated)


def test_decode_rows():
    for rows in (1, 2, 4, 16, 17, 33, 64, 128):
        for gated in (False, True):
            _check(rows, 1024, 1408, 8, torch.bfloat16, "silu", gated, rows % 2 == 0, "skewed", seed=rows)


def test_counts_on_the_host_and_table():
    y = _check(50, 64, 72, 3, torch.bfloat16, "gelu", False, True, "tail", host=True)
    x, weight, scale, b = _tensors(50, 64, 72, 3, torch.bfloat16, True)
    table = fmoe_native.segment_table(torch.tensor(_counts("tail", 50, 3), device="cuda"), 50)
    assert torch.equal(y, functions.linear_int8(x, None, weight, scale, b, torch.nn.GELU(), table=table))


def test_weights_that_lie_otherwise():
    x, weight, scale, b = _tensors(50, 70, 24, 3, torch.bfloat16, True)
    cnt = torch.tensor([20, 0, 30], device="cuda")
    want = functions.linear_int8(x, cnt, weight, scale, b)
    packed = weight.contiguous()                                              # rows of 70 bytes
    wide = torch.full((3, 24, 128), 77, dtype=torch.int8, device="cuda")      # rows of 128, other numbers behind them
    wide[:, :, :70] = weight
    turned = weight.transpose(1, 2).contiguous().transpose(1, 2)
    last = torch.empty(3 * 24 * 80 - 10, dtype=torch.int8, device="cuda").as_strided((3, 24, 70), (24 * 80, 80, 1))   # ends with its last number
    last.copy_(weight)
    for w in (packed, wide[:, :, :70], turned, last):
        assert torch.equal(functions.linear_int8(x, cnt, w, scale, b), want)


def test_rows_through_an_index():
    x, weight, scale, b = _tensors(20, 96, 40, 3, torch.bfloat16, True)
    index = torch.randint(0, 60, (45,), device="cuda")
    counts = [10, 15, 20]
    y = functions.linear_int8(x, torch.tensor(counts, device="cuda"), weight, scale, b, row_index=index, index_div=3)
    _close(y, _reference(x, counts, weight, scale, b, "none", False, at=index // 3))


def test_rows_behind_the_counted_ones_are_zeros_and_never_read():
    x, weight, scale, b = _tensors(40, 48, 33, 3, torch.bfloat16, True)
    x[25:] = float("nan")
    y = functions.linear_int8(x, torch.tensor([20, 0, 5], device="cuda"), weight, scale, b)
    assert not y[25:].any() and torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,d,out,experts,kind", [(1, 1, 4, 1, "even"), (1, 8192, 64, 2, "one"), (2, 4096, 520, 2, "even"), (8, 1024, 36, 3, "skewed"), (7, 1001, 128, 20, "even"),
                                                     (16, 512, 200, 3, "tail"), (16, 500, 132, 1, "one"), (16, 3, 8, 16, "even"), (5, 50, 2052, 600, "even"),
                                                     (17, 16, 8, 4, "even"), (3, 2736, 64, 2, "even")])
def test_few_rows_have_the_bits_that_they_have_among_many(rows, d, out, experts, kind, gated, dtype):
    """Rows rounded within the product (up to 16 of up to 8192 elements in all) and in a launch of their own."""
    x, weight, scale, b = _tensors(rows + 40, d, out * (2 if gated else 1), experts, dtype, True, seed=rows)
    counts = _counts(kind, rows, experts, seed=rows)
    here = sum(counts)
    if rows > 2:
        x[here // 2, d // 2] = float("inf")
    few = functions.linear_int8(x[:rows], torch.tensor(counts, device="cuda"), weight, scale, b, torch.nn.SiLU(), gated=gated)
    counts[-1] += 40
    many = functions.linear_int8(torch.cat([x[:here], x[rows:]]), torch.tensor(counts, device="cuda"), weight, scale, b, torch.nn.SiLU(), gated=gated)
    assert torch.equal(few[:here].nan_to_num(7.0), many[:here].nan_to_num(7.0)) and not few[here:].any()
    if rows > 2:
        assert torch.isnan(few[here // 2]).all()


def test_few_rows_through_an_index_and_strides():
    x, weight, scale, b = _tensors(20, 96, 40, 3, torch.bfloat16, True)
    index = torch.tensor([59, 0, 7, 7, 30, 58], device="cuda")
    counts = [2, 0, 3]
    wide = torch.full((20, 101), 9.0, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:97] = x
    for rows in (x, wide[:, 1:97]):
        y = functions.linear_int8(rows, torch.tensor(counts, device="cuda"), weight, scale, b, row_index=index, index_div=3)
        _close(y[:5], _reference(x, counts, weight, scale, b, "none", False, at=index[:5] // 3))
        assert not y[5:].any()
        _close(functions.linear_int8(rows[4:8], torch.tensor([1, 2, 1], device="cuda"), weight, scale, b),
               _reference(x[4:8], [1, 2, 1], weight, scale, b, "none", False))
    outside = functions.linear_int8(x, torch.tensor([1, 1, 1], device="cuda"), weight, scale, b, row_index=torch.tensor([-1, 60, 3], device="cuda"), index_div=3)
    assert torch.equal(outside[0], b[0]) and torch.equal(outside[1], b[1])   # (rows from nowhere are zeros)


def test_infinities_and_nan_show():
    x, weight, scale, b = _tensors(9, 48, 33, 1, torch.bfloat16, True)
    x[3, 5], x[7, 0] = float("inf"), float("nan")
    for act in ACTS:
        y = functions.linear_int8(x, torch.tensor([9], device="cuda"), weight, scale, b, ACTS[act][0])
        assert torch.isnan(y).all(dim=1).tolist() == [i in (3, 7) for i in range(9)] and torch.isfinite(y[[0, 1, 2, 4, 5, 6, 8]]).all()


def test_same_bits_on_another_stream_and_in_a_graph():
    x, weight, scale, b = _tensors(64, 256, 512, 8, torch.bfloat16, True)
    cnt = torch.tensor(_counts("even", 64, 8), device="cuda")
    run = lambda: functions.linear_int8(x, cnt, weight, scale, b, torch.nn.SiLU(), gated=True)
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.synchronize()
    assert torch.equal(first, second)
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


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype,d,h", [(torch.bfloat16, 64, 96), (torch.float16, 50, 33), (torch.float32, 64, 96)], ids=str)
def test_layer(gated, dtype, d, h):
    """The layer after quantize_experts against the two products of the float64 formula, each with the rows that the product before left."""
    torch.manual_seed(3)
    layer = (FMoEGatedMLP if gated else FMoETransformerMLP)(num_expert=6, d_model=d, d_hidden=h, top_k=2).to(dtype).cuda()
    with torch.no_grad():
        for p in layer.experts.parameters():
            p.copy_(torch.randn(p.shape) * (0.1 if p.dim() == 2 else p.shape[2] ** -0.5))
    plain = layer.experts
    x = torch.randn(5, 30, d, device="cuda").to(dtype)
    flat = x.reshape(-1, d)
    with torch.no_grad():
        before = layer(x)
        idx, score = layer.gate(flat)
        assert layer.quantize_experts() is layer
        for layer.enable_fuse in (False, True):
            after = layer(x)
            # 8 bits: a row's and a channel's steps are 1/254 of the largest of them, some 3 deviations: 1.2 % of a product each, four such
            assert ((after - before).float().norm() / before.float().norm()).item() <= 0.05
    # each token's experts one by one
    ex = layer.experts
    for t in range(0, 150, 17):
        got = torch.zeros(d, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(got)
        for k in range(2):
            e = int(idx[t, k])
            one = torch.tensor([1 if i == e else 0 for i in range(6)], device="cuda")
            mid = functions.linear_int8(flat[t:t + 1], one, ex.htoh4_weight, ex.htoh4_scale, ex.htoh4_bias, plain.activation, gated=gated)
            y = functions.linear_int8(mid, one, ex.h4toh_weight, ex.h4toh_scale, ex.h4toh_bias)
            got += y[0].double() * score[t, k].double()
            size += (y[0].double() * score[t, k].double()).abs()
        u = torch.finfo(dtype).eps / 2
        assert ((after.reshape(-1, d)[t].double() - got).abs() <= u * got.abs() + 4 * 2.0 ** -24 * size + 1e-7 * (dtype == torch.float16)).all()
    names = set(layer.state_dict())
    assert {"experts.htoh4_weight", "experts.h4toh_scale"} <= names and not any(n.startswith("experts.htoh4.") for n in names)
    with pytest.raises(NotImplementedError):
        layer(x.clone().requires_grad_(True))


def test_layer_moves_keep_the_scales():
    layer = FMoETransformerMLP(num_expert=2, d_model=32, d_hidden=48).cuda().quantize_experts()
    scale = layer.experts.htoh4_scale.clone()
    layer = layer.bfloat16()
    assert layer.experts.htoh4_scale.dtype == torch.float32 and torch.equal(layer.experts.htoh4_scale, scale)
    assert layer.experts.htoh4_bias.dtype == torch.bfloat16 and layer.experts.htoh4_weight.dtype == torch.int8
    with torch.no_grad():
        assert torch.isfinite(layer(torch.randn(5, 32, device="cuda").bfloat16())).all()


def test_wrong_tensors_are_refused():
    x, weight, scale, b = _tensors(8, 32, 24, 2, torch.bfloat16, True)
    cnt = torch.tensor([3, 5], device="cuda")
    call = lambda **kw: functions.linear_int8(*(kw.get(k, v) for k, v in (("x", x), ("cnt", cnt), ("weight", weight), ("scale", scale), ("bias", b))),
                                              kw.get("act"), gated=kw.get("gated", False), table=kw.get("table"))
    call()
    for error, kw in [(TypeError, {"weight": weight.short()}), (TypeError, {"scale": scale.double()}), (ValueError, {"scale": scale[:, :-1]}),
                      (ValueError, {"weight": weight[:, :, :-1]}), (ValueError, {"weight": weight[0]}), (TypeError, {"bias": b.float()}),
                      (ValueError, {"bias": b[:, :-1].contiguous()}), (TypeError, {"x": x.double()}), (ValueError, {"x": x[0]}), (ValueError, {"x": x.cpu()}),
                      (ValueError, {"weight": weight[:, :-1], "scale": scale[:, :-1], "bias": None, "gated": True}), (ValueError, {"cnt": cnt[:1]}),
                      (TypeError, {"cnt": cnt.int()}), (ValueError, {"cnt": torch.tensor([8, 1])}), (NotImplementedError, {"act": torch.nn.Tanh()}),
                      (NotImplementedError, {"x": x.clone().requires_grad_(True)}), (ValueError, {"table": fmoe_native.segment_table(cnt, 300)})]:
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(TypeError):
        functions.quantize_rows(x.double())
    with pytest.raises(_limit()):
        functions.linear_int8(torch.zeros(1, 131088, device="cuda"), torch.tensor([1], device="cuda"), torch.zeros(1, 1, 131088, dtype=torch.int8, device="cuda"),
                              torch.ones(1, 1, device="cuda"))


def _limit():
    from fastermoe_amd import _lib
    return _lib.FmoeHipError
