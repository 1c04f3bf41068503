"""The gate's balance loss, the experts' counts and mean probabilities, and the gradient of the logits against the definition in float64.

A probability is off by at most ``r = (20 + E / 64 + 2 range) 2^-24`` of itself: an exponential whose argument, a difference of logits within
``range``, was rounded, over a sum of ``E`` of them of which a lane adds ``E / 64`` one after the other.  Sums of probabilities over ``N`` tokens,
all positive, are off by ``(16 + N / 64) 2^-24`` more."""
import pytest
import torch

from fastermoe_amd import _lib, functions
from fastermoe_amd.gates import GShardGate, SwitchGate

pytestmark = pytest.mark.gpu
ULP32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _reference(logits, idx, mask, per, g_loss, g_prob):
    logits = logits.detach().double()
    n, e = logits.shape
    keep = torch.ones(n, dtype=torch.bool, device=logits.device) if mask is None else mask.reshape(-1) == 0
    full = keep & (logits > -float("inf")).any(1)
    named = idx.reshape(n, -1)[keep].reshape(-1) if n else idx.reshape(-1)
    named = named[(named >= 0) & (named < e)]
    counts = torch.zeros(e, dtype=torch.int64, device=logits.device).index_add_(0, named, torch.ones_like(named))
    p = torch.zeros_like(logits)
    p[full] = torch.softmax(logits[full], dim=1)
    t, s = int(keep.sum()), int(counts.sum())
    D = t if per == "token" else s
    total = p.sum(0)
    k = e / (D * D) if D else 0.0
    loss = k * float((counts * total).sum())
    prob = total / t if t else total * 0
    u = g_loss * k * (counts.double() - s / e)
    if g_prob is not None and t:
        u = u + g_prob.double() / t
    grad = p * (u - (p * u).sum(1, keepdim=True))
    finite = logits[full][logits[full].abs() < float("inf")]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    r = (20 + e / 64 + 2 * spread) * ULP32
    return counts, loss, prob, grad, p, u, r, (16 + n / 64) * ULP32


def _check(logits, idx, per="token", mask=None, g_loss=0.7, with_prob=True):
    logits = logits.detach().requires_grad_(True)
    n, e = logits.shape
    g_prob = torch.randn(e, device=logits.device) if with_prob else None
    loss, counts, prob = functions.balance_loss(logits, idx, per=per, mask=mask)
    outs, gs = [loss], [torch.tensor(g_loss, device=logits.device)]
    if with_prob:
        outs, gs = outs + [prob], gs + [g_prob]
    grad, = torch.autograd.grad(outs, logits, gs)
    counts64, loss64, prob64, grad64, p, u, r, chain = _reference(logits, idx, mask, per, g_loss, g_prob)
    assert counts.dtype == torch.int64 and torch.equal(counts, counts64)
    assert loss.dtype == prob.dtype == torch.float32 and loss.shape == () and grad.dtype == logits.dtype
    assert abs(float(loss.detach()) - loss64) <= (r + chain + 2 * ULP32) * abs(loss64)
    assert bool(((prob.double() - prob64).abs() <= (r + chain + 2 * ULP32) * prob64 + 1e-40).all())
    info = torch.finfo(logits.dtype)
    slack = 3 * r * p * (u.abs() + (p * u.abs()).sum(1, keepdim=True))
    limit = grad64.abs().clamp(min=info.smallest_normal) * (info.eps / 2) + slack
    off = (grad.double() - grad64).abs()
    assert bool((off <= limit).all()), float((off / limit).max())
    return loss.detach(), counts, prob.detach(), grad


def _inputs(n, e, k, dtype, seed=0, drop=0.0, skew=0.5):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(n, e, generator=gen) + skew * torch.randn(e, generator=gen)).to(TYPES[dtype])
    idx = logits.float().topk(k, dim=1).indices if n else torch.empty(0, k, dtype=torch.int64)
    if drop:
        idx = idx.masked_fill(torch.rand(n, k, generator=gen) < drop, -1)
    return logits.cuda(), idx.cuda()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("per", ["token", "slot"])
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (1, 2, 2), (1, 64, 1), (3, 5, 2), (1000, 16, 2), (777, 12, 1), (515, 8, 4), (4099, 7, 2),
                                   (300, 33, 8), (2048, 64, 1), (130, 100, 2), (257, 256, 8), (70, 500, 4), (65, 513, 2), (40, 1000, 2),
                                   (33, 2049, 1), (9, 4100, 2), (5, 8192, 8)])
def test_sizes(n, e, k, per, dtype, device):
    logits, idx = _inputs(n, e, k, dtype, drop=0.2 if per == "slot" else 0.0)
    _check(logits, idx, per, g_loss=300.0 if dtype == "f16" else 0.7)


@pytest.mark.parametrize("n", [20000, 262144])
def test_many_tokens(n, device):
    logits, idx = _inputs(n, 24, 2, "f32")
    _check(logits, idx)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("per", ["token", "slot"])
def test_padded_batches(per, dtype, device):
    """Masked tokens leave no trace, whatever their logits and indices hold; their gradients are zeros."""
    logits, idx = _inputs(600, 20, 2, dtype, drop=0.1)
    mask = torch.zeros(600, dtype=torch.bool, device=device)
    mask[550:] = True
    mask[::7] = True
    want = _check(logits, idx, per, mask)
    dirty = logits.clone()
    dirty[mask] = float("nan")
    dirty[::14, 3] = float("inf")
    torch.manual_seed(0)
    loss, counts, prob = functions.balance_loss(dirty.requires_grad_(True), idx.masked_fill(mask[:, None], 5), per, mask)
    assert torch.equal(loss, want[0]) and torch.equal(counts, want[1]) and torch.equal(prob, want[2])
    g, = torch.autograd.grad(loss, dirty)
    assert bool((g[mask] == 0).all()) and bool(g[~mask].isfinite().all())
    # the layer's own kind of mask: numbers, of any shape
    loss2 = functions.balance_loss(logits, idx, per, mask.view(3, 200).to(torch.int32) * 4)[0]
    assert torch.equal(loss2, want[0])


def test_everything_masked_dropped_or_absent(device):
    logits, idx = _inputs(50, 6, 2, "f32")
    for per in ("token", "slot"):
        loss, counts, prob, grad = _check(logits, idx, per, torch.ones(50, dtype=torch.bool, device=device))
        assert float(loss) == 0 and int(counts.sum()) == 0 and not bool(prob.any()) and not bool(grad.any())
        loss, counts, prob, grad = _check(logits, torch.full_like(idx, -1), per, with_prob=False)
        assert float(loss) == 0 and not bool(grad.any()) and abs(float(prob.sum()) - 1) < 1e-5
        loss, counts, prob, grad = _check(logits[:0], idx[:0], per)
        assert float(loss) == 0 and grad.shape == (0, 6)


def test_closed_experts_and_rows_without_any(device):
    """Logits of minus infinity: no probability and no gradient there, and none in rows of nothing else; the lowest finite number is a
    logit like any other."""
    logits, idx = _inputs(64, 9, 2, "f32")
    logits[:, 4] = -float("inf")
    logits[5] = -float("inf")
    logits[9] = torch.finfo(torch.float32).min
    logits[11, :3] = torch.finfo(torch.float32).min
    logits.requires_grad_(True)
    idx[idx == 4] = -1
    loss, counts, prob = functions.balance_loss(logits, idx)
    grad, = torch.autograd.grad(loss, logits)
    loss, prob = loss.detach(), prob.detach()
    p = torch.softmax(logits.detach().double(), 1)
    p[5] = 0
    want = 9 * float((counts * p.sum(0)).sum()) / 64 ** 2
    assert abs(float(loss) - want) <= 1e-6 * want and abs(float(prob[0]) - float(p[:, 0].sum() / 64)) < 1e-6
    assert bool(grad.isfinite().all()) and not bool(grad[5].any())
    closed = grad[:, 4] != 0
    closed[9] = False       # (that row's logits, the fourth among them, are all the lowest finite number)
    assert not bool(closed.any())
    nine = grad[9].double()
    u = 9 / 64 ** 2 * (counts.double() - counts.sum() / 9)
    p9 = p[9]
    assert torch.allclose(nine, p9 * (u - (p9 * u).sum()), rtol=1e-4, atol=1e-10)


def test_nan_shows(device):
    logits, idx = _inputs(40, 8, 1, "f32")
    logits[3, 2] = float("nan")
    loss, counts, prob = functions.balance_loss(logits.requires_grad_(True), idx)
    assert bool(loss.isnan())
    g, = torch.autograd.grad(loss, logits)
    assert bool(g[3].isnan().all()) and bool(g[4].isfinite().all())


def test_indices_out_of_range_are_skipped(device):
    logits, idx = _inputs(100, 8, 2, "f32")
    idx[3, 0], idx[4, 1], idx[5, 0], idx[6, 0] = 8, -7, 1 << 40, -(1 << 62)
    _check(logits, idx)
    _check(logits, idx.reshape(-1))     # as the noisy gate hands them out


def test_strided_logits_and_indices(device):
    logits, idx = _inputs(200, 16, 2, "bf16")
    wide = torch.zeros(200, 24, dtype=torch.bfloat16, device=device)
    wide[:, :16] = logits
    want = _check(logits, idx)
    torch.manual_seed(1)
    got = functions.balance_loss(wide[:, :16], idx.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(want[:3], got))
    one = torch.randn(1, 16, device=device, requires_grad=True)     # one row of logits for all tokens: its gradient is summed
    loss = functions.balance_loss(one.expand(50, 16), idx[:50])[0]
    g, = torch.autograd.grad(loss, one)
    flat = one.detach().expand(50, 16).contiguous().requires_grad_(True)
    full, = torch.autograd.grad(functions.balance_loss(flat, idx[:50])[0], flat)
    assert torch.allclose(g, full.sum(0, keepdim=True), rtol=1e-5, atol=1e-9)


def test_balanced_experts_lose_nothing_to_rounding(device):
    """Counts that are nearly equal: the gradient is the small difference, not the rounding of what it is the difference of."""
    n, e = 60000, 6
    idx = (torch.arange(n, device=device) % e).view(n, 1)
    idx[:3] = 0
    logits = torch.randn(n, e, device=device)
    _check(logits, idx, with_prob=False)


def test_gradients_against_differences(device):
    torch.manual_seed(2)
    logits, idx = _inputs(30, 7, 2, "f32", drop=0.2)
    mask = torch.arange(30, device=device) > 24
    gp = torch.randn(7, device=device)
    logits.requires_grad_(True)
    loss, counts, prob = functions.balance_loss(logits, idx, "slot", mask)
    g, = torch.autograd.grad([loss, prob], logits, [torch.tensor(1.0, device=device), gp])

    def value(l):
        p = torch.softmax(l, 1)[~mask].sum(0)
        s = float(counts.sum())
        return 7 * (counts * p).sum() / s ** 2 + (gp.double() * p / 25).sum()

    v = torch.randn(30, 7, dtype=torch.float64, device=device)
    at = logits.detach().double()
    want = float((value(at + 1e-5 * v) - value(at - 1e-5 * v)) / 2e-5)
    assert abs(float((g.double() * v).sum()) - want) <= 1e-5 * float((g.double() * v).abs().sum()) + 1e-9


@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives_and_one_gradient_alone(native, device, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_layer_call", None)
    logits, idx = _inputs(40, 6, 2, "f32")
    logits.requires_grad_(True)
    loss, counts, prob = functions.balance_loss(logits, idx)
    plain, = torch.autograd.grad(loss, logits, retain_graph=True)
    g, = torch.autograd.grad(loss, logits, create_graph=True)
    assert torch.allclose(g, plain, rtol=1e-4, atol=1e-9)
    second, = torch.autograd.grad(g.square().sum(), logits)
    l64 = logits.detach().double().requires_grad_(True)
    u = (6 / 40 ** 2 * (counts.double() - counts.sum() / 6))
    h, = torch.autograd.grad((torch.softmax(l64, 1) * u).sum(), l64, create_graph=True)
    want, = torch.autograd.grad(h.square().sum(), l64)
    assert torch.allclose(second.double(), want, rtol=1e-3, atol=1e-9)
    gp, = torch.autograd.grad(prob[2], logits, retain_graph=True)
    p = torch.softmax(logits.detach().double(), 1)
    assert torch.allclose(gp.double(), p * (torch.eye(6, device=device, dtype=torch.float64)[2] - p[:, 2:3]) / 40, rtol=1e-4, atol=1e-8)


def test_same_bits_every_time(device):
    logits, idx = _inputs(30000, 40, 2, "bf16")
    first = _check(logits, idx, with_prob=False)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _check(logits, idx, with_prob=False)))


def test_another_stream_and_a_graph(device):
    logits, idx = _inputs(1500, 24, 2, "f32")
    mask = torch.zeros(1500, dtype=torch.bool, device=device)

    def step():
        leaf = logits.detach().requires_grad_(True)
        loss, counts, prob = functions.balance_loss(leaf, idx, "slot", mask)
        return loss.detach(), counts, prob.detach(), torch.autograd.grad(loss, leaf)[0]

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
        logits.copy_(torch.randn(1500, 24, device=device))
        idx.copy_(logits.topk(2, dim=1).indices)
        mask.copy_(torch.rand(1500, device=device) < 0.1 * k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k


def test_both_nodes_give_the_same_bits(device, monkeypatch):
    """The node in native code and the Python one."""
    logits, idx = _inputs(500, 30, 2, "bf16", drop=0.1)
    mask = torch.rand(500, device=device) < 0.1
    g = torch.randn(30, device=device)

    def run():
        leaf = logits.detach().requires_grad_(True)
        loss, counts, prob = functions.balance_loss(leaf, idx, "slot", mask)
        return loss.detach(), counts, prob.detach(), torch.autograd.grad([loss, prob], leaf, [torch.tensor(2.0, device=device), g])[0]

    native = run()
    assert type(functions.balance_loss(logits.requires_grad_(True), idx)[0].grad_fn).__name__ != "BalanceLossBackward"
    monkeypatch.setattr(_lib, "_layer_call", None)
    assert type(functions.balance_loss(logits, idx)[0].grad_fn).__name__ == "BalanceLossBackward"
    assert all(torch.equal(a, b) for a, b in zip(native, run()))


def test_saved_tensors_may_come_back_otherwise(device):
    logits, idx = _inputs(60, 9, 2, "f32")
    logits.requires_grad_(True)
    want, = torch.autograd.grad(functions.balance_loss(logits, idx)[0], logits)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(device).t().contiguous().t()):
        loss = functions.balance_loss(logits, idx)[0]
    got, = torch.autograd.grad(loss, logits)
    assert torch.equal(got, want)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("order", ["sliced", "expanded", "transposed"])
def test_second_derivatives_of_logits_in_any_order(order, native, device, monkeypatch):
    """Logits that the kernels read a copy of: the gradient's gradient reaches them all the same.  (Some fifty float32 roundings on the way, 2^-24 each of
    magnitudes that cancel at most a hundredfold: 1e-3 of the largest.)"""
    if not native:
        monkeypatch.setattr(_lib, "_layer_call", None)
    shape, view = {"sliced": ((40, 9), lambda t: t[:, 2:8]), "expanded": ((1, 6), lambda t: t.expand(40, 6)), "transposed": ((6, 40), lambda t: t.t())}[order]
    leaf = torch.randn(shape, generator=torch.Generator().manual_seed(6)).to(device).requires_grad_(True)
    idx = torch.randint(6, (40, 2), generator=torch.Generator().manual_seed(7)).to(device)
    idx[::2] = 1
    gp = torch.linspace(-1, 1, 6, device=device)
    loss, counts, prob = functions.balance_loss(view(leaf), idx)
    first, = torch.autograd.grad([loss, prob], leaf, [torch.tensor(0.7, device=device), gp], create_graph=True)
    assert first.requires_grad
    second, = torch.autograd.grad(first.square().sum(), leaf)
    l64 = leaf.detach().double().requires_grad_(True)
    u = 0.7 * 6 / 40 ** 2 * (counts.double() - counts.sum() / 6) + gp.double() / 40
    h, = torch.autograd.grad((torch.softmax(view(l64), 1) * u).sum(), l64, create_graph=True)
    want, = torch.autograd.grad(h.square().sum(), l64)
    assert torch.allclose(first.detach().double(), h.detach(), rtol=1e-3, atol=1e-3 * float(h.abs().max()))
    assert torch.allclose(second.double(), want, rtol=1e-3, atol=1e-3 * float(want.abs().max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_small_probabilities(dtype, device):
    """Logits that lie whole numbers apart, so that no difference is rounded: an exponential is off by at most 4 steps of 2^-24, the sum of them by 12
    (additions of a lane and over the lanes), then a reciprocal, a product and a mean, by one each.  Twenty steps of every probability and gradient."""
    e = 81
    logits = -torch.arange(e, device=device, dtype=torch.float32).expand(7, e).to(TYPES[dtype]).contiguous().requires_grad_(True)
    idx = torch.zeros(7, 1, dtype=torch.int64, device=device)
    loss, counts, prob = functions.balance_loss(logits, idx)
    p = torch.softmax(logits.detach()[0].double(), 0)
    assert float(((prob.detach().double() - p).abs() / p).max()) <= 20 * ULP32
    if dtype == "f32":
        grad, = torch.autograd.grad(loss, logits, torch.tensor(1.0, device=device))
        u = e / 49 * (counts.double() - 7 / e)
        want = p * (u - (p * u).sum())
        # (u's own roundings, and those of a difference of two of its size)
        slack = 20 * ULP32 * p * (u.abs() + (p * u.abs()).sum())
        assert bool(((grad.double() - want).abs() <= slack + 20 * ULP32 * want.abs()).all())


@pytest.mark.parametrize("per", ["token", "slot"])
@pytest.mark.parametrize("n,e,dtype", [(65701, 60, "bf16"), (65701, 64, "f16"), (32901, 61, "f32"), (32901, 64, "f32"), (4201, 601, "bf16"), (4201, 600, "bf16"),
                                       (4201, 301, "f32"), (4201, 300, "f32"), (9000, 1100, "bf16"), (270001, 5, "f32")])
def test_several_tokens_ahead_in_the_backward(n, e, per, dtype, device):
    """Enough tokens for the backward to load several ahead, with experts in whole vectors and not, in one vector to a lane and two, one token behind a whole
    workgroup's."""
    logits, idx = _inputs(n, e, 2, dtype, drop=0.2 if per == "slot" else 0.0)
    mask = (torch.arange(n, device=device) % 11 == 0) if per == "slot" else None
    _check(logits, idx, per, mask, g_loss=300.0 if dtype == "f16" else 0.7)
