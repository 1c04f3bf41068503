"""Gated experts, their rounding to 8-bit integers and the products of those as a program uses them together: trained, rounded, served a token at a time; from two
streams at once; captured; and by way of Python where the native calls are off."""
import copy

import pytest
import torch

from fastermoe_amd import FMoEGatedMLP, FMoEPositionwiseFF, FMoETransformerMLP, _lib, fmoe_native, functions

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _layer(dtype, d=64, h=96, experts=6, seed=0):
    torch.manual_seed(seed)
    layer = FMoEGatedMLP(num_expert=experts, d_model=d, d_hidden=h, top_k=2).to(dtype).cuda()
    with torch.no_grad():
        for p in layer.experts.parameters():
            p.copy_(torch.randn(p.shape) * (0.1 if p.dim() == 2 else p.shape[2] ** -0.5))
    return layer


def _tensors(rows, d, h, experts, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *shape, scale=1.0: (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)
    return (make(rows, d), make(experts, 2 * h, d, scale=d ** -0.5), make(experts, 2 * h, scale=0.1), make(experts, d, h, scale=h ** -0.5),
            make(experts, d, scale=0.1))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d,h", [(64, 96), (50, 33)])
def test_train_round_serve(dtype, d, h):
    """Steps of a block with gated experts move every parameter; its layer, rounded, answers near what it did, and a token at a time gives the bits that the tokens
    give together (the rows' sums are integers)."""
    torch.manual_seed(1)
    block = FMoEPositionwiseFF(num_expert=4, d_model=d, d_hidden=h, top_k=2, gated=True, pre_lnorm=True).to(dtype).cuda()
    with torch.no_grad():
        for p in block.experts.parameters():
            p.copy_(torch.randn(p.shape) * (0.1 if p.dim() == 2 else p.shape[2] ** -0.5))
    before = copy.deepcopy(block.state_dict())
    x = torch.randn(3, 20, d, device="cuda").to(dtype)
    opt = torch.optim.SGD(block.parameters(), lr=0.5)
    for _ in range(2):
        opt.zero_grad()
        block(x).float().square().mean().backward()
        grads = {n: p.grad for n, p in block.named_parameters()}
        assert all(g is not None and torch.isfinite(g).all() for g in grads.values())
        opt.step()
    moved = [n for n, p in block.named_parameters() if not torch.equal(p, before[n])]
    assert all(any(part in n for n in moved) for part in ("htoh4.weight", "h4toh.weight", "gate", "layer_norm"))
    with torch.no_grad():
        full = block(x)
        block.quantize_experts()
        rounded = block(x)
        # 8 bits: about 1.2 % of a product each (see tests/test_int8_gpu.py), two products and a gate's: 5 % of the experts' part, whose size is of the rows'
        spread = (full.float() - x.float()).square().mean().sqrt()
        assert ((rounded.float() - full.float()).square().mean().sqrt() <= 0.05 * spread + 4 * torch.finfo(dtype).eps * full.float().abs().max())
        flat = x.reshape(-1, d)
        together = block(flat)
        for i in (0, 17, 59):
            # (the gate's logits and the norm are made row by row too)
            one = block(flat[i:i + 1])
            assert (one[0].float() - together[i].float()).abs().max() <= 8 * torch.finfo(dtype).eps * together.float().abs().max()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,d,h", [(9, 64, 96), (9, 50, 33), (400, 64, 96), (400, 51, 34)])
def test_the_python_way_has_the_same_bits(monkeypatch, dtype, rows, d, h):
    x, w1, b1, w2, b2 = _tensors(rows, d, h, 3, dtype)
    counts = torch.tensor([rows // 3, 0, rows // 2], device="cuda")
    gy = torch.randn(rows, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(dtype)
    q, s = functions.quantize_rows(w1)

    def both():
        leaves = [t.clone().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
        y = functions.gated_mlp(leaves[0], counts, *leaves[1:], torch.nn.SiLU())
        grads = torch.autograd.grad(y, leaves, gy)
        return [y.detach(), *grads, functions.linear_int8(x, counts, q, s, b1, torch.nn.GELU(), gated=True)]
    native = both()
    monkeypatch.setattr(_lib, "load_layer_call", lambda: None)
    for a, b in zip(native, both()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,d,h", [(torch.bfloat16, 64, 96), (torch.bfloat16, 51, 33), (torch.float32, 64, 96), (torch.float32, 50, 33)], ids=str)
def test_two_streams_at_once(dtype, d, h):
    """The same weights, different rows, workspaces of their own: each call has the bits that it has alone."""
    _, w1, b1, w2, b2 = _tensors(1, d, h, 4, dtype)
    xs = [_tensors(n, d, h, 4, dtype, seed=n)[0] for n in (700, 650, 12, 300)]
    counts = [torch.tensor([n // 2, 0, n // 4, n // 8], device="cuda") for n in (700, 650, 12, 300)]
    q, s = functions.quantize_rows(w1)

    def run(i):
        leaves = [t.detach().requires_grad_(True) for t in (xs[i], w1, b1, w2, b2)]
        y = functions.gated_mlp(leaves[0], counts[i], *leaves[1:], torch.nn.SiLU())
        return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y)), functions.linear_int8(xs[i], counts[i], q, s, b1, torch.nn.SiLU(), gated=True)]
    alone = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(3):
        results = []
        for i, stream in enumerate(streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                results.append(run(i))
        torch.cuda.synchronize()
        for a, b in zip(alone, results):
            for one, other in zip(a, b):
                assert torch.equal(one, other)


@pytest.mark.parametrize("dtype,d,h", [(torch.bfloat16, 64, 96), (torch.float16, 51, 33), (torch.float32, 64, 96), (torch.float32, 50, 33)], ids=str)
def test_captured_forward_and_backward(dtype, d, h):
    """Two graphs of different sizes, replayed in turn with eager work between; counts and rows change between replays."""
    graphs = []
    for n in (90, 40):
        x, w1, b1, w2, b2 = _tensors(n, d, h, 3, dtype, seed=n)
        gy = _tensors(n, d, h, 3, dtype, seed=n + 1)[0]
        counts = torch.tensor([n // 3, n // 4, n // 5], device="cuda")

        def run(x=x, w1=w1, b1=b1, w2=w2, b2=b2, gy=gy, counts=counts):
            leaves = [t.detach().requires_grad_(True) for t in (x, w1, b1, w2, b2)]
            y = functions.gated_mlp(leaves[0], counts, *leaves[1:], torch.nn.GELU())
            return [y.detach(), *torch.autograd.grad(y, leaves, gy)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        graphs.append((graph, held, run, x, counts))
    gen = torch.Generator(device="cuda").manual_seed(9)
    for _ in range(4):
        for graph, held, run, x, counts in graphs:
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
            counts.copy_(counts.roll(1))
            graph.replay()
        torch.cuda.synchronize()
        for graph, held, run, x, counts in graphs:
            for a, b in zip(held, run()):
                assert torch.equal(a, b)


def test_a_captured_token_of_a_rounded_layer():
    layer = _layer(torch.bfloat16, 128, 256, 8).quantize_experts().eval()
    token = torch.randn(1, 128, device="cuda").bfloat16()
    with torch.no_grad():
        layer(token)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(token)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(token)
        gen = torch.Generator(device="cuda").manual_seed(2)
        for _ in range(4):
            token.copy_(torch.randn(token.shape, device="cuda", generator=gen))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, layer(token))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_the_same_row_twice_and_weights_of_one_expert_for_all(dtype):
    """Rows that an index names more than once; weights that are one expert's, seen by several (8-bit ones expanded, others copied, their gradient summed; expanded ones, as any
    weights that are not contiguous, are refused)."""
    x, w1, b1, w2, b2 = _tensors(10, 64, 48, 1, dtype)
    q, s = functions.quantize_rows(w1)
    index = torch.tensor([3, 3, 3, 0, 9, 9], device="cuda")
    counts = torch.tensor([6], device="cuda")
    assert torch.equal(functions.linear_int8(x, counts, q, s, b1, row_index=index), functions.linear_int8(x[index], counts, q, s, b1))
    shared = q.expand(3, -1, -1)
    three = functions.linear_int8(x, torch.tensor([4, 3, 3], device="cuda"), shared, s.expand(3, -1), b1.expand(3, -1))
    assert torch.equal(three, functions.linear_int8(x, torch.tensor([10], device="cuda"), q, s, b1))
    w = w1.clone().requires_grad_(True)
    rows = torch.tensor([4, 3, 3], device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        functions.gated_mlp(x, rows, w.expand(3, -1, -1), b1.expand(3, -1), w2.expand(3, -1, -1), None, torch.nn.SiLU())
    three_times = [t.expand(3, *t.shape[1:]).contiguous() for t in (w, b1, w2)]
    y = functions.gated_mlp(x, rows, *three_times, None, torch.nn.SiLU())
    (shared_grad,) = torch.autograd.grad(y, w, torch.ones_like(y))
    one = w1.clone().requires_grad_(True)
    z = functions.gated_mlp(x, torch.tensor([10], device="cuda"), one, b1, w2, None, torch.nn.SiLU())
    (grad,) = torch.autograd.grad(z, one, torch.ones_like(z))
    assert torch.equal(y, z)
    # three parts, each rounded to the type, and two sums of those: 5 half steps of the largest
    assert (shared_grad.float() - grad.float()).abs().max() <= 5 * torch.finfo(dtype).eps / 2 * 3 * grad.float().abs().max()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d,h", [(64, 96), (51, 33)])
@pytest.mark.parametrize("rows", [0, 1, 7, 300, 3000])
def test_no_expert_has_rows(rows, dtype, d, h):
    """All rows behind the experts': zeros, as their gradients and the weights' are, whatever the rows hold."""
    x, w1, b1, w2, b2 = _tensors(rows, d, h, 3, dtype)
    x.fill_(float("nan"))
    counts = torch.zeros(3, dtype=torch.int64, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w1, b1, w2, b2)]
    y = functions.gated_mlp(leaves[0], counts, *leaves[1:], torch.nn.SiLU())
    assert y.shape == (rows, d) and not y.any()
    for t, g in zip(leaves, torch.autograd.grad(y, leaves, torch.full_like(y, float("nan")))):
        assert g.shape == t.shape and not g.any()
    q, s = functions.quantize_rows(w1.detach())
    with torch.no_grad():
        y = functions.linear_int8(x, counts, q, s, b1, torch.nn.GELU(), gated=True)
    assert y.shape == (rows, h) and not y.any()


def test_tables_of_other_sizes_are_refused():
    x, w1, b1, w2, b2 = _tensors(10, 64, 48, 2, torch.bfloat16)
    counts = torch.tensor([4, 4], device="cuda")
    wrong = fmoe_native.segment_table(counts, 500)
    q, s = functions.quantize_rows(w1)
    for call in (lambda: functions.gated_mlp(x, None, w1, b1, w2, b2, torch.nn.SiLU(), table=wrong),
                 lambda: functions.linear_int8(x, None, q, s, b1, table=wrong)):
        with pytest.raises((ValueError, TypeError)):
            call()


class _Adapter(torch.nn.Module):
    """A linear with something added, and a ``weight`` of its own."""

    def __init__(self, linear, features):
        super().__init__()
        self.linear, self.more = linear, torch.nn.Parameter(torch.linspace(-1, 1, features, device="cuda"))

    weight = property(lambda self: self.linear.weight)
    bias = property(lambda self: self.linear.bias)

    def forward(self, inp, fwd_expert_count):
        return self.linear(inp, fwd_expert_count) + self.more


@pytest.mark.parametrize("name", ["htoh4", "h4toh"])
@pytest.mark.parametrize("fuse", [False, True])
def test_gated_experts_call_what_stands_in_a_linears_place(name, fuse):
    """A module in a linear's place, or a hook on it, takes part: as with a bias of as much more."""
    torch.manual_seed(5)
    layer = FMoEGatedMLP(num_expert=4, d_model=24, d_hidden=40, top_k=2).cuda()
    linear = getattr(layer.experts, name)
    x = torch.randn(30, 24, device="cuda", requires_grad=True)
    more = torch.linspace(-1, 1, linear.out_feat, device="cuda")
    layer.enable_fuse = fuse
    plain = layer(x).detach()
    with torch.no_grad():
        linear.bias += more
        want = layer(x)
        linear.bias -= more
    # (float32 all through: products in another order)
    close = lambda got: torch.allclose(got, want, rtol=1e-4, atol=1e-5) and not torch.allclose(got, plain, rtol=1e-2, atol=1e-2)
    hook = linear.register_forward_hook(lambda module, args, out: out + more)
    assert close(layer(x))
    hook.remove()
    adapter = _Adapter(linear, linear.out_feat)
    setattr(layer.experts, name, adapter)
    y = layer(x)
    assert close(y)
    y.square().sum().backward()
    assert adapter.more.grad is not None and adapter.more.grad.abs().max() > 0 and linear.weight.grad is not None


def test_gated_experts_past_one_calls_sizes():
    """float32 weights of 2 GiB to an expert: module by module.  Errors: sums of n float32 products, 16 2^-24 sqrt(n) of their norm (see tests/test_gated_gpu.py)
    for each of the two products, and as much again for what the first one's do to the second."""
    d = h = 1 << 14
    with torch.device("cuda"):
        layer = FMoEGatedMLP(num_expert=1, d_model=d, d_hidden=h, top_k=1, bias=False)
        with torch.no_grad():
            layer.experts.htoh4.weight.normal_().mul_(d ** -0.5)
            layer.experts.h4toh.weight.normal_().mul_(h ** -0.5)
    assert not fmoe_native.gated_mlp_supported(torch.float32, d, h)
    x = torch.randn(5, d, device="cuda", requires_grad=True)
    y = layer(x)
    gy = torch.randn_like(y)
    y.backward(gy)
    ex = layer.experts
    with torch.no_grad():
        score = layer.gate(x)[1].double().reshape(5, 1)
        w1, w2 = ex.htoh4.weight[0].double(), ex.h4toh.weight[0].double()
        g, u = (x.double() @ w1.t()).chunk(2, dim=1)
        a = torch.nn.functional.silu(g)
        want = (a * u) @ w2.t() * score
        norm = lambda t: t.double().norm().item()
        tol = 4 * 16 * 2.0 ** -24 * (d ** 0.5)
        assert norm(y - want) <= tol * norm(want)
        dy = gy.double() * score
        assert norm(ex.h4toh.weight.grad[0] - dy.t() @ (a * u)) <= tol * norm(dy.t() @ (a * u))
        dm = dy @ w2
        s = torch.sigmoid(g)
        dg = dm * u * s * (1 + g * (1 - s))
        got = ex.htoh4.weight.grad[0]
        assert norm(got[:h] - dg.t() @ x.double()) <= tol * norm(dg.t() @ x.double())
        assert norm(got[h:] - (dm * a).t() @ x.double()) <= tol * norm((dm * a).t() @ x.double())
    layer.zero_grad(set_to_none=True)


@pytest.mark.parametrize("kind", [FMoETransformerMLP, FMoEGatedMLP])
def test_experts_past_the_sizes_of_8_bit_products_stay_as_they_are(kind):
    with torch.device("cuda"):
        layer = kind(num_expert=1, d_model=16, d_hidden=(1 << 21) + 16, top_k=1).half()
    before = layer.experts
    x = torch.randn(3, 16, device="cuda").half()
    with torch.no_grad():
        want = layer(x)
        with pytest.raises(NotImplementedError, match="htoh4"):
            layer.quantize_experts()
        assert layer.experts is before and torch.equal(layer(x), want)
