"""Layer norm, balance loss and activations kept in 8 bits where the package runs them: the gates, the experts, and a block of all three."""
import pytest
import torch
import torch.nn.functional as F

import fastermoe_amd as fmoe
from fastermoe_amd import fmoe_native
from fastermoe_amd.gates import GShardGate, SwitchGate
from helpers import TOL, assert_close
from test_act_checkpoint_gpu import CODES, act64, hold

pytestmark = pytest.mark.gpu


# ---- the gates' loss ------------------------------------------------------------------------

@pytest.mark.parametrize("gate_class", [GShardGate, SwitchGate])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("train", [True, False])
def test_gate_losses_and_gradients_are_those_of_the_torch_operators(gate_class, dtype, train, device, monkeypatch):
    """To float32's accuracy; 16-bit GShard logits, whose loss is of 16-bit means, to the bit."""
    torch.manual_seed(0)
    gate = gate_class(64, 12, 1, capacity=(0.2, 0.3)).to(device, dtype).train(train)
    x = torch.randn(700, 64, device=device, dtype=dtype)

    def run():
        gate.zero_grad()
        torch.manual_seed(7)
        leaf = x.detach().requires_grad_(True)
        idx, score = gate(leaf)
        loss = gate.get_loss()
        (loss * 3 + score.float().square().sum() * 1e-3).backward()
        return idx, loss.detach(), leaf.grad, gate.gate.weight.grad.clone()

    kernel = run()
    monkeypatch.setenv("FMOE_BALANCE_LOSS_KERNEL", "0")
    plain = run()
    assert torch.equal(kernel[0], plain[0]) and kernel[1].dtype == plain[1].dtype
    if gate_class is GShardGate and dtype != torch.float32:
        assert all(torch.equal(a, b) for a, b in zip(kernel, plain))
        return
    assert abs(float(kernel[1]) - float(plain[1])) <= 2e-6 * abs(float(plain[1]))
    tol = 2e-5 if dtype == torch.float32 else 2.0 ** -7
    for a, b in zip(kernel[2:], plain[2:]):
        assert_close(a, b, tol)


def test_gate_loss_reads_nothing_on_the_host(device):
    gate = GShardGate(32, 8, 1).to(device)
    x = torch.randn(300, 32, device=device)
    gate(x)
    torch.cuda.set_sync_debug_mode("error")
    try:
        gate(x)
        gate.get_loss().backward()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert gate.gate.weight.grad is not None


def test_gates_under_inference_mode(device):
    x = torch.randn(100, 32, device=device)
    for gate in (GShardGate(32, 8, 1).to(device), SwitchGate(32, 8, 1).to(device).eval()):
        with torch.no_grad():
            torch.manual_seed(1)
            gate(x)
            want = float(gate.get_loss())
        with torch.inference_mode():
            torch.manual_seed(1)
            gate(x)
            assert float(gate.get_loss()) == want


# ---- experts that keep their activations in 8 bits -----------------------------------------------

def _layer(dtype, act, d=96, h=160, e=6, k=2, **kwargs):
    torch.manual_seed(3)
    module = {"gelu": torch.nn.GELU(), "relu": torch.nn.ReLU(), "none": None}[act]
    layer = fmoe.FMoETransformerMLP(num_expert=e, d_model=d, d_hidden=h, top_k=k, activation=module, **kwargs)
    with torch.no_grad():
        for p in layer.experts.parameters():
            p.normal_(0, 0.1)
    return layer.to("cuda", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "relu", "none"])
@pytest.mark.parametrize("d,h", [(96, 160), (50, 77)])
@pytest.mark.parametrize("drops", [False, True])
def test_same_output_and_gradients_from_what_was_kept(d, h, act, dtype, drops, device):
    """The output to the bit.  The experts' gradients against float64 from the numbers that are held of the layer's own pre-activations, on feature sizes
    that the products over a device table take and others, with and without dropped slots."""
    kwargs = {"gate": lambda *a: GShardGate(*a, capacity=(0.3, 0.3))} if drops else {}
    layer = _layer(dtype, act, d, h, **kwargs)
    x = torch.randn(301, d, device=device).to(dtype)
    idx, score = (t.detach() for t in layer.gate(x))
    layer.gate.forward = lambda inp: (idx, score)
    experts = layer.experts
    dy = torch.randn(301, d, device=device).to(dtype)

    def run(on):
        layer.act_checkpoint = on
        layer.zero_grad()
        leaf = x.detach().requires_grad_(True)
        out = layer(leaf)
        out.backward(dy)
        return out.detach(), [leaf.grad] + [p.grad.clone() for p in experts.parameters()]

    out, _ = run(False)
    kept_out, grads = run(True)
    assert torch.equal(out, kept_out)
    # the layer's own pre-activations: the product over the sorted rows
    counts, pos, s2r = fmoe_native.route(idx, 6)
    n = int(counts.sum())
    rows = fmoe_native.gather_rows(x, pos[:n], index_div=2)
    w1, b1, w2, b2 = (t.detach() for t in (experts.htoh4.weight, experts.htoh4.bias, experts.h4toh.weight, experts.h4toh.bias))
    mid, pre = fmoe_native.linear_act_forward(rows, counts.cpu(), w1, b1, CODES[act], act == "gelu")
    v = hold(pre if act == "gelu" else mid)[2]
    mid64, slope = act64(v, act)
    owner = torch.repeat_interleave(torch.arange(6, device=device), counts)
    token = pos[:n] // 2
    g = dy.double()[token] * score.double().reshape(-1)[pos[:n]].unsqueeze(1)
    g_pre = torch.empty(n, h, dtype=torch.float64, device=device)
    want = {"w1": torch.zeros(6, h, d), "b1": torch.zeros(6, h), "w2": torch.zeros(6, d, h), "b2": torch.zeros(6, d)}
    want = {name: t.double().to(device) for name, t in want.items()}
    g_rows = torch.empty(n, d, dtype=torch.float64, device=device)
    for e in range(6):
        s = owner == e
        g_pre[s] = (g[s] @ w2[e].double()) * slope[s]
        want["w1"][e], want["b1"][e] = g_pre[s].t() @ rows[s].double(), g_pre[s].sum(0)
        want["w2"][e], want["b2"][e] = g[s].t() @ mid64[s], g[s].sum(0)
        g_rows[s] = g_pre[s] @ w1[e].double()
    g_x = torch.zeros(301, d, dtype=torch.float64, device=device).index_add_(0, token, g_rows)
    # (helpers.TOL is what the layer's gradients may be off from the oracle: the numbers held are given here)
    for got, ref in zip(grads, (g_x, want["w1"], want["b1"], want["w2"], want["b2"])):
        assert_close(got, ref, TOL[dtype])


def test_gradients_stay_near_the_whole_ones(device):
    """What keeping 8 bits costs: every element that is held is off by at most 2^-4 of itself, at random, so a sum over hundreds is off by far less."""
    layer = _layer(torch.float32, "gelu", 128, 256, 4)
    x = torch.randn(2000, 128, device=device)
    dy = torch.randn(2000, 128, device=device)

    def run(on):
        layer.act_checkpoint = on
        layer.zero_grad()
        layer(x).backward(dy)
        return [p.grad.clone() for p in layer.experts.parameters()]

    for a, b in zip(run(True), run(False)):
        assert float((a - b).norm() / b.norm()) <= 2.0 ** -4


@pytest.mark.parametrize("act,whole,kept", [("gelu", 8, 1), ("relu", 4, 1)])
def test_memory_between_forward_and_backward(act, whole, kept, device):
    """Bytes per element of [slots, d_hidden]: 8 (two float32 tensors), or 4 with ReLU, become one and a thirty-second."""
    layer = _layer(torch.float32, act, 64, 4096, 4, 1)
    x = torch.randn(1024, 64, device=device)
    held = {}
    for on in (False, True, False, True):
        layer.act_checkpoint = on
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = layer(x)
        held[on] = torch.cuda.memory_allocated() - before
        del out
    elements = 1024 * 4096
    assert held[False] >= whole * elements and held[True] <= (kept + 1 / 32) * elements + held[False] - whole * elements + (1 << 16)


def test_act_checkpoint_switch(device, monkeypatch):
    layer = _layer(torch.float32, "gelu")
    assert layer.act_checkpoint is False and "act_checkpoint" not in layer.state_dict()
    layer.act_checkpoint = True
    x = torch.randn(20, 96, device=device)
    name = lambda out: type(out.grad_fn.next_functions[0][0]).__name__
    assert name(layer(x)) == "MOERoutedMLPCheckpointedBackward"
    with torch.no_grad():
        layer(x)
    layer.enable_fuse = True       # the pipeline stands back
    assert name(layer(x)) == "MOERoutedMLPCheckpointedBackward"
    layer.enable_fuse = False
    layer.experts.activation = torch.nn.Tanh()
    with pytest.raises(NotImplementedError, match="act_checkpoint"):
        layer(x)
    with torch.no_grad():
        layer(x)                   # (nothing is kept)
    layer.experts.activation = torch.nn.GELU()
    with pytest.raises(NotImplementedError, match="float64"):
        layer.double()(x.double())
    monkeypatch.setenv("FMOE_ACT_CHECKPOINT", "1")
    assert _layer(torch.float32, "gelu").act_checkpoint
    other = fmoe.FMoETransformerMLP(num_expert=2, d_model=8, d_hidden=8)
    other.experts = torch.nn.Linear(8, 8)
    assert other.act_checkpoint is False
    with pytest.raises(AttributeError):
        other.act_checkpoint = True


def test_inside_an_activation_checkpoint(device):
    """torch.utils.checkpoint around a layer that keeps 8 bits: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    layer = _layer(torch.bfloat16, "gelu")
    layer.act_checkpoint = True
    x = torch.randn(64, 96, device=device).to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn(64, 96, device=device).to(torch.bfloat16)
    params = [x] + list(layer.experts.parameters())
    want = torch.autograd.grad(layer(x), params, dy)
    got = torch.autograd.grad(checkpoint(layer, x, use_reentrant=False), params, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- a block ------------------------------------------------------------------------------------

def _reference_block(block, x, idx, dy, loss_weight):
    """Output and gradients in float64 of FMoEPositionwiseFF with GELU experts that keep 8 bits and a top-2 gate with GShard's loss."""
    ps = {name: p.detach().double().requires_grad_(True) for name, p in block.named_parameters()}
    x64 = x.detach().double().requires_grad_(True)
    n, d = x.shape
    norm = lambda t: F.layer_norm(t, (d,), ps["layer_norm.weight"], ps["layer_norm.bias"], block.layer_norm.eps)
    inp = norm(x64) if block.pre_lnorm else x64
    logits = inp @ ps["gate.gate.weight"].t() + ps["gate.gate.bias"]
    e = logits.shape[1]
    counts = torch.bincount(idx.reshape(-1), minlength=e).double()
    loss = e * (counts / n * torch.softmax(logits, 1).mean(0)).sum()
    out = torch.zeros_like(x64)

    class Kept(torch.autograd.Function):
        @staticmethod
        def forward(ctx, pre):
            ctx.v = hold(pre.float())[2]
            return F.gelu(pre)

        @staticmethod
        def backward(ctx, g):
            return g * act64(ctx.v, "gelu")[1]

    class Second(torch.autograd.Function):   # a linear layer whose weight gradient is made from the activation again
        @staticmethod
        def forward(ctx, mid, pre, w):
            ctx.save_for_backward(pre, w)
            return mid @ w.t()

        @staticmethod
        def backward(ctx, g):
            pre, w = ctx.saved_tensors
            return g @ w, None, g.t() @ act64(hold(pre.float())[2], "gelu")[0]

    for j in range(2):
        for k in range(e):
            rows = (idx[:, j] == k).nonzero().reshape(-1)
            if rows.numel() == 0:
                continue
            pre = inp[rows] @ ps["experts.htoh4.weight"][k].t() + ps["experts.htoh4.bias"][k]
            y = Second.apply(Kept.apply(pre), pre.detach(), ps["experts.h4toh.weight"][k]) + ps["experts.h4toh.bias"][k]
            out = out.index_add(0, rows, y * logits.gather(1, idx)[rows, j:j + 1])
    out = x64 + out if block.pre_lnorm else norm(x64 + out)
    names = list(ps)
    grads = torch.autograd.grad([out, loss], [x64] + [ps[k] for k in names], [dy.double(), torch.tensor(loss_weight, dtype=torch.float64, device=x.device)])
    return out.detach(), loss.detach(), grads[0], dict(zip(names, grads[1:]))


@pytest.mark.parametrize("pre_lnorm", [True, False])
@pytest.mark.parametrize("n", [1, 333])
def test_a_training_step_of_a_block(n, pre_lnorm, device):
    """Norm, gate with its loss, experts that keep 8 bits, residual: a float32 step against float64."""
    torch.manual_seed(11)
    d, h, e = 64, 96, 5
    block = fmoe.FMoEPositionwiseFF(num_expert=e, d_model=d, d_hidden=h, top_k=2, pre_lnorm=pre_lnorm,
                                    gate=lambda *a: GShardGate(*a, capacity=(8.0, 8.0))).to(device)
    block.gate.random_routing = False
    block.act_checkpoint = True
    with torch.no_grad():
        for name, p in block.named_parameters():
            p.add_(torch.randn_like(p) * 0.1)
    x, dy = torch.randn(n, d, device=device), torch.randn(n, d, device=device)
    leaf = x.clone().requires_grad_(True)
    seen = {}
    block.gate_hook = lambda idx, score, _: seen.update(idx=idx)
    out = block(leaf)
    loss = block.gate.get_loss()
    torch.autograd.backward([out, loss], [dy, torch.tensor(0.05, device=device)])
    want_out, want_loss, want_x, want = _reference_block(block, x, seen["idx"], dy, 0.05)
    assert_close(out.detach(), want_out, 1e-5, "out")
    assert abs(float(loss.detach()) - float(want_loss)) <= 1e-5 * float(want_loss)
    # (float32 products of a step: helpers.TOL, on magnitudes that the norm's gradient, a difference, may lose a digit of)
    assert_close(leaf.grad, want_x, 1e-4, "grad_x")
    for name, p in block.named_parameters():
        assert_close(p.grad, want[name], 1e-4, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pre_lnorm", [True, False])
def test_block_is_the_layer_and_the_norm(pre_lnorm, dtype, device):
    """Against the module's layer and torch's layer norm in float32, on inputs of three dimensions; parameter names; dropout."""
    torch.manual_seed(2)
    block = fmoe.FMoEPositionwiseFF(num_expert=4, d_model=32, d_hidden=64, top_k=2, pre_lnorm=pre_lnorm, dropout=0.5).to(device, dtype).eval()
    assert {"layer_norm.weight", "layer_norm.bias", "gate.gate.weight", "experts.htoh4.weight"} <= set(block.state_dict())
    x = torch.randn(6, 5, 32, device=device).to(dtype)
    layer = super(fmoe.FMoEPositionwiseFF, block).forward
    norm = lambda t: F.layer_norm(t.float(), (32,), block.layer_norm.weight.float(), block.layer_norm.bias.float(), block.layer_norm.eps)
    with torch.no_grad():
        got = block(x)
        want = x.float() + layer(norm(x).to(dtype)).float() if pre_lnorm else norm((x + layer(x)).to(dtype))
        assert got.shape == x.shape and got.dtype == dtype
        # (a half step of the type on the sum and on the result, and what the norm's scale, here below 4, makes of the first)
        assert_close(got, want, 1e-5 if dtype == torch.float32 else 2.0 ** -6)
        block.train()
        torch.manual_seed(4)
        a = block(x)
        torch.manual_seed(4)
        assert torch.equal(a, block(x)) and not torch.equal(a, got)


def test_block_with_a_module_of_the_users(device):
    """A replaced or hooked norm is called."""
    block = fmoe.FMoEPositionwiseFF(num_expert=4, d_model=32, d_hidden=64, pre_lnorm=True).to(device)
    x = torch.randn(9, 32, device=device)
    with torch.no_grad():
        want = block(x)
        calls = []
        handle = block.layer_norm.register_forward_hook(lambda *a: calls.append(1))
        assert torch.allclose(block(x), want, rtol=1e-5, atol=1e-5) and calls == [1]
        handle.remove()
        block.layer_norm = torch.nn.RMSNorm(32).to(device)
        assert not torch.allclose(block(x), want, rtol=1e-3, atol=1e-3)


def test_block_in_a_graph(device):
    """A training step of a block captured and replayed on new inputs, between eager work: every replay as the eager step."""
    torch.manual_seed(9)
    block = fmoe.FMoEPositionwiseFF(num_expert=8, d_model=64, d_hidden=128, top_k=2, pre_lnorm=True).to(device, torch.bfloat16)
    block.act_checkpoint = True
    x, dy = (torch.randn(256, 64, device=device).to(torch.bfloat16) for _ in range(2))
    weights = [p.detach() for p in block.parameters()]

    def step():
        leaves = [w.detach().requires_grad_(True) for w in weights]
        leaf = x.detach().requires_grad_(True)
        out = torch.func.functional_call(block, dict(zip([n for n, _ in block.named_parameters()], leaves)), (leaf,))
        return (out.detach(),) + torch.autograd.grad(out, [leaf] + leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(torch.randn(256, 64, device=device))
        dy.copy_(torch.randn(256, 64, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k


class _UsersExperts(torch.nn.Module):
    """Experts of a user's own that the fused pipeline takes, with a switch that happens to have the name of this package's."""
    act_checkpoint = True

    def __init__(self):
        super().__init__()
        self.htoh4, self.h4toh = fmoe.FMoELinear(4, 32, 64), fmoe.FMoELinear(4, 64, 32)
        self.activation = torch.nn.GELU()

    def forward(self, inp, fwd_expert_count):
        return self.h4toh(self.activation(self.htoh4(inp, fwd_expert_count)), fwd_expert_count)


def test_users_experts_with_a_switch_of_that_name(device):
    layer = fmoe.FMoE(num_expert=4, d_model=32, top_k=2)
    layer.experts, layer.experts_fused = _UsersExperts(), True
    layer = layer.to(device)
    x = torch.randn(50, 32, device=device, requires_grad=True)
    want = layer(x)
    layer.enable_fuse = True
    got = layer(x)
    assert_close(got.detach(), want.detach(), TOL[torch.float32])
    got.sum().backward()


def test_block_with_parameters_and_tokens_that_the_kernel_does_not_take(device):
    """Parameters that lie apart go to the module, as any module's would; tokens of another length are the module's error."""
    block = fmoe.FMoEPositionwiseFF(num_expert=4, d_model=32, d_hidden=64, pre_lnorm=True).to(device)
    x = torch.randn(9, 32, device=device)
    with torch.no_grad():
        block.layer_norm.weight.normal_()
        want = block(x)
        wide = torch.empty(32, 2, device=device)
        wide[:, 0] = block.layer_norm.weight
        block.layer_norm.weight = torch.nn.Parameter(wide[:, 0])
        assert not block.layer_norm.weight.is_contiguous()
        assert torch.allclose(block(x), want, rtol=1e-5, atol=1e-5)
        block.layer_norm = torch.nn.LayerNorm(32, elementwise_affine=False).to(device)
        for pre in (True, False):
            block.pre_lnorm = pre
            with pytest.raises(RuntimeError, match="normalized_shape"):
                block(torch.randn(4, 64, device=device))
