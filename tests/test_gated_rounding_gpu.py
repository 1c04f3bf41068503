"""What a gated block of 16-bit types rounds, to the bit, and its sizes whose offsets pass 31 bits.

The backward rounds dg = dm u act'(g) and du = dm act(g) once each, from float32: neither dm = dy W2 is rounded before, nor are g and u, which the forward leaves for it.
Rows x = (r, 0, ..) make g and u columns of the weights, times r: with r = 1 exact in the type, else products of two numbers of 8 bits, exact in float32 only; dy = (p, 0, ..) makes dm = p W2[0], a product of two numbers of 8 bits, exact in float32 and not in the type;
columns of W1 that x does not see pick single elements of (dg, du) out for the gradient of x, exact as well."""
import pytest
import torch

from fastermoe_amd import fmoe_native, functions
from test_gated_gpu import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", [None, torch.nn.ReLU()], ids=["none", "relu"])
@pytest.mark.parametrize("rows,d,h,experts", [(1, 64, 96, 2), (40, 64, 96, 3), (3000, 512, 1024, 4), (9000, 1024, 2048, 2), (30, 51, 33, 3), (700, 501, 1303, 5),
                                              (9000, 501, 1303, 2)])
@pytest.mark.parametrize("exact", [True, False], ids=["exact", "products"])
def test_the_gradients_of_the_halves_are_rounded_once(dtype, act, rows, d, h, experts, exact):
    gen = torch.Generator().manual_seed(rows + d)
    whole = lambda *shape: torch.randint(128, 256, shape, generator=gen).float() * (1 - 2 * torch.randint(0, 2, shape, generator=gen))
    e_of = torch.arange(rows) * experts // rows
    counts = torch.bincount(e_of, minlength=experts)
    gate, lin = whole(experts, h) / 128, whole(experts, h) / 128
    w1 = torch.zeros(experts, 2 * h, d)
    w1[:, :h, 0], w1[:, h:, 0] = gate, lin
    picked = torch.randint(0, 2 * h, (experts, d - 1), generator=gen)
    for e in range(experts):
        w1[e, picked[e], torch.arange(1, d)] = 1
    w2 = torch.zeros(experts, d, h)
    w2[:, 0] = whole(experts, h) / 4096
    x, gy = torch.zeros(rows, d), torch.zeros(rows, d)
    gy[:, 0] = whole(rows) / 16
    x[:, 0] = 1 if exact else whole(rows) / 128
    x, w1, w2, gy = (t.to(dtype).cuda() for t in (x, w1, w2, gy))
    x.requires_grad_(True)
    y = functions.gated_mlp(x, counts.cuda(), w1, None, w2, None, act)
    got, = torch.autograd.grad(y, x, gy)

    f = lambda t: t.float().cpu()
    dm = f(gy)[:, :1] * f(w2)[e_of, 0]

    def halves(dm, held=torch.float32):
        g, u = ((f(x)[:, :1] * half[e_of]).to(held).float() for half in (gate, lin))
        slope = (g > 0).float() if act is not None else torch.ones_like(g)
        return torch.cat([(dm * u * slope).to(dtype), (dm * (g.clamp(min=0) if act is not None else g)).to(dtype)], dim=1)
    want = halves(dm)
    assert (want != halves(dm.to(dtype).float())).float().mean() > 0.05   # (a rounded dm would show)
    assert exact or (want != halves(dm, dtype)).float().mean() > 0.05     # (and so would g and u)
    at = picked[e_of]
    assert torch.equal(got.cpu()[:, 1:], want.gather(1, at) + 0)


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("d,h", [(16384, 32768), (16, (1 << 20) + 8), (16, 1 << 20)])
def test_weights_and_rows_past_31_bits(rows, d, h):
    """An expert's W1 of 2 GiB, and more than 2^21 columns of g and u, on the 16-byte grid: the kernels for sizes off it take them.  With 2^21 the others do: a
    tile's g and u just within 2 GiB."""
    assert fmoe_native.gated_mlp_supported(torch.bfloat16, d, h)
    _check(rows, d, h, 1, torch.bfloat16, "silu", True, "even")
    torch.cuda.empty_cache()
