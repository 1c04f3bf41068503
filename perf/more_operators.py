"""Gated experts, trained and served, and experts served in 8-bit integers, as cases that can be timed: in the package's own
kernels (``own``) or in elementary torch operations.

``op`` of a case says which:

* ``"gated"``: the gated feed-forward block ``W2 (act(Wg x) * (Wu x))`` of each expert over its rows; a forward, or (``train``)
  a forward and a backward with the gradients of the rows, the weights and the biases.
* ``"int8"``: the experts' product of rows, rounded to 8-bit integers under a scale of their own, with weights held in 8-bit
  integers under a scale for each output channel; plain, with an activation, or (``gated``) a gate's and its linear half's
  product at once.

Rows lie sorted by expert, as the routing leaves them, ``skew`` says how unevenly (shares ``1 / rank^skew``).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
INT8_MAX = 127.0
LEAST_SCALE = 2.0 ** -126


def _gated(name, rows, d, h, experts, dtype, act, bias, train, skew=0.0):
    case = {"op": "gated", "rows": rows, "d": d, "h": h, "experts": experts, "dtype": dtype, "act": act, "bias": bias, "train": train,
            "skew": skew}
    return dict(case, name=name) if name else case


def _int8(name, rows, d, h, experts, dtype, act, gated, bias, skew=0.0):
    """``d`` features in, ``h`` out."""
    case = {"op": "int8", "rows": rows, "d": d, "h": h, "experts": experts, "dtype": dtype, "act": act, "gated": gated, "bias": bias,
            "skew": skew}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token of a text being generated, two experts of a layer of the default size
        _gated("gated-decode-1", 2, 1024, 4096, 32, "bf16", "silu", False, False),
        # a decoding step of 64 sequences through few large experts: every weight once
        _gated("gated-decode-64-large", 128, 4096, 14336, 8, "bf16", "silu", False, False, 0.5),
        # a small training step, feature sizes that are no multiple of the vector width
        _gated("gated-train-1554-odd", 1554, 500, 1302, 12, "f16", "gelu", True, True, 0.3),
        # the benchmark's float32 layer
        _gated("gated-train-8192-f32", 8192, 512, 1024, 8, "f32", "silu", True, True, 0.3),
        # many experts with skewed use
        _gated("gated-train-16384-many", 16384, 1024, 2048, 64, "bf16", "gelu", False, True, 0.6),
        # the benchmark's large layer: 16384 tokens, two experts each
        _gated("gated-train-32768-large", 32768, 4096, 14336, 8, "bf16", "silu", False, True, 0.2),
        # one token, the first product of a layer of the default size
        _int8("int8-decode-1", 2, 1024, 4096, 32, "bf16", "gelu", False, True),
        # the gate's and its linear half's product for 64 sequences through few large experts
        _int8("int8-decode-64-gated", 128, 4096, 14336, 8, "bf16", "silu", True, False, 0.5),
        # a short prompt, features that are no multiple of the vector width
        _int8("int8-prompt-1018-odd", 1018, 1302, 500, 12, "f16", "none", False, True, 0.3),
        # a prompt through experts of middle size
        _int8("int8-prompt-8192", 8192, 2048, 2048, 16, "bf16", "relu", False, True, 0.5),
        # a batch of prompts through the large experts: gated product, and the product back
        _int8("int8-prompt-32768-gated", 32768, 4096, 14336, 8, "bf16", "silu", True, False, 0.2),
        _int8("int8-prompt-32768-down", 32768, 14336, 4096, 8, "bf16", "none", False, False, 0.2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd(rng, v, step):
    """``v`` in whole steps two times of three."""
    return max(step, v // step * step) if rng.random() < 0.67 else v


def draw(rng):
    op = rng.choice(["gated", "int8"])
    while True:
        rows, experts = _log_int(rng, 1, 32768), _log_int(rng, 1, 128)
        d, h = _odd(rng, _log_int(rng, 64, 8192), 64), _odd(rng, _log_int(rng, 64, 14336), 64)
        if experts * d * h <= 400_000_000 and rows * d * h <= 400_000_000_000:
            break
    skew = rng.choice([0.0, 0.3, 0.6, 1.0])
    if op == "gated":
        return _gated("", rows, d, h, experts, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["silu", "silu", "gelu", "relu", "none"]),
                      rng.random() < 0.5, rows >= 16 and rng.random() < 0.6, skew)
    return _int8("", rows, d, h, experts, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["silu", "gelu", "relu", "none", "none"]),
                 rng.random() < 0.4, rng.random() < 0.5, skew)


def _counts(case):
    """Rows of each expert: shares ``1 / rank^skew``, ranks spread over the experts, whole rows by largest remainder."""
    n, rows = case["experts"], case["rows"]
    step = next(s for s in range(n // 2 + 1, 2 * n + 2) if math.gcd(s, n) == 1)
    share = [(i * step % n + 1.0) ** -case["skew"] for i in range(n)]
    exact = [rows * s / sum(share) for s in share]
    counts = [int(x) for x in exact]
    by_rest = sorted(range(n), key=lambda i: (counts[i] - exact[i], i))
    for i in by_rest[:rows - sum(counts)]:
        counts[i] += 1
    return counts


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows, d, h, n = case["rows"], case["d"], case["h"], case["experts"]
    counts = _counts(case)
    normal = lambda *shape: torch.randn(shape, device=dev, generator=gen)
    # normalised rows, each with a spread of its own
    x = normal(rows, d).mul_(torch.exp(0.3 * normal(rows, 1))).to(dtype)
    state = {"case": case, "x": x, "counts": counts, "table": None}
    if own:   # the segments of the rows, which the routing leaves on the device
        from fastermoe_amd import fmoe_native
        state["table"] = fmoe_native.segment_table(torch.tensor(counts, device=dev), rows)

    def uniform(*shape):   # a linear layer's weights, an expert at a time (the large ones are gigabytes)
        w = torch.empty(shape, dtype=dtype, device=dev)
        for e in range(shape[0]):
            w[e] = torch.rand(shape[1:], device=dev, generator=gen).sub_(0.5).mul_(3.4 / math.sqrt(shape[-1])).to(dtype)
        return w
    if case["op"] == "gated":
        state.update(w1=uniform(n, 2 * h, d), w2=uniform(n, d, h), b1=None, b2=None, gy=None)
        if case["bias"]:
            state.update(b1=normal(n, 2 * h).mul_(0.1).to(dtype), b2=normal(n, d).mul_(0.1).to(dtype))
        if case["train"]:
            state["gy"] = normal(rows, d).to(dtype)
            for name in ("x", "w1", "b1", "w2", "b2"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    # weights in 8 bits, each channel under its scale; rows of whole 16-byte pieces, laid out once
    out = (2 if case["gated"] else 1) * h
    held = torch.zeros(n, out, -(-d // 16) * 16, dtype=torch.int8, device=dev)
    scale = torch.empty(n, out, device=dev)
    for e in range(n):
        w = torch.randn(out, d, device=dev, generator=gen).mul_(1.0 / math.sqrt(d))
        scale[e] = w.abs().amax(dim=1) / INT8_MAX
        held[e, :, :d] = (w / scale[e][:, None]).round().to(torch.int8)
    state.update(held=held[:, :, :d], scale=scale, bias=normal(n, out).mul_(0.1).to(dtype) if case["bias"] else None)
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------

def _segments(counts):
    """(expert, first row, end) of the experts with rows."""
    at = 0
    for e, c in enumerate(counts):
        if c:
            yield e, at, at + c
        at += c


def _plain_act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return x.clamp(min=0) if act == "relu" else x


def _plain_act_grad(x, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return s * (1.0 + x * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    return (x > 0).to(x.dtype) if act == "relu" else torch.ones_like(x)


def _plain_gated(s):
    case, x, w1, w2, b1, b2, gy = (s[n] for n in ("case", "x", "w1", "w2", "b1", "b2", "gy"))
    act, h = case["act"], case["h"]
    out = {"y": torch.zeros_like(x)}
    if gy is not None:
        out.update(grad_x=torch.zeros_like(x), grad_w1=torch.zeros_like(w1), grad_w2=torch.zeros_like(w2))
        if b1 is not None:
            out.update(grad_b1=torch.zeros_like(b1), grad_b2=torch.zeros_like(b2))
    for e, lo, hi in _segments(s["counts"]):
        xe, w1e, w2e = x[lo:hi].float(), w1[e].float(), w2[e].float()
        pre = xe @ w1e.t()
        if b1 is not None:
            pre = pre + b1[e].float()
        g, u = pre[:, :h], pre[:, h:]
        a = _plain_act(g, act)
        mid = a * u
        y = mid @ w2e.t()
        if b2 is not None:
            y = y + b2[e].float()
        out["y"][lo:hi] = y.to(x.dtype)
        if gy is None:
            continue
        gye = gy[lo:hi].float()
        gmid = gye @ w2e
        gpre = torch.cat([gmid * u * _plain_act_grad(g, act), gmid * a], dim=1)
        out["grad_x"][lo:hi] = (gpre @ w1e).to(x.dtype)
        out["grad_w1"][e] = (gpre.t() @ xe).to(x.dtype)
        out["grad_w2"][e] = (gye.t() @ mid).to(x.dtype)
        if b1 is not None:
            out["grad_b1"][e] = gpre.sum(dim=0).to(x.dtype)
            out["grad_b2"][e] = gye.sum(dim=0).to(x.dtype)
    return out


def _plain_int8(s):
    case, x, held, scale, bias = (s[n] for n in ("case", "x", "held", "scale", "bias"))
    h, act = case["h"], case["act"]
    x32 = x.float()
    # (quotients next to a border between two numbers: 64 bits)
    row_scale = (x32.abs().amax(dim=1, keepdim=True).double() / INT8_MAX).float().clamp(min=LEAST_SCALE)
    q = torch.round(x32.double() / row_scale.double()).float()
    y = torch.zeros(x.shape[0], h, dtype=x.dtype, device=x.device)
    for e, lo, hi in _segments(s["counts"]):
        pre = (q[lo:hi] @ held[e].float().t()) * row_scale[lo:hi] * scale[e]
        if bias is not None:
            pre = pre + bias[e].float()
        y[lo:hi] = (_plain_act(pre[:, :h], act) * pre[:, h:] if case["gated"] else _plain_act(pre, act)).to(x.dtype)
    return {"y": y}


# ---- the package's calls ---------------------------------------------------------------------------------------------

ACTIVATIONS = {"silu": torch.nn.SiLU(), "gelu": torch.nn.GELU(), "relu": torch.nn.ReLU(), "none": None}


def _own_gated(s):
    from fastermoe_amd import functions
    x, w1, b1, w2, b2, gy = (s[n] for n in ("x", "w1", "b1", "w2", "b2", "gy"))
    with torch.set_grad_enabled(gy is not None):
        y = functions.gated_mlp(x, None, w1, b1, w2, b2, ACTIVATIONS[s["case"]["act"]], table=s["table"])
    if gy is None:
        return {"y": y}
    names = [n for n in ("x", "w1", "b1", "w2", "b2") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], gy)
    return dict({"y": y.detach()}, **{"grad_" + n: g for n, g in zip(names, grads)})


def _own_int8(s):
    from fastermoe_amd import functions
    with torch.no_grad():
        return {"y": functions.linear_int8(s["x"], None, s["held"], s["scale"], s["bias"], ACTIVATIONS[s["case"]["act"]],
                                           gated=s["case"]["gated"], table=s["table"])}


def run(state):
    gated = state["case"]["op"] == "gated"
    if own:
        return _own_gated(state) if gated else _own_int8(state)
    with torch.no_grad():
        return _plain_gated(state) if gated else _plain_int8(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _exact_act(act):
    return {"silu": torch.nn.functional.silu, "gelu": lambda t: t * torch.special.ndtr(t), "relu": torch.relu, "none": lambda t: t}[act]


def _exact_gated(case, s):
    act, h, train = _exact_act(case["act"]), case["h"], case["train"]
    zeros = lambda name: torch.zeros(s[name].shape, dtype=torch.float64, device=s[name].device)
    out = {"y": zeros("x")}
    params = [p for p in ("w1", "b1", "w2", "b2") if s[p] is not None]
    if train:
        out.update({"grad_" + p: zeros(p) for p in ["x"] + params})
    at = 0
    for e, count in enumerate(s["counts"]):
        part = slice(at, at + count)
        at += count
        if count == 0:
            continue
        leaves = {p: s[p].detach()[e].double().requires_grad_(train) for p in params}
        leaves["x"] = s["x"].detach()[part].double().requires_grad_(train)
        gate, linear = leaves["w1"].split(h)
        g, u = leaves["x"].mm(gate.t()), leaves["x"].mm(linear.t())
        if "b1" in leaves:
            bg, bu = leaves["b1"].split(h)
            g, u = g + bg, u + bu
        y = torch.mm(act(g) * u, leaves["w2"].t())
        if "b2" in leaves:
            y = y + leaves["b2"]
        out["y"][part] = y.detach()
        if train:
            names = list(leaves)
            for p, grad in zip(names, torch.autograd.grad(y, [leaves[p] for p in names], s["gy"][part].double())):
                out["grad_" + p][part if p == "x" else e] = grad
    return out


def _exact_int8(case, s):
    x, act = s["x"].double(), _exact_act(case["act"])
    # a row's scale is the float32 number next to a 127th of its largest magnitude
    step = torch.clamp((torch.linalg.vector_norm(x, ord=math.inf, dim=1) / 127).float().double(), min=2.0 ** -126)
    whole = torch.round(x / step[:, None])
    y = torch.zeros(x.shape[0], case["h"], dtype=torch.float64, device=x.device)
    at = 0
    for e, count in enumerate(s["counts"]):
        part = slice(at, at + count)
        at += count
        if count == 0:
            continue
        w = s["held"][e].double() * s["scale"][e].double()[:, None]
        pre = torch.mm(whole[part] * step[part, None], w.t())
        if s["bias"] is not None:
            pre += s["bias"][e].double()
        if case["gated"]:
            g, u = pre.split(case["h"], dim=1)
            y[part] = act(g) * u
        else:
            y[part] = act(pre)
    return {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_gated(case, s) if case["op"] == "gated" else _exact_int8(case, s)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    rows, d, h, n = case["rows"], case["d"], case["h"], case["experts"]
    live = sum(1 for c in _counts(case) if c)      # experts whose weights are needed
    if case["op"] == "gated":
        weights, biases = 3 * d * h, (2 * h + d if case["bias"] else 0)
        if not case["train"]:
            return {"bytes": size * (2 * rows * d + live * (weights + biases)), "flops": 6 * rows * d * h}
        return {"bytes": size * (4 * rows * d + (live + n) * (weights + biases)), "flops": 18 * rows * d * h}
    out = (2 if case["gated"] else 1) * h
    return {"bytes": size * rows * (d + h) + live * out * (d + 4 + (size if case["bias"] else 0)), "flops": 2 * rows * d * out}
