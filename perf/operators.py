"""The operators around the experts that a training step of a Mixture-of-Experts block runs beside the products, as
cases that can be timed: in the package's own kernels (``own``) or in elementary torch operations.

``op`` of a case says which:

* ``"norm"``: layer norm of token rows, alone or of their sum with a residual; a forward, or (``train``) a forward and a backward.
* ``"balance"``: the gate's balance loss with the experts' counts and mean probabilities, and the gradient of the logits.
* ``"checkpoint"``: an activation over the experts' rows whose argument is kept in 8 bits, and the backward from what was kept
  (gradient of the argument, and the activation again for the next linear's weight gradient).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5
BLOCK = 32          # elements that share a scale
E4M3_MAX = 448.0


def _norm(name, rows, d, dtype, residual, train, params="same", gap=0):
    """``params`` "f32": weight and bias in float32 whatever the rows are; ``gap``: elements between the rows (rows that are a
    slice of a wider tensor)."""
    case = {"op": "norm", "rows": rows, "d": d, "dtype": dtype, "residual": residual, "train": train, "params": params, "gap": gap}
    return dict(case, name=name) if name else case


def _balance(name, tokens, experts, top_k, dtype, per, dropped=0.0, padded=0.0, skew=0.5):
    """``per`` "token" or "slot": what the loss counts in; ``dropped``: share of the slots that a capacity took away;
    ``padded``: share of the tokens that are padding; ``skew``: spread of the experts' biases."""
    case = {"op": "balance", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype, "per": per,
            "dropped": dropped, "padded": padded, "skew": skew}
    return dict(case, name=name) if name else case


def _checkpoint(name, rows, d, dtype, act):
    case = {"op": "checkpoint", "rows": rows, "d": d, "dtype": dtype, "act": act}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the norm before a layer of the default size while one token is generated
        _norm("norm-decode-1", 1, 1024, "bf16", False, False),
        # a prompt of odd length at the end of a block: residual and norm, parameters kept in float32
        _norm("norm-prompt-509", 509, 4096, "f16", True, False, "f32"),
        # training steps: the benchmark's float32 layer; odd features in rows of a wider tensor; the benchmark's large layer, with
        # the residual stream
        _norm("norm-train-4096-f32", 4096, 512, "f32", False, True),
        _norm("norm-train-777-odd", 777, 1302, "bf16", True, True, "same", 10),
        _norm("norm-train-16384", 16384, 4096, "bf16", True, True),
        # the gate of a small layer, tokens of one short batch
        _balance("balance-1000", 1000, 16, 2, "f32", "token"),
        # top-1 with a capacity, skewed use
        _balance("balance-16384-top1", 16384, 64, 1, "f32", "slot", 0.2, 0.0, 1.0),
        # many experts, a padded batch
        _balance("balance-32768-many-experts", 32768, 256, 8, "bf16", "token", 0.0, 0.15),
        # the experts' rows of a short ragged batch with odd features
        _checkpoint("checkpoint-1554-odd", 1554, 1302, "f16", "relu"),
        _checkpoint("checkpoint-8192-f32", 8192, 1024, "f32", "gelu"),
        # the large layer's rows: 16384 tokens, two experts each
        _checkpoint("checkpoint-32768-large", 32768, 14336, "bf16", "gelu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd(rng, v, step):
    """``v`` in whole steps as often as not."""
    return max(step, v // step * step) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["norm", "norm", "balance", "checkpoint"])
    if op == "norm":
        d = _odd(rng, _log_int(rng, 16, 16384), 64)
        rows = _odd(rng, _log_int(rng, 1, min(65536, 60_000_000 // d)), 16)
        return _norm("", min(rows, 60_000_000 // d), d, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.5, rng.random() < 0.7,
                     rng.choice(["same", "same", "f32"]), rng.choice([0, 0, 0, 8, 10]))
    if op == "balance":
        experts = _odd(rng, _log_int(rng, 2, 1024), 8)
        tokens = _odd(rng, _log_int(rng, 1, min(131072, 8_000_000 // experts)), 64)
        return _balance("", min(tokens, 8_000_000 // experts), experts, rng.choice([k for k in (1, 2, 4, 8) if k <= experts]),
                        rng.choice(["bf16", "f16", "f32", "f32"]), rng.choice(["token", "slot"]), rng.choice([0.0, 0.0, 0.2]),
                        rng.choice([0.0, 0.0, 0.15]), rng.choice([0.0, 0.5, 1.5]))
    d = _odd(rng, _log_int(rng, 32, 14336), 64)
    rows = _odd(rng, _log_int(rng, 1, min(65536, 400_000_000 // d)), 16)
    return _checkpoint("", min(rows, 400_000_000 // d), d, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["gelu", "gelu", "relu", "none"]))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, device=dev, generator=gen)
    if case["op"] == "norm":
        rows, d, gap = case["rows"], case["d"], case["gap"]
        # rows of a residual stream: a spread of their own each, and an offset
        stream = normal(rows, d + gap).mul_(torch.exp(0.5 * normal(rows, 1))).add_(0.3 * normal(rows, 1)).to(dtype)[:, :d]
        ptype = torch.float32 if case["params"] == "f32" else dtype
        state = {"case": case, "x": stream, "r": None, "ds": None, "dy": None,
                 "w": (1.0 + 0.2 * normal(d)).to(ptype), "b": (0.1 * normal(d)).to(ptype)}
        if case["residual"]:
            state["r"] = normal(rows, d).to(dtype)
        if case["train"]:
            state["dy"] = normal(rows, d).to(dtype)
            if case["residual"]:
                state["ds"] = normal(rows, d).to(dtype)
            for name in ("x", "r", "w", "b"):
                if state[name] is not None:
                    state[name] = state[name].detach().requires_grad_(True)
        return state
    if case["op"] == "balance":
        n, e, k = case["tokens"], case["experts"], case["top_k"]
        logits = (normal(n, e) + case["skew"] * normal(e)).to(dtype)
        idx = logits.float().topk(k, dim=1).indices
        if case["dropped"]:
            idx = idx.masked_fill(torch.rand(n, k, device=dev, generator=gen) < case["dropped"], -1)
        mask = None
        if case["padded"]:   # sequences of a batch, padded to one length
            length = max(1, min(512, n))
            real = (length * (1.0 - 2.0 * case["padded"] * torch.rand(-(-n // length), device=dev, generator=gen))).round()
            mask = (torch.arange(length, device=dev)[None, :] >= real.clamp(min=1)[:, None]).reshape(-1)[:n]
        # the loss enters with a small weight; a float16 step scales its losses up
        weight = torch.tensor(0.01 * (65536.0 if dtype == torch.float16 else 1.0), device=dev)
        return {"case": case, "logits": logits.requires_grad_(True), "idx": idx, "mask": mask, "weight": weight}
    # pre-activations: an expert's bias in each feature, a spread of its own for each row
    rows, d = case["rows"], case["d"]
    x = normal(rows, d).mul_(torch.exp(0.3 * normal(rows, 1))).add_(0.2 * normal(1, d)).to(dtype)
    return {"case": case, "x": x, "g": normal(rows, d).to(dtype)}


# ---- plain forms ------------------------------------------------------------------------------------------------

def _plain_norm(s):
    x, r, w, b, dy, ds = (s[n] for n in ("x", "r", "w", "b", "dy", "ds"))
    total = x if r is None else (x.float() + r.float()).to(x.dtype)
    t = total.float()
    centred = t - t.mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    hat = centred * rstd
    out = {"y": (hat * w.float() + b.float()).to(x.dtype)}
    if r is not None:
        out["sum"] = total
    if dy is not None:
        g = dy.float()
        gw = g * w.float()
        gx = rstd * (gw - gw.mean(dim=1, keepdim=True) - hat * (gw * hat).mean(dim=1, keepdim=True))
        if ds is not None:
            gx = gx + ds.float()
        out.update(grad_x=gx.to(x.dtype), grad_w=(g * hat).sum(dim=0).to(w.dtype), grad_b=g.sum(dim=0).to(b.dtype))
        if r is not None:
            out["grad_r"] = out["grad_x"].clone()
    return out


def _plain_balance(s):
    case, logits, idx, mask, weight = (s[n] for n in ("case", "logits", "idx", "mask", "weight"))
    n, e = logits.shape
    l32 = logits.float()
    ex = torch.exp(l32 - l32.max(dim=1, keepdim=True).values)
    p = ex / ex.sum(dim=1, keepdim=True)
    if mask is not None:
        keep = ~mask
        idx = torch.where(keep[:, None], idx, -1)
        p = p * keep[:, None]
        tokens = keep.sum()
    else:
        tokens = torch.tensor(n, device=logits.device)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=logits.device).index_add_(
        0, idx.reshape(-1) + 1, torch.ones_like(idx).reshape(-1))[1:]
    slots = counts.sum()
    # (sums over many tokens, and counts less their mean: 64 bits)
    total = p.double().sum(dim=0)
    per = (tokens if case["per"] == "token" else slots).clamp(min=1).double()
    loss = (counts * total).sum() * e / (per * per)
    u = ((counts - slots.double() / e) * (weight.double() * e / (per * per))).float()
    grad = p * (u - (p * u).sum(dim=1, keepdim=True))
    return {"loss": loss.float(), "counts": counts, "prob": (total / tokens.clamp(min=1)).float(), "grad": grad.to(logits.dtype)}


def _plain_act(x, act):
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return x.clamp(min=0) if act == "relu" else x


def _plain_act_grad(x, act):
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    return (x > 0).to(x.dtype) if act == "relu" else torch.ones_like(x)


def _blocks(x):
    """``x [rows, d]`` as blocks, zeros after the row's end."""
    pad = -x.shape[1] % BLOCK
    return torch.nn.functional.pad(x, (0, pad)).reshape(x.shape[0], -1, BLOCK)


def _plain_checkpoint(s):
    case, x, g = s["case"], s["x"], s["g"]
    x32 = x.float()
    y = _plain_act(x32, case["act"])
    blocks = _blocks(x32)
    most, exponent = torch.frexp(blocks.abs().amax(dim=2, keepdim=True))   # most in [0.5, 1): 448 = 0.875 * 2^9
    exponent = (exponent - 9 + (most > E4M3_MAX / 512).to(exponent.dtype)).clamp(min=-126)
    power = ((exponent + 127) << 23).view(torch.float32)    # 2^exponent, exactly
    held = (blocks / power).to(torch.float8_e4m3fn)
    kept = (held.float() * power).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return {"y": y.to(x.dtype), "grad": (g.float() * _plain_act_grad(kept, case["act"])).to(x.dtype),
            "mid": _plain_act(kept, case["act"]).to(x.dtype)}


# ---- the package's calls ---------------------------------------------------------------------------------------------

def _own_norm(s):
    from fastermoe_amd import functions
    x, r, w, b = (s[n] for n in ("x", "r", "w", "b"))
    with torch.set_grad_enabled(s["dy"] is not None):
        if r is None:
            y = functions.layer_norm(x, w, b, EPS)
            out, outs, ins, gs = {"y": y}, [y], [x, w, b], [s["dy"]]
        else:
            y, total = functions.add_layer_norm(x, r, w, b, EPS)
            out, outs, ins, gs = {"y": y, "sum": total}, [y, total], [x, w, b, r], [s["dy"], s["ds"]]
    if s["dy"] is None:
        return out
    grads = torch.autograd.grad(outs, ins, gs)
    out = {name: t.detach() for name, t in out.items()}
    out.update(zip(("grad_x", "grad_w", "grad_b", "grad_r"), grads))
    return out


def _own_balance(s):
    from fastermoe_amd import functions
    loss, counts, prob = functions.balance_loss(s["logits"], s["idx"], per=s["case"]["per"], mask=s["mask"])
    grad, = torch.autograd.grad(loss, s["logits"], s["weight"])
    return {"loss": loss.detach(), "counts": counts, "prob": prob.detach(), "grad": grad}


def _own_checkpoint(s):
    from fastermoe_amd import fmoe_native
    act = {"none": 0, "relu": 1, "gelu": 2}[s["case"]["act"]]
    y, held, scale = fmoe_native.act_checkpoint_forward(s["x"], act)
    grad, mid = fmoe_native.act_checkpoint_backward(s["g"], held, scale, act)
    return {"y": y, "grad": grad, "mid": mid}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "balance": _own_balance, "checkpoint": _own_checkpoint}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "balance": _plain_balance, "checkpoint": _plain_checkpoint}[op](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _exact_norm(case, s):
    dtype = DTYPES[case["dtype"]]
    v, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
    if s["r"] is not None:
        v = (v + s["r"].detach().double()).to(dtype).double()   # what is normalised is the sum as its type holds it
    var, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
    sigma = (var + EPS).sqrt()
    z = (v - mean) / sigma
    out = {"y": torch.addcmul(b, z, w)}
    if s["r"] is not None:
        out["sum"] = v
    if case["train"]:
        dy = s["dy"].double()
        a = dy * w
        # the projection of the gradient that neither shifts nor stretches the row
        gx = (a - a.mean(1, keepdim=True) - z * (a * z).mean(1, keepdim=True)) / sigma
        if s["ds"] is not None:
            gx = gx + s["ds"].double()
        out.update(grad_x=gx, grad_w=torch.einsum("rd,rd->d", dy, z), grad_b=dy.sum(0))
        if s["r"] is not None:
            out["grad_r"] = gx
    return out


def _exact_balance(case, s):
    logits = s["logits"].detach().double().requires_grad_(True)
    n, e = logits.shape
    keep = torch.ones(n, dtype=torch.bool, device=logits.device) if s["mask"] is None else ~s["mask"]
    named = s["idx"][keep].reshape(-1)
    counts = torch.bincount(named[named >= 0], minlength=e)
    prob = torch.softmax(logits[keep], dim=1).sum(0)
    tokens, slots = int(keep.sum()), int(counts.sum())
    per = max(1, tokens if case["per"] == "token" else slots)
    loss = e * torch.dot(counts.double() / per, prob / per)
    # the gradient does not feel a constant added to every count: without their mean, nothing large cancels
    centred = e * torch.dot((counts.double() - slots / e) / per, prob / per)
    grad, = torch.autograd.grad(centred, logits, s["weight"].double())
    return {"loss": loss.detach(), "counts": counts, "prob": prob.detach() / max(1, tokens), "grad": grad}


def _exact_checkpoint(case, s):
    x, g = s["x"].double(), s["g"].double()
    d = x.shape[1]
    blocks = torch.cat([x, x.new_zeros(x.shape[0], -d % BLOCK)], dim=1).view(x.shape[0], -1, BLOCK)
    top = blocks.abs().amax(2, keepdim=True).clamp(min=2.0 ** -126 * E4M3_MAX)
    scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
    scale = torch.where(scale * E4M3_MAX < top, 2 * scale, scale)            # (where the logarithm was rounded over a whole number)
    scale = torch.where(scale * (E4M3_MAX / 2) >= top, scale / 2, scale).clamp(min=2.0 ** -126)
    v = blocks / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)   # three bits after the first; 2^-9 below 2^-6
    kept = (torch.round(v / step) * step * scale).reshape(x.shape[0], -1)[:, :d]
    del blocks, v, step
    if case["act"] == "gelu":
        act = lambda t: t * torch.special.ndtr(t)
        slope = torch.special.ndtr(kept) + kept * torch.exp(-kept.square() / 2) / math.sqrt(2 * math.pi)
    elif case["act"] == "relu":
        act, slope = torch.relu, torch.heaviside(kept, torch.zeros((), dtype=kept.dtype, device=kept.device))
    else:
        act, slope = (lambda t: t), 1.0
    return {"y": act(x), "grad": g * slope, "mid": act(kept)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "balance": _exact_balance, "checkpoint": _exact_checkpoint}[case["op"]](case, s)


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n, d = case["rows"], case["d"]
        psize = 4 if case["params"] == "f32" else size
        tensors = 2 + (2 if case["residual"] else 0)            # rows in and out
        if case["train"]:
            tensors += 2 + (1 if case["residual"] else 0)       # gradients in and out
        return {"bytes": n * d * size * tensors + d * psize * (4 if case["train"] else 2), "flops": n * d * (20 if case["train"] else 8)}
    if case["op"] == "balance":
        n, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": 2 * n * e * size + 8 * n * k + (n if case["padded"] else 0) + 12 * e, "flops": 12 * n * e}
    n, d = case["rows"], case["d"]
    return {"bytes": n * d * (5 * size + 1) + n * -(-d // BLOCK), "flops": 40 * n * d}
