"""Cases for timing the fine-tuning operators: a Linear with its epilogue, counter-based dropout and the
unmerged low-rank adapter, each forward and with its gradients.

``own = False`` computes them in plain torch operations in 32 bits, rounded once at the end; ``own = True``
calls ``interior_amd.ops``. ``exact`` computes the same outputs in 64 bits from the definitions.

Sizes: token rows are images x tokens of the vision towers (50, 197 and 577 tokens) or prompts x 77 of the
text tower; widths are 512, 768 and 1024 and the four times wider hidden layers of the 512 and 1024 ones.
"""
import functools
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# the widest drawn problem costs no more than the largest listed one
_MOST = 2.0 * 36928 * 1024 * 4096 * 3


def _linear(name, m, k, n, dtype, act="none", bias=True, residual=False, p=0.0, grad=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "p": p, "grad": grad}


def _dropout(name, m, n, dtype, p, residual=False, grad=False):
    return {"name": name, "op": "dropout", "m": m, "n": n, "dtype": dtype, "p": p, "residual": residual, "grad": grad}


def _lora(name, m, k, n, r, dtype, p=0.0, grad=False):
    return {"name": name, "op": "lora", "m": m, "k": k, "n": n, "r": r, "dtype": dtype, "p": p, "grad": grad}


def listed():
    return [
        # one pooled row through a hidden layer: a single prompt answered, the call's latency
        _linear("linear-one-row", 1, 512, 2048, "fp16", "quick_gelu"),
        # one image of 50 tokens through the attention's output projection with its residual
        _linear("linear-one-image", 50, 768, 768, "fp16", residual=True),
        # the largest vision tower's hidden layer on a batch of 32 images of 577 tokens
        _linear("linear-hidden-577x32", 577 * 32, 1024, 4096, "fp16", "quick_gelu"),
        # a fine-tuning step of that tower's second MLP layer at 197 tokens: dropout on the branch, residual added
        _linear("linear-branch-step", 197 * 64, 4096, 1024, "bf16", residual=True, p=0.1, grad=True),
        # a fine-tuning step of the text tower's first MLP layer, 64 prompts
        _linear("linear-text-step", 77 * 64, 512, 2048, "bf16", "gelu", grad=True),
        # a label head with odd class and feature counts, trained
        _linear("linear-odd-step", 1237, 765, 437, "fp16", "silu", grad=True),
        # the largest training step: 64 images of 577 tokens
        _linear("linear-hidden-step", 577 * 64, 1024, 4096, "fp16", "quick_gelu", grad=True),
        # dropout of one prompt's tokens
        _dropout("dropout-one-prompt", 77, 512, "bf16", 0.1),
        # a branch of the largest tower: dropout and residual, with its gradient
        _dropout("dropout-branch-step", 577 * 64, 1024, "fp16", 0.1, residual=True, grad=True),
        # fp32 rows of an odd width
        _dropout("dropout-odd-fp32", 12611, 2049, "fp32", 0.25, grad=True),
        # an adapter served unmerged, one prompt
        _lora("lora-one-prompt", 77, 512, 2048, 4, "fp16"),
        # an adapter's training step on the largest tower (its Linear frozen)
        _lora("lora-step", 577 * 32, 1024, 4096, 16, "bf16", p=0.1, grad=True),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Layer widths are mostly multiples of 64, some of 8, a few odd ones."""
    step = rng.choice((64, 64, 64, 8, 8, 1))
    return max(1, _between(rng, low, high) // step) * step


def draw(rng):
    op = rng.choice(("linear", "linear", "dropout", "lora"))
    dtype = rng.choice(("bf16", "fp16"))
    grad = rng.random() < 0.5
    p = rng.choice((0.0, 0.1, 0.25, 0.5))
    while True:
        m, k, n = _between(rng, 1, 577 * 64), _width(rng, 64, 4096), _width(rng, 64, 4096)
        if 2.0 * m * k * n * (3 if grad else 1) <= _MOST:
            break
    if op == "dropout":
        case = _dropout("", m, n, rng.choice(("bf16", "fp16", "fp32")), p or 0.1, rng.random() < 0.5, grad)
    elif op == "lora":
        case = _lora("", m, k, n, rng.choice((4, 8, 16, 32)), dtype, p, grad)
    else:
        case = _linear("", m, k, n, dtype, rng.choice(("none", "quick_gelu", "gelu", "silu")), rng.random() < 0.8,
                       rng.random() < 0.4, rng.choice((0.0, p)), grad)
    del case["name"]
    return case


def prepare(case, seed):
    """Inputs as they reach such a layer: unit-variance rows (after a LayerNorm), weights of 1/sqrt(K)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)

    m, n, op = case["m"], case["n"], case["op"]
    s = {"case": case, "x": normal(m, n if op == "dropout" else case["k"]), "seed": 0x5DEECE66D + seed, "offset": 7 * seed + 1}
    if op != "dropout":
        s["w"] = normal(n, case["k"], scale=case["k"] ** -0.5)
    s["b"] = normal(n, scale=0.5) if op == "lora" or case.get("bias") else None
    s["r"] = normal(m, n) if case.get("residual") else None
    if op == "lora":
        s["scaling"] = 2.0
        s["A"] = normal(case["k"], case["r"], scale=case["k"] ** -0.5)
        s["B"] = normal(case["r"], n, scale=0.1)
    if case["grad"]:
        s["dy"] = normal(m, n)
        for name in ("x", "r") if op == "dropout" else ("x", "A", "B") if op == "lora" else ("x", "w", "b", "r"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain form
_LOW = 0xFFFFFFFF


def _round(state, _):
    """One round of Philox4x32 (Salmon et al., SC 2011) on 32-bit words held in int64."""
    c0, c1, c2, c3, k0, k1 = state
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    return (((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW,
            (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW)


def _keep(m, n, p, seed, offset, device):
    """keep[m, n]: word n % 4 of the counter (n // 4, m, offset), key seed, is at least p 2^32."""
    quad = torch.arange((n + 3) // 4, device=device).expand(m, -1)
    row = torch.arange(m, device=device)[:, None].expand_as(quad)
    low, high = torch.full_like(quad, offset & _LOW), torch.full_like(quad, offset >> 32)
    words = functools.reduce(_round, range(10), (quad, row, low, high, seed & _LOW, seed >> 32))[:4]
    return torch.stack(words, -1).reshape(m, -1)[:, :n] >= round(p * 2 ** 32)


def _drop(v, keep, p):
    return torch.where(keep, v / (1.0 - p), torch.zeros_like(v))


def _act(z, kind):
    """The activation's value and its derivative."""
    if kind == "none":
        return z, None
    if kind == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    beta = 1.702 if kind == "quick_gelu" else 1.0
    c = 1.0 / (1.0 + torch.exp(-beta * z))
    return z * c, c + beta * z * c * (1.0 - c)


def _plain_linear(s):
    c = s["case"]
    t, p = s["x"].dtype, c["p"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y, d = _act(z, c["act"])
    keep = _keep(c["m"], c["n"], p, s["seed"], s["offset"], x.device) if p else None
    if p:
        y = _drop(y, keep, p)
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    out = {"y": y.to(t)}
    if c["grad"]:
        dz = s["dy"].float()
        if p:
            dz = _drop(dz, keep, p)
        if d is not None:
            dz = dz * d
        out["dx"], out["dw"] = (dz @ w).to(t), (dz.t() @ x).to(t)
        if s["b"] is not None:
            out["db"] = dz.sum(0).to(t)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _plain_dropout(s):
    c = s["case"]
    x, t = s["x"].detach().float(), s["x"].dtype
    keep = _keep(c["m"], c["n"], c["p"], s["seed"], s["offset"], x.device)
    y = _drop(x, keep, c["p"])
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    out = {"y": y.to(t)}
    if c["grad"]:
        out["dx"] = _drop(s["dy"].float(), keep, c["p"]).to(t)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _plain_lora(s):
    c = s["case"]
    t, p = s["x"].dtype, c["p"]
    x, w, A, B = (s[name].detach().float() for name in ("x", "w", "A", "B"))
    keep = _keep(c["m"], c["k"], p, s["seed"], s["offset"], x.device) if p else None
    xd = _drop(x, keep, p) if p else x
    u = (xd @ A) * s["scaling"]
    out = {"y": (x @ w.t() + s["b"].float() + u @ B).to(t)}
    if c["grad"]:
        dy = s["dy"].float()
        du = (dy @ B.t()) * s["scaling"]
        dxd = du @ A.t()
        out["dx"] = (dy @ w + (_drop(dxd, keep, p) if p else dxd)).to(t)
        out["dA"], out["dB"] = (xd.t() @ du).to(t), (u.t() @ dy).to(t)
    return out


# ---------------------------------------------------------------- the framework's operators
def _ops():
    import amd_pkg
    amd_pkg.load()
    from interior_amd import ops
    return ops


def _grads(s, out, names):
    wanted = [(key, s[leaf]) for key, leaf in names if s[leaf] is not None]
    for (key, _), g in zip(wanted, torch.autograd.grad(out["y"], [leaf for _, leaf in wanted], s["dy"])):
        out[key] = g
    out["y"] = out["y"].detach()
    return out


def _own(s):
    ops, c = _ops(), s["case"]
    if c["op"] == "linear":
        out = {"y": ops.linear(s["x"], s["w"], s["b"], s["r"], activation=c["act"], dropout_p=c["p"], seed=s["seed"],
                               offset=s["offset"])}
        return _grads(s, out, (("dx", "x"), ("dw", "w"), ("db", "b"), ("dr", "r"))) if c["grad"] else out
    if c["op"] == "dropout":
        out = {"y": ops.dropout(s["x"], c["p"], seed=s["seed"], offset=s["offset"], residual=s["r"])}
        return _grads(s, out, (("dx", "x"), ("dr", "r"))) if c["grad"] else out
    out = {"y": ops.lora_linear(s["x"], s["w"], s["A"], s["B"], s["b"], scaling=s["scaling"], dropout_p=c["p"],
                                seed=s["seed"], offset=s["offset"])}
    return _grads(s, out, (("dx", "x"), ("dA", "A"), ("dB", "B"))) if c["grad"] else out


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "dropout": _plain_dropout, "lora": _plain_lora}[state["case"]["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    m, n, grad = case["m"], case["n"], case["grad"]
    res = m * n if case.get("residual") else 0
    if case["op"] == "dropout":  # x (and the residual) to y; dy to dx, the residual's gradient is dy itself
        return {"bytes": size * (2 * m * n + res + (2 * m * n if grad else 0)), "flops": (2 if grad else 1) * m * n}
    k = case["k"]
    product, bytes_ = 2 * m * n * k, m * k + n * k + m * n + res
    if case["op"] == "lora":
        r = case["r"]
        low = 2 * m * r * (k + n)
        bytes_ += k * r + r * n + n
        if grad:  # dy in; dx, dA, dB out; x again for dA
            bytes_ += m * n + 2 * m * k + n * k + 2 * (k * r + r * n)
        return {"bytes": size * bytes_, "flops": (2 * product + 3 * low) if grad else product + low}
    bytes_ += n if case["bias"] else 0
    if grad:  # dy, x, W in; dx, dW, db out
        bytes_ += m * n + 2 * m * k + 2 * n * k + (n if case["bias"] else 0)
    return {"bytes": size * bytes_, "flops": product * (3 if grad else 1)}


# ---------------------------------------------------------------- 64 bits, from the definitions
def _times(word, constant):
    """High and low halves of a 32-bit word times a 32-bit constant, from 16-bit limbs."""
    a1, a0, b1, b0 = word // 65536, word % 65536, constant // 65536, constant % 65536
    middle = a1 * b0 + (a0 * b0) // 65536
    low_middle = middle % 65536 + a0 * b1
    return a1 * b1 + middle // 65536 + low_middle // 65536, (low_middle % 65536) * 65536 + (a0 * b0) % 65536


def _kept(rows, cols, p, seed, offset):
    """The definition's mask, one column of each group of four at a time."""
    words = -(-cols // 4)
    counter = [torch.arange(words, device="cuda")[None].repeat(rows, 1), torch.arange(rows, device="cuda")[:, None].repeat(1, words),
               torch.tensor(offset % 2 ** 32, device="cuda"), torch.tensor(offset // 2 ** 32, device="cuda")]
    key = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        high0, low0 = _times(counter[0], 0xD2511F53)
        high2, low2 = _times(counter[2], 0xCD9E8D57)
        counter = [torch.bitwise_xor(torch.bitwise_xor(high2, counter[1]), key[0]), low2,
                   torch.bitwise_xor(torch.bitwise_xor(high0, counter[3]), key[1]), low0]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    kept = torch.empty(rows, 4 * words, dtype=torch.float64, device="cuda")
    for lane in range(4):
        kept[:, lane::4] = (counter[lane] >= int(p * 2 ** 32 + 0.5)).double()
    return kept[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    d = {name: v.detach().double() for name, v in s.items() if torch.is_tensor(v)}
    m, p, op = case["m"], case["p"], case["op"]
    mask = 1.0
    if p:
        mask = _kept(m, case["k"] if op == "lora" else case["n"], p, s["seed"], s["offset"]) / (1.0 - p)
    if op == "dropout":
        out = {"y": d["x"] * mask + d.get("r", 0.0)}
        if case["grad"]:
            out["dx"] = d["dy"] * mask
            if "r" in d:
                out["dr"] = d["dy"]
        return out
    if op == "lora":
        weight = d["w"].t()
        dropped = d["x"] * mask
        out = {"y": torch.addmm(d["b"], d["x"], weight) + s["scaling"] * (dropped @ d["A"] @ d["B"])}
        if case["grad"]:
            back = s["scaling"] * (d["dy"] @ d["B"].t())
            out["dx"] = d["dy"] @ d["w"] + (back @ d["A"].t()) * mask
            out["dA"] = dropped.t() @ back
            out["dB"] = s["scaling"] * ((dropped @ d["A"]).t() @ d["dy"])
        return out
    z = d["x"] @ d["w"].t() + d.get("b", 0.0)
    if case["act"] == "none":
        value, slope = z, 1.0
    elif case["act"] == "gelu":
        area = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        value, slope = z * area, area + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    else:
        beta = 1.702 if case["act"] == "quick_gelu" else 1.0
        gate = torch.sigmoid(beta * z)
        value, slope = z * gate, gate * (1.0 + beta * z * (1.0 - gate))
    out = {"y": value * mask + d.get("r", 0.0)}
    if case["grad"]:
        dz = d["dy"] * mask * slope
        out["dx"], out["dw"] = dz @ d["w"], dz.t() @ d["x"]
        if "b" in d:
            out["db"] = dz.sum(0)
        if "r" in d:
            out["dr"] = d["dy"]
    return out
