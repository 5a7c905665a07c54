"""Plain 64-bit restatement of the fine-tuning operators (interior_amd.ops) with elementwise error bounds.

Every bound is arithmetic, fixed before any run: a rounding to type t costs at most eps(t) / 2 of the value
(plus half its smallest subnormal), an fp32 sum of K products in any order at most (K + 8) 2^-24 of the sum of
magnitudes (each product of two 16-bit values is exact in fp32), the activations' fp32 evaluation ACT_REL of
their value plus ACT_ABS per unit of |z| (erff, v_exp_f32 and v_rcp_f32 are within a few 2^-23), and the saved
derivative half of its 2^-14 step.
"""
import math

import torch

U32 = 0xFFFFFFFF
ACT_REL, ACT_ABS, SLOPE_ABS = 2.0 ** -20, 2.0 ** -21, 2.0 ** -15 + 2.0 ** -19


def philox(c, k, rounds=10):
    """Philox4x32 on int64 tensors (or ints) of 32-bit words."""
    c0, c1, c2, c3 = c
    k0, k1 = k
    for _ in range(rounds):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & U32) ^ c1 ^ k0, b & U32, ((a >> 32) & U32) ^ c3 ^ k1, a & U32
        k0, k1 = (k0 + 0x9E3779B9) & U32, (k1 + 0xBB67AE85) & U32
    return c0, c1, c2, c3


def keep_mask(rows, cols, p, seed, offset):
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    q = torch.arange((cols + 3) // 4).expand(rows, -1)
    m = torch.arange(rows)[:, None].expand_as(q)
    z = torch.zeros_like(q)
    w = philox((q, m, z + (offset & U32), z + (offset >> 32)), (seed & U32, seed >> 32))
    return torch.stack(w, -1).reshape(rows, -1)[:, :cols] >= round(p * 2 ** 32)


def half_step(t, dtype):
    """Largest error of rounding values of this magnitude to dtype."""
    return t.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act(z, kind):
    """(value, derivative) in 64 bits."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp_min(0), (z > 0).double()
    if kind == "gelu":
        c = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    b = 1.702 if kind == "quick_gelu" else 1.0
    s = torch.sigmoid(b * z)
    return z * s, s * (1 + b * z * (1 - s))


def product(a, b, da=0.0, db=0.0):
    """a @ b in 64 bits and the bound of its fp32 evaluation, with operands off by at most da, db."""
    k = a.shape[1]
    aa, ab = a.abs() + da, b.abs() + db
    err = (k + 8) * 2.0 ** -24 * (aa @ ab)
    if torch.is_tensor(da):
        err = err + da @ ab
    if torch.is_tensor(db):
        err = err + aa @ db
    return a @ b, err


def linear(x, w, b=None, r=None, kind="none", mask=None, dy=None):
    """Value and gradients of residual + mask * act(x w^T + b) as {name: (value, bound)}; mask holds 0 or
    1 / (1 - p). Inputs are the 16-bit tensors on the CPU; outputs are rounded to their type."""
    t = x.dtype
    X, W = x.double(), w.double()
    z, ez = product(X, W.t())
    if b is not None:
        z = z + b.double()
        ez = ez + z.abs() * 2.0 ** -23
    v, s = act(z, kind)
    ev = 1.2 * ez + (0 if kind == "none" else ACT_REL * v.abs() + ACT_ABS * z.abs().clamp_max(8))
    if mask is not None:
        v, ev = v * mask, ev * mask + (v * mask).abs() * 2.0 ** -23
    if r is not None:
        v = v + r.double()
        ev = ev + v.abs() * 2.0 ** -23
    out = {"y": (v, ev + half_step(v.abs() + ev, t))}
    if dy is None:
        return out
    g = dy.double()
    if mask is not None:
        g = g * mask
    dz = g * s
    changed = kind != "none" or mask is not None
    # |act''| <= 1.2 for all of these; relu's derivative jumps at 0, where its tests keep z away
    eg = g.abs() * ((SLOPE_ABS + (0 if kind == "relu" else 1.2) * ez) if kind != "none" else 0) + dz.abs() * 2.0 ** -22
    ed = eg + half_step(dz.abs() + eg, t) if changed else torch.zeros_like(dz)
    for name, (val, err) in (("dx", product(dz, W, ed)), ("dw", product(dz.t().contiguous(), X, ed.t().contiguous()))):
        out[name] = (val, err + half_step(val.abs() + err, t))
    if b is not None:
        val = dz.sum(0)
        err = eg.sum(0) + (dz.shape[0] + 8) * 2.0 ** -24 * dz.abs().sum(0)
        out["db"] = (val, err + half_step(val.abs() + err, b.dtype))
    if r is not None:
        out["dr"] = (dy.double(), torch.zeros_like(g))
    return out


def lora(x, w, A, B, b=None, scaling=1.0, mask=None, dy=None):
    """The same for x w^T + b + scaling (mask * x) A B; the thin products are rounded to the type once."""
    t = x.dtype
    X, W, a, bb = x.double(), w.double(), A.double(), B.double()
    xd = X if mask is None else X * mask
    base, eb = product(X, W.t())
    u, eu = product(xd, a)
    u, eu = u * scaling, eu * abs(scaling)
    eu = eu + u.abs() * 2.0 ** -22
    eu = eu + half_step(u.abs() + eu, t)
    low, el = product(u, bb, eu)
    y = base + low + (0 if b is None else b.double())
    err = eb + el + y.abs() * 2.0 ** -22 + (base.abs() + low.abs()) * 2.0 ** -23
    out = {"y": (y, err + half_step(y.abs() + err, t))}
    if dy is None:
        return out
    g = dy.double()
    du, ed = product(g, bb.t().contiguous())
    du, ed = du * scaling, ed * abs(scaling)
    # the kernels carry 1 / (1 - p) in the rounded thin product, so the mask itself is exact
    keep = torch.ones_like(X) if mask is None else (mask != 0).double()
    c = 1.0 if mask is None else float(mask.max().clamp_min(0))
    du, ed = du * c, ed * c
    ed = ed + du.abs() * 2.0 ** -22
    ed = ed + half_step(du.abs() + ed, t)
    main, em = product(g, W)
    low, el = product(du, a.t().contiguous(), ed)
    val, err = main + keep * low, em + keep * el + (main.abs() + low.abs()) * 2.0 ** -23
    out["dx"] = (val, err + half_step(val.abs() + err, t))
    val, err = product((keep * X).t().contiguous(), du, 0.0, ed)
    out["dA"] = (val, err + half_step(val.abs() + err, t))
    val, err = product(u.t().contiguous(), g, eu.t().contiguous())
    out["dB"] = (val, err + half_step(val.abs() + err, t))
    val, err = product(g.t().contiguous(), X)
    out["dw"] = (val, err + half_step(val.abs() + err, t))
    if b is not None:
        val = g.sum(0)
        err = (g.shape[0] + 8) * 2.0 ** -24 * g.abs().sum(0)
        out["db"] = (val, err + half_step(val.abs() + err, b.dtype))
    return out


def check(got, want, what=""):
    """Every element of a device or CPU tensor within its bound."""
    val, err = want
    d = (got.detach().double().cpu() - val).abs()
    assert got.shape == val.shape, (what, got.shape, val.shape)
    bad = ~(d <= err)
    assert not bool(bad.any()), (what, "off at", bad.nonzero()[:4].tolist(), "worst ratio",
                                 float((d / err.clamp_min(1e-300)).nan_to_num(float("inf")).max()))
