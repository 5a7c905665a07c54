"""Gradients of the activations where their derivative is small: the saved derivative keeps its relative precision there.

With an identity as weight and ones as dy, dz = act'(z) and dx, dw and db are read off it. Bounds, relative to the true
derivative: its saved code is half a step of its type's format (bf16 2^-8, fp16 2^-10), dz and each output are rounded once
more (eps / 2 each), and the fp32 evaluation is off by at most 2^-13 of the value (gelu's polynomial 2^-13.4; the exponent
of an exponential, at most 128, in three roundings: 128 * 3 * 2^-24 * ln 2 = 2^-15.9). Below 2^-118 (bf16) the code, and the
exponentials' 2^-126, end in zero; fp16 ends at half its smallest subnormal, 2^-25."""
import math

import pytest
import torch

import finetune_ref as R
from interior_amd import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {BF: 2.0 ** -8, HF: 2.0 ** -10}
FLOOR = {BF: 2.0 ** -117, HF: 2.0 ** -25}
EVAL = 2.0 ** -13
KINDS = ("quick_gelu", "silu", "gelu", "gelu_tanh")


def phi(z):
    """Phi(z) and its density in 64 bits; erfc keeps its relative precision."""
    return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def value_and_slope(z, kind):
    """act(z) and act'(z) in 64 bits without cancellation for negative z."""
    if kind == "gelu":
        c, d = phi(z)
        return z * c, c + z * d
    if kind == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        t, dt = a * (z + 0.044715 * z ** 3), a * (1 + 3 * 0.044715 * z * z)
    else:
        b = 1.702 if kind == "quick_gelu" else 1.0
        t, dt = b * z, torch.full_like(z, b)
    s, one_minus = torch.sigmoid(t), torch.sigmoid(-t)
    return z * s, s + z * s * one_minus * dt


def grads(gpu, z, kind, dy):
    x, w, b = z.to(gpu).requires_grad_(), torch.eye(8, dtype=z.dtype, device=gpu).requires_grad_(), torch.zeros(8, device=gpu, requires_grad=True)
    y = ops.linear(x, w, b, activation=kind)
    return y, *torch.autograd.grad(y, (x, w, b), dy.to(gpu))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", KINDS)
def test_tail_gradients_are_relative(gpu, dtype, kind):
    z = torch.linspace(-12, -3, 8 * 500).view(500, 8).to(dtype)
    val, slope = value_and_slope(z.double(), kind)
    half = torch.finfo(dtype).eps / 2
    y, dx, dw, db = grads(gpu, z, kind, torch.ones_like(z))
    R.check(y, (val, val.abs() * (EVAL + half) + FLOOR[dtype]), "y")
    rel = CODE[dtype] + EVAL + half
    R.check(dx, (slope, slope.abs() * rel + FLOOR[dtype]), "dx")
    # every term of these sums has the same sign: dw = dz^T z, db = sum of the unrounded dz
    val = slope.t() @ z.double()
    R.check(dw, (val, val.abs() * (rel + half + 510 * 2.0 ** -24) + (FLOOR[dtype] * z.double().abs()).sum(0) + FLOOR[dtype]), "dw")
    val = slope.sum(0)
    R.check(db, (val, val.abs() * (CODE[dtype] + EVAL + 510 * 2.0 ** -24) + 500 * FLOOR[dtype]), "db")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", KINDS)
def test_gradients_over_the_whole_range(gpu, dtype, kind):
    """Every z in [-14, 14]: off by at most 2^-15 of the saved derivative (its steps of 2^-14 near 1), 2^-19 of its
    evaluation and the rounding of dz, whatever the sign of the derivative; relative where it is below 2^-5."""
    z = torch.linspace(-14, 14, 8 * 2000).view(2000, 8).to(dtype)
    _, slope = value_and_slope(z.double(), kind)
    _, dx, _, _ = grads(gpu, z, kind, torch.ones_like(z))
    err = torch.minimum(torch.full_like(slope, 2.0 ** -15), slope.abs() * CODE[dtype]) + 2.0 ** -19
    R.check(dx, (slope, err + R.half_step(slope.abs() + err, dtype)))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_exact_slopes_and_nan(gpu, dtype):
    """0 and 1 are exact (relu, the limits of the others), NaN stays NaN, and a zero slope gives a zero."""
    z = torch.tensor([[-1e4, -3.0, -0.0, 0.0, 2.0, 300.0, 1e4, float("nan")]], dtype=dtype)
    for kind in ("relu", *KINDS):
        _, dx, _, _ = grads(gpu, z[:, :7].contiguous().repeat(1, 2)[:, :8], kind, torch.ones(1, 8, dtype=dtype))
        dx = dx.cpu()[0]
        assert dx[0] == 0 and dx[5] == 1 and dx[6] == 1, kind
        if kind == "relu":
            assert dx[:7].tolist() == [0, 0, 0, 0, 1, 1, 1]
    x = z[:, 7:].to(gpu).requires_grad_()
    for kind in ("relu", *KINDS):
        y = ops.linear(x, torch.ones(1, 1, dtype=dtype, device=gpu), activation=kind)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert bool(dx.isnan().all()), kind
