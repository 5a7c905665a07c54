"""The matrix product of the fine-tuning operators, tile by tile: chosen launches on integers (exact sums) and with the
whole epilogue, and the launches that the library's own rule takes at sizes of several k-tiles, which are asserted."""
import ctypes

import pytest
import torch

import finetune_ref as R
from interior_amd import _lib, ops
from test_matmul_plan import RULE, plan

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = {BF: _lib.BF16, HF: _lib.F16, F32: _lib.F32}
SEED, OFFSET = 0x123456789ABCDEF, (5 << 32) + 77


def rand(gpu, *shape, dtype=BF, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device=gpu) * scale).to(dtype)


def mask_of(gpu, rows, cols, p):
    """finetune_ref.keep_mask's mask / (1 - p), drawn on the GPU in integer arithmetic."""
    q = torch.arange((cols + 3) // 4, device=gpu).expand(rows, -1)
    m = torch.arange(rows, device=gpu)[:, None].expand_as(q)
    z = torch.zeros_like(q)
    w = R.philox((q, m, z + (OFFSET & R.U32), z + (OFFSET >> 32)), (SEED & R.U32, SEED >> 32))
    return (torch.stack(w, -1).reshape(rows, -1)[:, :cols] >= round(p * 2 ** 32)).double() / (1 - p)


def check(got, want, what):
    R.check(got, (want[0].cpu(), want[1].cpu()), what)


def linear_with(parts, x, w, b=None, r=None, activation="none", p=0.0, slope=False):
    """ops.linear's forward with chosen launches (rows, tile, slices), and the saved derivative's codes where asked for."""
    (m, k), n, L = x.shape, w.shape[0], _lib.lib()
    y = torch.full((m, n), float("nan"), dtype=x.dtype, device=x.device)
    codes = torch.empty(m, n, dtype=torch.int16, device=x.device) if slope else None
    a = _lib.LinearArgs(dtype=TYPES[x.dtype], activation=ops.ACTIVATIONS[activation], bias_dtype=TYPES[(x if b is None else b).dtype], M=m, N=n, K=k,
                        x=x.data_ptr(), x_row=x.stride(0), x_col=x.stride(1), w=w.data_ptr(), w_row=w.stride(0), w_col=w.stride(1),
                        bias=None if b is None else b.data_ptr(), residual=None if r is None else r.data_ptr(),
                        residual_stride=0 if r is None else r.stride(0), y=y.data_ptr(), y_stride=n, slope=None if codes is None else codes.data_ptr(),
                        dropout=_lib.DropoutArgs(p, SEED, OFFSET, None))
    chosen, need = (_lib.MatmulPart * len(parts))(*(_lib.MatmulPart(*q, 0) for q in parts)), ctypes.c_size_t()
    _lib.check(L.clipvit_linear_test(None, ctypes.byref(a), chosen, len(parts), None, 0, ctypes.byref(need)))
    ws = torch.empty(need.value + 256, dtype=torch.uint8, device=x.device)
    at = (ws.data_ptr() + 255) // 256 * 256
    _lib.check(L.clipvit_linear_test(torch.cuda.current_stream().cuda_stream, ctypes.byref(a), chosen, len(parts), at, need.value, None))
    torch.cuda.synchronize()
    return (y, codes) if slope else y


def decoded(codes, dtype):
    """The saved derivative that the codes stand for: sign, and fixed point in steps of 2^-14 joined by a float below."""
    bits, low = (7, -118) if dtype == BF else (9, -33)
    off, join = ((127 + low) << bits) - 1, ((bits - 14 - low) << bits) + 1
    m = codes.int() & 0x7FFF
    tail = ((m + off) << (23 - bits)).view(F32).double() * (m > 0)
    a = torch.where(m < join, tail, (m - (join - (1 << bits))).double() * 2.0 ** -14)
    return torch.where(codes < 0, -a, a)


LAYOUTS = [(True, True), (True, False), (False, True), (False, False)]


def laid_out(t, rows):
    """The same matrix, contiguous along its rows or its columns."""
    return t if rows else t.t().contiguous().t()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("ak, bk", LAYOUTS)
def test_integers_are_exact(gpu, dtype, tile, ak, bk):
    """Whole numbers up to 4: every sum is exact in fp32, so the output is the exact sum rounded once, whichever k-tile, slice
    or LDS slot a term passed through. k-tiles of 1 to 35, the last one whole, ragged or of odd length (copied first), one
    slice and several, the last of fewer k-tiles; tiles ragged in both directions."""
    for m, n in ((297, 520), (256, 264), (40, 1048)):
        x, w = (torch.randint(-4, 5, (s, 35 * 64), generator=torch.Generator(device="cuda").manual_seed(s), device=gpu).to(dtype) for s in (m, n))
        for nk in (1, 2, 3, 4, 5, 8, 9, 35):
            for cut in (0, 24, 61):
                k = nk * 64 - cut
                xs, ws = laid_out(x[:, :k].contiguous(), ak), laid_out(w[:, :k].contiguous(), bk)
                want = (xs.double() @ ws.double().t()).to(dtype)
                for slices in {1, 2, 3, 4, 7} if nk > 1 else {1}:
                    got = linear_with([(m, tile, slices)], xs, ws)
                    assert torch.equal(got, want), (m, n, k, slices)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ak, bk", LAYOUTS)
@pytest.mark.parametrize("parts", [[(512, 256, 1), (104, 64, 1)], [(256, 256, 2), (360, 128, 3)], [(512, 128, 1), (104, 256, 3)], [(256, 64, 1), (360, 64, 4)], [(616, 256, 3)]])
def test_chosen_launches_carry_the_epilogue(gpu, dtype, ak, bk, parts):
    """Bias, activation with its saved derivative, dropout and residual of two launches go by the whole operand's rows: within
    the bounds of the 64-bit restatement, the derivative within half a step and its evaluation's error."""
    m, n, p = 616, 328, 0.25
    for k in (64 * 7 - 16, 64 * 7 - 3):
        x, w = laid_out(rand(gpu, m, k, dtype=dtype), ak), laid_out(rand(gpu, n, k, dtype=dtype, scale=k ** -0.5, seed=1), bk)
        b, r = rand(gpu, n, dtype=F32, seed=2), rand(gpu, m, n + 8, dtype=dtype, seed=3)[:, :n]
        y, codes = linear_with(parts, x, w, b, r, "gelu", p, slope=True)
        check(y, R.linear(x, w, b, r, "gelu", mask_of(gpu, m, n, p))["y"], k)
        z, ez = R.product(x.double(), w.double().t())
        _, slope = R.act(z + b.double(), "gelu")
        check(decoded(codes, dtype), (slope, R.SLOPE_ABS + 1.2 * (ez + (z + b.double()).abs() * 2.0 ** -23)), "slope")


def grads(x, w, b, r, dy, **kw):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    y = ops.linear(*leaves, **kw)
    return dict(zip(("dx", "dw", "db", "dr"), torch.autograd.grad(y, leaves, dy))) | {"y": y}


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("name", ["rest in slices", "hidden layer", "ragged everywhere"])
def test_rule_at_training_sizes(gpu, name, rows):
    """Forward and gradients with the whole epilogue where the rule takes 256-wide tiles of up to 65 k-tiles, slices of unequal
    length, and rounds with remaining rows; x contiguous along either dimension."""
    m, k, n, *plans = RULE[name]
    assert [plan(m, n, k), plan(m, k, n), plan(n, k, m)] == plans
    x, w = laid_out(rand(gpu, m, k), rows), rand(gpu, n, k, scale=k ** -0.5, seed=1)
    b, r, dy = rand(gpu, n, seed=2), rand(gpu, m, n, seed=3), rand(gpu, m, n, seed=4)
    got = grads(x, w, b, r, dy, activation="quick_gelu", dropout_p=0.1, seed=SEED, offset=OFFSET)
    want = R.linear(x, w, b, r, "quick_gelu", mask_of(gpu, m, n, 0.1), dy)
    for key, g in got.items():
        check(g, want[key], key)


@pytest.mark.parametrize("name, rank", [("rest in slices", 40), ("rest in slices, back", 16), ("hidden layer", 16), ("hidden layer, back", 33)])
def test_rule_with_an_adapter(gpu, name, rank):
    """The same with the low-rank term, whose dx is masked: by the whole operand's rows in both launches and in the join."""
    m, k, n, *plans = RULE[name]
    assert [plan(m, n, k), plan(m, k, n)] == plans[:2]
    x, w, A, B, dy = rand(gpu, m, k), rand(gpu, n, k, scale=k ** -0.5, seed=1), rand(gpu, k, rank, scale=k ** -0.5, seed=2), rand(gpu, rank, n, scale=0.3, seed=3), rand(gpu, m, n, seed=4)
    leaves = [t.requires_grad_() for t in (x, A, B)]
    y = ops.lora_linear(x, w, A, B, scaling=2.0, dropout_p=0.1, seed=SEED, offset=OFFSET)
    got = dict(zip(("dx", "dA", "dB"), torch.autograd.grad(y, leaves, dy))) | {"y": y}
    want = R.lora(*(t.detach() for t in (x, w, A, B)), None, 2.0, mask_of(gpu, m, k, 0.1), dy)
    for key, g in got.items():
        check(g, want[key], key)
