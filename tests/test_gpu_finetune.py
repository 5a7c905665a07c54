"""Fine-tuning operators on the GPU against the 64-bit restatement of tests/finetune_ref.py, elementwise within its
arithmetic bounds: every layout and tile path, odd and ragged sizes, views, empty sizes, masks, streams, graphs."""
import pytest
import torch

import finetune_ref as R
from interior_amd import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
SEED, OFFSET = 0x123456789ABCDEF, (5 << 32) + 77


def rand(*shape, dtype=BF, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(hash((shape, seed)) & 0x7FFFFFFF)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def mask_of(rows, cols, p, seed=SEED, offset=OFFSET):
    if p == 0:
        return None
    keep = R.keep_mask(rows, cols, p, seed, offset).double()
    return keep / (1 - p) if p < 1 else keep * 0


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 4), (3, 5), (77, 512), (130, 1021), (1000, 33), (5, 4099), (2100, 8)])
def test_dropout_mask_is_the_definition(gpu, dtype, rows, cols):
    p = 0.37
    y = ops.dropout(torch.ones(rows, cols, dtype=dtype, device=gpu), p, seed=SEED, offset=OFFSET)
    keep = R.keep_mask(rows, cols, p, SEED, OFFSET)
    one = torch.tensor(1 / (1 - p), dtype=F32).to(dtype)
    assert torch.equal(y.cpu(), torch.where(keep, one, torch.zeros((), dtype=dtype)))


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("p", [0.0, 2.0 ** -33, 0.25, 1 - 2.0 ** -33, 1.0])
def test_dropout_residual_and_gradient(gpu, dtype, p):
    x, r, dy = (rand(61, 203, dtype=dtype, seed=i) for i in range(3))
    xd, rd = x.to(gpu).requires_grad_(), r.to(gpu).requires_grad_()
    y = ops.dropout(xd, p, seed=SEED, offset=OFFSET, residual=rd)
    dx, dr = torch.autograd.grad(y, (xd, rd), dy.to(gpu))
    mask = torch.ones(61, 203).double() if p < 2.0 ** -32 else mask_of(61, 203, p)
    # y = fl(r + fl(x scale)): each fp32 rounding is at most 2^-24 of its result, the scale's own 2^-24 of x scale, and
    # |r + x scale| <= |r| + |x scale|, so 2^-24 (3 |x scale| + |r|) in all, whatever cancels in the sum
    for got, val, size in ((y, r.double() + mask * x.double(), r.double().abs() + (mask * x.double()).abs()),
                           (dx, mask * dy.double(), (mask * dy.double()).abs())):
        err = size * 2.0 ** -22
        R.check(got, (val, err + R.half_step(val.abs() + err, dtype)))
    assert torch.equal(dr.cpu(), dy)


def test_dropout_views_and_poison(gpu):
    """Column slices, expanded and transposed views, leading dimensions; NaN and inf in dropped places give 0."""
    big = rand(64, 96, dtype=HF).to(gpu)
    for v in (big[:, 3:50], big[::2, 8:72], big.t(), big[5:6].expand(40, 96), big.view(4, 16, 96)):
        y = ops.dropout(v, 0.5, seed=SEED, offset=OFFSET)
        rows = v.numel() // v.shape[-1]
        want = v.double().cpu().reshape(rows, -1) * mask_of(rows, v.shape[-1], 0.5)
        assert torch.equal(y.double().cpu().reshape(rows, -1), want)  # scale 2: exact
    x = torch.full((33, 40), float("nan"), device=gpu)
    x[:, ::2] = float("inf")
    keep = R.keep_mask(33, 40, 0.5, SEED, OFFSET)
    y = ops.dropout(x, 0.5, seed=SEED, offset=OFFSET).cpu()
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())
    assert ops.dropout(big[:0], 0.5, seed=1).shape == (0, 96) and ops.dropout(big[:, :0], 0.5, seed=1).shape == (64, 0)


def test_dropout_row_counter_past_16_bits(gpu):
    """Many short rows: every row draws its own counter (rows 65536 apart differ)."""
    y = ops.dropout(torch.ones(140000, 4, device=gpu), 0.5, seed=SEED, offset=OFFSET).cpu()
    assert torch.equal(y != 0, R.keep_mask(140000, 4, 0.5, SEED, OFFSET))


# ---------------------------------------------------------------- linear, forward
# (M, K, N): one row, fewer rows than a tile, ragged in each dimension, odd, and each tile size of the launch rule
SHAPES = [(1, 1, 1), (1, 512, 512), (2, 64, 130), (7, 33, 9), (16, 8, 16), (50, 768, 768), (65, 40, 100), (77, 512, 2048),
          (129, 96, 257), (300, 765, 437), (1024, 64, 1024), (1300, 72, 1500), (2049, 100, 2056), (4100, 48, 2304), (3000, 33, 3001)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m, k, n", SHAPES)
def test_linear_shapes(gpu, dtype, m, k, n):
    x, w, b = rand(m, k, dtype=dtype), rand(n, k, dtype=dtype, scale=k ** -0.5, seed=1), rand(n, dtype=dtype, seed=2)
    y = ops.linear(x.to(gpu), w.to(gpu), b.to(gpu), activation="quick_gelu")
    R.check(y, R.linear(x, w, b, kind="quick_gelu")["y"], (m, k, n))


@pytest.mark.parametrize("kind", ["none", "quick_gelu", "gelu", "gelu_tanh", "silu", "relu"])
def test_linear_activations(gpu, kind):
    x, w = rand(65, 96, dtype=HF, scale=2.0), rand(70, 96, dtype=HF, scale=0.2, seed=1)
    y = ops.linear(x.to(gpu), w.to(gpu), activation=kind)
    R.check(y, R.linear(x, w, kind=kind)["y"])
    # the activations' limits
    e = torch.eye(8, dtype=BF, device=gpu)
    z = torch.tensor([[-3e4, -100.0, -20.0, -0.0, 0.0, 20.0, 100.0, 3e4]], dtype=BF, device=gpu)
    y = ops.linear(z, e, activation=kind)
    want = z.clone() if kind == "none" else z.clamp_min(0)
    assert torch.allclose(y.float(), want.float(), atol=3e-8 * 20, rtol=0)
    z = torch.tensor([[float("nan")] + [1.0] * 7], dtype=BF, device=gpu)
    assert bool(torch.isnan(ops.linear(z, e[:1].contiguous(), activation=kind)).all())


@pytest.mark.parametrize("m, k, n", [(33, 64, 48), (300, 130, 333), (2100, 64, 2048)])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_linear_epilogue(gpu, m, k, n, p):
    x, w, r = rand(m, k), rand(n, k, scale=k ** -0.5, seed=1), rand(m, n, seed=3)
    for b in (None, rand(n, dtype=F32, seed=2)):
        y = ops.linear(x.to(gpu), w.to(gpu), None if b is None else b.to(gpu), r.to(gpu), activation="gelu", dropout_p=p,
                       seed=SEED, offset=OFFSET)
        R.check(y, R.linear(x, w, b, r, "gelu", mask_of(m, n, p))["y"])


def test_linear_mask_is_dropouts(gpu):
    """The fused mask is the mask of ops.dropout on the [rows, N] output."""
    x, w = rand(131, 64).to(gpu), rand(517, 64, seed=1).to(gpu)
    a = ops.linear(x, w, dropout_p=0.5, seed=SEED, offset=OFFSET)
    b = ops.dropout(ops.linear(x, w), 0.5, seed=SEED, offset=OFFSET)
    assert torch.equal(a, b)


@pytest.mark.parametrize("m, k, n", [(40, 64, 72), (300, 96, 264), (2300, 64, 2048)])
def test_linear_views(gpu, m, k, n):
    """Transposed, sliced, misaligned and expanded operands, residual and leading dimensions."""
    bx, bw = rand(m + 3, k + 16).to(gpu), rand(n + 5, k + 24, scale=k ** -0.5, seed=1).to(gpu)
    xt, wt = rand(k, m, seed=2).to(gpu), rand(k, n, scale=k ** -0.5, seed=3).to(gpu)
    res = rand(m, n + 8, seed=4).to(gpu)
    xs = [bx[:m, :k], bx[3:, 8:k + 8], bx[1:m + 1, 5:k + 5], xt.t(), bx[:1, :k].expand(m, k)]
    ws = [bw[:n, :k], bw[2:n + 2, 3:k + 3], wt.t(), bw[:n, 8:k + 8]]
    for i, x in enumerate(xs):
        for j, w in enumerate(ws):
            r = res[:, :n] if (i + j) % 2 else res[:, 3:n + 3]
            y = ops.linear(x, w, None, r)
            R.check(y, R.linear(x.cpu(), w.cpu(), None, r.cpu())["y"], (i, j))
    x3 = bx[:m, :k].contiguous().view(2, m // 2, k)
    y = ops.linear(x3, ws[0])
    assert y.shape == (2, m // 2, n)
    R.check(y.view(m, n), R.linear(x3.cpu().view(m, k), ws[0].cpu())["y"])
    R.check(ops.linear(x3[0, 0], ws[0]).view(1, n), R.linear(x3[0, 0].cpu().view(1, k), ws[0].cpu())["y"])


def test_linear_nan_and_inf_stay_in_their_row(gpu):
    """A poisoned row of x and poisoned memory around a view reach no other row, whatever the tile's padding reads."""
    big = torch.full((300, 160), float("nan"), dtype=BF, device=gpu)
    x = big[7:206, 16:112]
    x.copy_(rand(199, 96))
    w = rand(150, 96, scale=0.1, seed=1)
    want = R.linear(x.cpu(), w)["y"]
    R.check(ops.linear(x, w.to(gpu)), want)
    x[11, 5] = float("inf")
    y = ops.linear(x, w.to(gpu)).cpu()
    rows = [i for i in range(199) if i != 11]
    R.check(y[rows], (want[0][rows], want[1][rows]))
    assert not bool(torch.isfinite(y[11]).any())
    # the same on the transposed layouts (k past the matrix is another row's data)
    xt = big[7:40, 16:112]
    xt.copy_(rand(33, 96, seed=9))
    wt = rand(33, 72, scale=0.1, seed=2)
    R.check(ops.linear(xt.t(), wt.to(gpu).t()), R.linear(xt.cpu().t(), wt.t())["y"])


def test_linear_empty(gpu):
    w, b = rand(5, 8).to(gpu), rand(5, seed=1).to(gpu)
    assert ops.linear(torch.empty(0, 8, dtype=BF, device=gpu), w).shape == (0, 5)
    assert ops.linear(torch.empty(3, 0, 8, dtype=BF, device=gpu), w).shape == (3, 0, 5)
    y = ops.linear(torch.empty(4, 0, dtype=BF, device=gpu), torch.empty(5, 0, dtype=BF, device=gpu), b)
    assert torch.equal(y, b.expand(4, 5))
    x = torch.empty(0, 8, dtype=BF, device=gpu, requires_grad=True)
    w.requires_grad_(), b.requires_grad_()
    dx, dw, db = torch.autograd.grad(ops.linear(x, w, b, activation="silu"), (x, w, b), torch.empty(0, 5, dtype=BF, device=gpu))
    assert dx.shape == (0, 8) and not bool(dw.any()) and not bool(db.any())


# ---------------------------------------------------------------- linear, gradients
def grads(gpu, x, w, b, r, dy, **kw):
    leaves = [t.to(gpu).requires_grad_() if t is not None else None for t in (x, w, b, r)]
    y = ops.linear(*leaves, **kw)
    live = [t for t in leaves if t is not None]
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None]
    return dict(zip(names, torch.autograd.grad(y, live, dy.to(gpu)))) | {"y": y}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m, k, n", [(1, 16, 8), (5, 7, 3), (77, 64, 128), (130, 765, 437), (1000, 136, 200), (700, 96, 2048), (5000, 40, 72),
                                     (2100, 2048, 64), (2048, 1024, 2304)])
def test_linear_gradients(gpu, dtype, m, k, n):
    x, w, b, dy = rand(m, k, dtype=dtype), rand(n, k, dtype=dtype, scale=k ** -0.5, seed=1), rand(n, dtype=dtype, seed=2), rand(m, n, dtype=dtype, seed=3)
    want = R.linear(x, w, b, None, "none", None, dy)
    for name, g in grads(gpu, x, w, b, None, dy).items():
        R.check(g, want[name], name)


@pytest.mark.parametrize("kind", ["quick_gelu", "gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("m, k, n", [(150, 72, 203), (300, 64, 512)])
def test_linear_gradients_through_the_epilogue(gpu, kind, p, m, k, n):
    x, w, b, r, dy = rand(m, k), rand(n, k, scale=k ** -0.5, seed=1), rand(n, dtype=F32, seed=2), rand(m, n, seed=4), rand(m, n, seed=3)
    if kind == "relu":  # keep z away from the kink, where one ulp decides
        z = x.double() @ w.double().t() + b.double()
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    want = R.linear(x, w, b, r, kind, mask_of(m, n, p), dy)
    for name, g in grads(gpu, x, w, b, r, dy, activation=kind, dropout_p=p, seed=SEED, offset=OFFSET).items():
        R.check(g, want[name], name)


def test_linear_gradient_views(gpu):
    """Expanded and sliced dy, a transposed weight leaf, a broadcast residual, a 3-D x."""
    x, f, r1 = rand(4, 25, 48).to(gpu).requires_grad_(), rand(48, 64, scale=0.15, seed=1).to(gpu).requires_grad_(), rand(64, seed=2).to(gpu).requires_grad_()
    y = ops.linear(x, f.t(), None, r1.expand(4, 25, 64))
    for dy in (torch.ones((), dtype=BF, device=gpu).expand(4, 25, 64), rand(4, 25, 80, seed=3).to(gpu)[..., 7:71]):
        dx, df, dr = torch.autograd.grad(y, (x, f, r1), dy, retain_graph=True)
        d2 = dy.cpu().reshape(100, 64)
        want = R.linear(x.detach().cpu().view(100, 48), f.detach().cpu().t(), None, None, "none", None, d2)
        R.check(dx.view(100, 48), want["dx"])
        R.check(df.t(), want["dw"])
        assert torch.allclose(dr.double().cpu(), d2.double().sum(0), atol=1e-9, rtol=2.0 ** -8 * 3)


def test_linear_gradient_against_differences(gpu):
    """The product is linear in each factor, so a difference of two forwards is the directional derivative (up to
    the outputs' rounding: 2^-9 relative to each y, and dy sums 64 x 96 of them)."""
    x, w, dy, d = rand(64, 128, dtype=HF), rand(96, 128, dtype=HF, scale=0.1, seed=1), rand(64, 96, dtype=HF, seed=2), rand(96, 128, dtype=HF, scale=0.1, seed=3)
    g = grads(gpu, x, w, None, None, dy)
    a, b = ops.linear(x.to(gpu), (w + d).to(gpu)), ops.linear(x.to(gpu), (w - d).to(gpu))
    step = ((w + d).double() - (w - d).double())
    num = ((a.double() - b.double()) * dy.to(gpu).double()).sum().item()
    ana = (g["dw"].double().cpu() * step).sum().item()
    slack = 2.0 ** -11 * ((a.double().abs() + b.double().abs()) * dy.to(gpu).double().abs()).sum().item() + 2.0 ** -11 * (g["dw"].double().cpu() * step).abs().sum().item()
    assert abs(num - ana) <= slack


def test_linear_partial_gradients(gpu):
    """Only what is asked for is computed, with the same values; inference and training forwards agree."""
    x, w, b, dy = rand(90, 64).to(gpu), rand(80, 64, scale=0.1, seed=1).to(gpu), rand(80, seed=2).to(gpu), rand(90, 80, seed=3).to(gpu)
    kw = dict(activation="gelu", dropout_p=0.2, seed=SEED, offset=OFFSET)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    y = ops.linear(*full, **kw)
    want = torch.autograd.grad(y, full, dy)
    assert torch.equal(y, ops.linear(x, w, b, **kw))
    for i in range(3):
        one = [t.clone().requires_grad_() if j == i else t for j, t in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(ops.linear(*one, **kw), one[i], dy)
        assert torch.equal(g, want[i])
    r = x.new_zeros(90, 80).requires_grad_()
    (g,) = torch.autograd.grad(ops.linear(x, w, b, r, **kw), r, dy)
    assert torch.equal(g, dy)


def test_linear_repeats_bit_for_bit(gpu):
    """Split products and column sums are joined in a fixed order."""
    x, w, b, dy = rand(9000, 72), rand(136, 72, scale=0.1, seed=1), rand(136, seed=2), rand(9000, 136, seed=3)
    a, b2 = (grads(gpu, x, w, b, None, dy, activation="silu") for _ in range(2))
    for k in a:
        assert torch.equal(a[k], b2[k])


def test_changed_offset_is_refused_in_backward(gpu):
    off = torch.tensor([3], device=gpu)
    x, w = rand(8, 16).to(gpu).requires_grad_(), rand(8, 16, seed=1).to(gpu)
    y = ops.linear(x, w, dropout_p=0.5, seed=1, offset=off)
    off += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---------------------------------------------------------------- LoRA linear
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("p", [0.0, 0.25, 1.0])
@pytest.mark.parametrize("m, k, n, r", [(1, 64, 48, 4), (77, 512, 200, 4), (130, 765, 437, 8), (33, 40, 72, 1), (300, 96, 264, 33), (2300, 64, 2048, 16)])
def test_lora_linear(gpu, dtype, p, m, k, n, r):
    x, w, A, B = rand(m, k, dtype=dtype), rand(n, k, dtype=dtype, scale=k ** -0.5, seed=1), rand(k, r, dtype=dtype, scale=k ** -0.5, seed=2), rand(r, n, dtype=dtype, scale=0.3, seed=3)
    b, dy = rand(n, dtype=dtype, seed=4), rand(m, n, dtype=dtype, seed=5)
    leaves = [t.to(gpu).requires_grad_() for t in (x, w, A, B, b)]
    kw = dict(scaling=2.0, dropout_p=p, seed=SEED, offset=OFFSET)
    y = ops.lora_linear(*leaves, **kw)
    got = dict(zip(("dx", "dw", "dA", "dB", "db"), torch.autograd.grad(y, leaves, dy.to(gpu)))) | {"y": y}
    want = R.lora(x, w, A, B, b, 2.0, mask_of(m, k, p), dy)
    for name, g in got.items():
        R.check(g, want[name], name)
    with torch.no_grad():
        assert torch.equal(ops.lora_linear(*leaves, **kw), y)


@pytest.mark.parametrize("m, k, n, r, dtype", [(4091, 64, 4088, 33, BF), (4091, 4088, 64, 70, HF), (4091, 4088, 64, 16, BF), (4360, 64, 4096, 96, HF)])
def test_lora_linear_wide_tiles(gpu, m, k, n, r, dtype):
    """Output (and dx) of 16 x 16 tiles of 256, ragged, with one to three steps of 32 ranks; 4360 rows are a round and a rest."""
    test_lora_linear(gpu, dtype, 0.25, m, k, n, r)


@pytest.mark.parametrize("r,k", [(4, 64), (4, 61), (20, 128)])
def test_lora_infinity_stays_an_infinity(gpu, r, k):
    """Positive operands, one infinite element: the row is +inf as in the formula (a padded rank times it would be NaN),
    the others are untouched, and so is everything where the mask drops the element."""
    x, w, A, B = (rand(*s, seed=i).abs() + 0.1 for i, s in enumerate(((40, k), (24, k), (k, r), (r, 24))))
    args = [t.to(gpu) for t in (x, w, A, B)]
    clean = ops.lora_linear(*args, scaling=2.0)
    args[0][7, 5] = float("inf")
    y = ops.lora_linear(*args, scaling=2.0)
    assert bool((y[7] == float("inf")).all())
    rows = [i for i in range(40) if i != 7]
    assert torch.equal(y[rows], clean[rows])
    args[1][:, 5] = 0  # the base product is NaN there; with p = 1 the adapter's side adds nothing
    assert bool(ops.lora_linear(*args, scaling=2.0, dropout_p=1.0, seed=1)[7].isnan().all())
    x2 = x.to(gpu).requires_grad_()
    dy = torch.ones(40, 24, dtype=BF, device=gpu)
    dy[3, 2] = float("inf")
    dx, = torch.autograd.grad(ops.lora_linear(x2, w.to(gpu), *args[2:], scaling=2.0), x2, dy)
    assert bool((dx[3] == float("inf")).all()) and bool(torch.isfinite(dx[:3]).all()) and bool(torch.isfinite(dx[4:]).all())


def test_lora_equals_merge_and_frozen_weight(gpu):
    """B = 0 gives the base Linear bit for bit (the reference's initial state, main.py:27), with a gradient for B."""
    x, w, A = rand(200, 128).to(gpu), rand(96, 128, scale=0.1, seed=1).to(gpu), rand(128, 4, scale=0.02, seed=2).to(gpu).requires_grad_()
    B = torch.zeros(4, 96, dtype=BF, device=gpu, requires_grad=True)
    y = ops.lora_linear(x, w, A, B, scaling=2.0)
    assert torch.equal(y, ops.linear(x, w))
    dA, dB = torch.autograd.grad(y, (A, B), rand(200, 96, seed=3).to(gpu))
    assert not bool(dA.any()) and bool(dB.any())


# ---------------------------------------------------------------- together: streams, graphs, a block under training
def mlp_step(x, p, dy, offset):
    """A residual block's MLP under adapter training: c_fc with its adapter, then c_proj with dropout and residual."""
    h = ops.lora_linear(x, p["w1"], p["A1"], p["B1"], p["b1"], scaling=2.0, dropout_p=0.1, seed=11, offset=offset)
    h = ops.linear(h, p["eye"], activation="quick_gelu")
    y = ops.linear(h, p["w2"], p["b2"], x, dropout_p=0.1, seed=12, offset=offset)
    return (y, *torch.autograd.grad(y, [x, p["A1"], p["B1"], p["w2"], p["b2"]], dy))


def mlp_params(gpu, d=64, f=256):
    p = {"w1": rand(f, d, scale=d ** -0.5, seed=1), "A1": rand(d, 4, scale=0.1, seed=2), "B1": rand(4, f, scale=0.1, seed=3), "b1": rand(f, seed=4),
         "w2": rand(d, f, scale=f ** -0.5, seed=5), "b2": rand(d, seed=6), "eye": torch.eye(f, dtype=BF)}
    p = {k: v.to(gpu) for k, v in p.items()}
    for k in ("A1", "B1", "w2", "b2"):
        p[k].requires_grad_()
    return p


def test_block_step_matches_64_bits(gpu):
    """The chain's outputs within 4 roundings of bf16 (2-norm) of the same chain in 64 bits: y, dx pass h, the
    activation's output, the thin product and dz, each rounded once (2^-9 relative each, in quadrature under 2^-7.5)."""
    p, m = mlp_params(gpu), 150
    x, dy = rand(m, 64, seed=7).to(gpu).requires_grad_(), rand(m, 64, seed=8).to(gpu)
    got = mlp_step(x, p, dy, 5)
    d = {k: v.detach().double().cpu().requires_grad_(v.requires_grad) for k, v in p.items()}
    X = x.detach().double().cpu().requires_grad_()
    h = X @ d["w1"].t() + d["b1"] + 2.0 * (X * mask_of(m, 64, 0.1, 11, 5)) @ d["A1"] @ d["B1"]
    h = h * torch.sigmoid(1.702 * h)
    y = X + mask_of(m, 64, 0.1, 12, 5) * (h @ d["w2"].t() + d["b2"])
    want = (y, *torch.autograd.grad(y, [X, d["A1"], d["B1"], d["w2"], d["b2"]], dy.double().cpu()))
    for a, b in zip(got, want):
        assert (a.detach().double().cpu() - b.detach()).norm() <= 2.0 ** -7.5 * b.detach().norm()


def test_side_stream(gpu):
    p, x, dy = mlp_params(gpu), rand(300, 64, seed=7).to(gpu).requires_grad_(), rand(300, 64, seed=8).to(gpu)
    want = mlp_step(x, p, dy, 5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = mlp_step(x, p, dy, 5)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_step_replays(gpu):
    """Forward and backward in one graph with the offset in device memory: every replay draws the mask of the offset it
    finds and equals the eager step; eager work runs between the replays."""
    p, x, dy = mlp_params(gpu), rand(300, 64, seed=7).to(gpu).requires_grad_(), rand(300, 64, seed=8).to(gpu)
    off = torch.zeros(1, dtype=torch.int64, device=gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            mlp_step(x, p, dy, off)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mlp_step(x, p, dy, off)
    seen = []
    for i in (0, 7, 2 ** 33 + 1, 7):
        off.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = mlp_step(x, p, dy, i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        seen.append(got[0])
    assert torch.equal(seen[1], seen[3]) and not torch.equal(seen[0], seen[1])


def test_capture_beside_a_live_eager_graph_is_refused(gpu):
    """While an eager graph of the same leaves lives, a captured forward for a backward raises before it records anything;
    once that graph is gone the capture works."""
    p, x, dy = mlp_params(gpu), rand(40, 64, seed=7).to(gpu).requires_grad_(), rand(40, 64, seed=8).to(gpu)
    want = [t.detach().clone() for t in mlp_step(x, p, dy, 3)]
    eager = ops.dropout(x, 0.5, seed=1)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.dropout(x, 0.5, seed=1)
    del eager
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mlp_step(x, p, dy, 3)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_one_column_of_many_rows(gpu):
    """K = 1 on 2^26 + 100 rows: the operand is one run of elements, whose length passes what a tile's offsets hold."""
    m = 2 ** 26 + 100
    x, w = torch.randn(m, 1, device=gpu).to(BF), torch.tensor([[2.0], [-0.5], [1.0], [4.0], [0.25], [-1.0], [8.0], [0.5]], dtype=BF, device=gpu)
    y = ops.linear(x, w)
    assert torch.equal(y, x * w.t())  # powers of two: exact


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_rounds_and_remaining_rows(gpu, p):
    """7300 x 2304 is one round of 256-wide tiles (28 rows of 9) and 132 rows more, a launch of their own: masks, residual,
    slope and the low-rank term go by the whole operand's rows. Row- and column-contiguous x (the wide direction is dx's too)."""
    m, k, n = 7300, 64, 2304
    x, w, b, r, dy = rand(m, k), rand(n, k, scale=k ** -0.5, seed=1), rand(n, seed=2), rand(m, n, seed=4), rand(m, n, seed=3)
    want = R.linear(x, w, b, r, "gelu", mask_of(m, n, p), dy)
    for name, g in grads(gpu, x, w, b, r, dy, activation="gelu", dropout_p=p, seed=SEED, offset=OFFSET).items():
        R.check(g, want[name], name)
    xt = x.to(gpu).t().contiguous().t()
    R.check(ops.linear(xt, w.to(gpu), b.to(gpu)), R.linear(x, w, b)["y"])
    # dx of this one is [7300, 2304], with the masked low-rank term
    x, w, A, B, dy = rand(m, n, seed=5), rand(k, n, scale=n ** -0.5, seed=6), rand(n, 4, scale=n ** -0.5, seed=7), rand(4, k, scale=0.3, seed=8), rand(m, k, seed=9)
    leaves = [t.to(gpu).requires_grad_() for t in (x, A, B)]
    y = ops.lora_linear(leaves[0], w.to(gpu), *leaves[1:], scaling=2.0, dropout_p=p, seed=SEED, offset=OFFSET)
    want = R.lora(x, w, A, B, None, 2.0, mask_of(m, n, p), dy)
    for name, g in zip(("dx", "dA", "dB"), torch.autograd.grad(y, leaves, dy.to(gpu))):
        R.check(g, want[name], name)
    R.check(y, want["y"])


def test_long_rows_offsets_past_32_bits(gpu):
    """A [rows, 4096] output of more than 2^32 bytes: the last rows are addressed in 64 bits (checked on slices against
    the same rows computed alone)."""
    m, k, n = 530000, 32, 4096
    x, w = torch.randn(m, k, device=gpu, dtype=BF), rand(n, k, scale=0.2, seed=1).to(gpu)
    y = ops.linear(x, w)
    for a in (0, 262143, m - 300):
        assert torch.equal(y[a:a + 300], ops.linear(x[a:a + 300], w))
    (dw,) = torch.autograd.grad(ops.linear(x, w.requires_grad_()), w, y)
    want = torch.zeros(n, k, dtype=torch.float64, device=gpu)
    for a in range(0, m, 53000):
        want += y[a:a + 53000].double().t() @ x[a:a + 53000].double()
    assert (dw.double() - want).norm() <= 2.0 ** -8 * want.norm()


def test_graph_is_run_once_unless_retained(gpu):
    x = rand(40, 24, dtype=BF, seed=1).to(gpu).requires_grad_()
    w = rand(16, 24, dtype=BF, seed=2).to(gpu).requires_grad_()
    A, B = (rand(*s, dtype=BF, seed=i).to(gpu).requires_grad_() for i, s in ((3, (24, 4)), (4, (4, 16))))
    for make, leaves in ((lambda: ops.linear(x, w, activation="gelu", dropout_p=0.2, seed=1), (x, w)),
                         (lambda: ops.dropout(x, 0.3, seed=1), (x,)),
                         (lambda: ops.lora_linear(x, w, A, B, scaling=0.5, dropout_p=0.2, seed=1), (x, w, A, B))):
        y = make()
        dy = torch.ones_like(y)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        second = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(first, second))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, leaves, dy)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(make(), leaves, dy, create_graph=True)


def test_operand_changed_in_place_is_refused_in_backward(gpu):
    x = rand(3, 5, 24, dtype=HF, seed=1).to(gpu)
    w = rand(16, 24, dtype=HF, seed=2).to(gpu).requires_grad_()
    y = ops.linear(x, w)
    x.mul_(2)  # a view of it is what the node saved
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_two_threads(gpu):
    import threading
    x, w = rand(300, 64, dtype=BF, seed=1).to(gpu), rand(128, 64, dtype=BF, seed=2).to(gpu)
    want = ops.linear(x, w, activation="silu", dropout_p=0.1, seed=5)
    got = [None] * 4

    def work(i):
        xs = x.clone().requires_grad_()
        for _ in range(20):
            got[i] = ops.linear(xs, w, activation="silu", dropout_p=0.1, seed=5)
            got[i].backward(torch.ones_like(got[i]))
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(g, want) for g in got)


def test_forward_mode_is_refused(gpu):
    import torch.autograd.forward_ad as fwd
    x, w = rand(4, 8, seed=1).to(gpu), rand(6, 8, seed=2).to(gpu)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.linear(d, w), lambda: ops.dropout(d, 0.5, seed=1), lambda: ops.lora_linear(x, w, d.t()[:, :2], w.t()[:2, :6])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_saved_tensor_hooks(gpu):
    x, w, A, B = (rand(*s, seed=i).to(gpu).requires_grad_() for i, s in enumerate(((40, 24), (16, 24), (24, 4), (4, 16))))
    dy = rand(40, 16, seed=9).to(gpu)

    def step():
        y = ops.linear(x, w, activation="silu", dropout_p=0.2, seed=1) + ops.lora_linear(x, w, A, B, scaling=0.5, dropout_p=0.2, seed=2)
        return torch.autograd.grad(y, (x, w, A, B), dy)

    want = step()
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    # another layout may change the order of a sum, so the last bit of an output or of du (eps / 2 of a value each, twice)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().contiguous(), lambda t: t.t()):
        for a, b in zip(step(), want):
            assert float((a - b).float().norm()) <= 2 * torch.finfo(BF).eps * float(b.float().norm())
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1]), pytest.raises(RuntimeError, match="saved tensor came back"):
        step()
    offset = torch.ones(1, dtype=torch.int64, device=gpu)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu()), pytest.raises(RuntimeError, match="saved tensor came back"):
        torch.autograd.grad(ops.dropout(x, 0.5, seed=1, offset=offset), x, rand(40, 24).to(gpu))
