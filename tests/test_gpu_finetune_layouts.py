"""Layouts of the fine-tuning operators' operands: an adapter's factors, one long column."""
import pytest
import torch

import finetune_ref as R
from interior_amd import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def rand(*shape, dtype=BF, scale=1.0, seed=0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def test_one_column_of_a_row_length_that_wraps(gpu):
    """K = 1 on 2^26 - 1 rows: copied to a padded row of 2^26 elements, 32 times whose bytes is 2^32; an infinity stays one."""
    m = 2 ** 26 - 1
    x, w = torch.ones(m, 1, dtype=BF, device=gpu), torch.tensor([[2.0], [-0.5], [1.0], [4.0], [0.25], [-1.0], [8.0], [0.5]], dtype=BF, device=gpu)
    x[5] = float("inf")
    assert torch.equal(ops.linear(x, w), x * w.t())  # powers of two: exact


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("m, k, n, r", [(90, 72, 120, 5), (300, 96, 264, 33)])
def test_lora_views(gpu, p, m, k, n, r):
    """Column-contiguous, sliced and strided factors, a sliced and a three-dimensional x, an expanded dy and an fp32 bias."""
    bx, w, bias = rand(m + 2, k + 16).to(gpu), rand(n, k, scale=k ** -0.5, seed=1).to(gpu).requires_grad_(), rand(n, dtype=F32, seed=4).to(gpu).requires_grad_()
    bA, bB = rand(k + 3, 2 * r + 8, scale=k ** -0.5, seed=2).to(gpu), rand(2 * r + 1, n + 8, scale=0.3, seed=3).to(gpu)
    At, Bt = bA[:k, :r].t().contiguous(), bB[:r, :n].t().contiguous()
    As = [bA[:k, :r], At.t(), bA[3:, 5:5 + r], bA[:k, :2 * r:2]]
    Bs = [bB[:r, :n], Bt.t(), bB[1:r + 1, 3:n + 3], bB[:2 * r:2, :n]]
    xs = [bx[:m, :k], bx[2:, 8:k + 8], bx[1:m + 1, 5:k + 5], bx[:m, :k].contiguous().view(2, m // 2, k)]
    dys = [rand(m, n, seed=5).to(gpu), torch.full((), 0.5, dtype=BF, device=gpu).expand(m, n), rand(m, n + 8, seed=6).to(gpu)[:, 3:n + 3]]
    mask = None if p == 0 else R.keep_mask(m, k, p, 7, 8).double() / (1 - p)
    for i in range(4):
        for j in range(3):
            x, A, B = (t.detach().requires_grad_() for t in (xs[i], As[(i + j) % 4], Bs[(i + 2 * j) % 4]))
            dy = dys[j]
            y = ops.lora_linear(x, w, A, B, bias, scaling=2.0, dropout_p=p, seed=7, offset=8)
            got = dict(zip(("dx", "dw", "dA", "dB", "db"), torch.autograd.grad(y, (x, w, A, B, bias), dy.view(y.shape)))) | {"y": y}
            want = R.lora(x.detach().cpu().reshape(m, k), w.detach().cpu(), A.detach().cpu(), B.detach().cpu(), bias.detach().cpu(), 2.0, mask, dy.cpu())
            for name, g in got.items():
                R.check(g.reshape(want[name][0].shape), want[name], (name, i, j))


def test_lora_factor_gradients_without_dx(gpu):
    """A frozen x and Linear: dA and dB alone, and each alone, with the values of the full backward pass."""
    m, k, n, r = 700, 136, 200, 16
    x, w, A, B, dy = (rand(*s, scale=c, seed=i).to(gpu) for i, (s, c) in enumerate((((m, k), 1), ((n, k), k ** -0.5), ((k, r), k ** -0.5), ((r, n), 0.3), ((m, n), 1))))
    want = R.lora(x.cpu(), w.cpu(), A.cpu(), B.cpu(), None, 2.0, R.keep_mask(m, k, 0.25, 7, 8).double() / 0.75, dy.cpu())
    for wanted in ("AB", "A", "B"):
        leaves = {"A": A.clone(), "B": B.clone()}
        for c in wanted:
            leaves[c].requires_grad_()
        y = ops.lora_linear(x, w, leaves["A"], leaves["B"], scaling=2.0, dropout_p=0.25, seed=7, offset=8)
        for c, g in zip(wanted, torch.autograd.grad(y, [leaves[c] for c in wanted], dy)):
            assert bool(g.any())
            R.check(g, want["d" + c], wanted)
