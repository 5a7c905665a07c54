"""What the fine-tuning operators keep between forward and backward: what the wanted gradients read, nothing else."""
import pytest
import torch

import finetune_ref as R
from interior_amd import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
M, K, N, RANK = 40, 24, 16, 4


def rand(*shape, dtype=BF, scale=1.0, seed=0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def operands(gpu):
    return {k: rand(*s, seed=i).to(gpu) for i, (k, s) in enumerate({"x": (M, K), "w": (N, K), "b": (N,), "r": (M, N), "A": (K, RANK), "B": (RANK, N)}.items())}


def saved(call):
    """The data pointers of what a forward packs for its backward, and its result."""
    kept = []

    def pack(t):
        kept.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = call()
    return y, kept


def names(kept, ops_of):
    ptr = {t.data_ptr(): k for k, t in ops_of.items()}
    return sorted(ptr.get(t.data_ptr(), "slope" if t.dtype == torch.int16 else "offset" if t.dtype == torch.int64 else "u") for t in kept)


@pytest.mark.parametrize("wanted, keeps", [("x", ["slope", "w"]), ("w", ["slope", "x"]), ("b", ["slope"]), ("r", []), ("xw", ["slope", "w", "x"]), ("br", ["slope"])])
def test_linear_saves_what_its_gradients_read(gpu, wanted, keeps):
    t = operands(gpu)
    for k in wanted:
        t[k].requires_grad_()
    offset = torch.zeros(1, dtype=torch.int64, device=gpu)
    for act in ("gelu", "none"):
        for off in (offset, 3):
            _, kept = saved(lambda: ops.linear(t["x"], t["w"], t["b"], t["r"], activation=act, dropout_p=0.2, seed=1, offset=off))
            want = [k for k in keeps if act != "none" or k != "slope"] + (["offset"] if torch.is_tensor(off) and wanted != "r" else [])
            assert names(kept, t) == sorted(want), (wanted, act)


@pytest.mark.parametrize("wanted, keeps", [("x", ["A", "B", "w"]), ("w", ["x"]), ("A", ["B", "x"]), ("B", ["u"]), ("b", []), ("AB", ["B", "u", "x"]),
                                           ("xwABb", ["A", "B", "u", "w", "x"])])
def test_lora_saves_what_its_gradients_read(gpu, wanted, keeps):
    t = operands(gpu)
    for k in wanted:
        t[k].requires_grad_()
    dy = rand(M, N, seed=9).to(gpu)
    y, kept = saved(lambda: ops.lora_linear(t["x"], t["w"], t["A"], t["B"], t["b"], scaling=0.5, dropout_p=0.25, seed=1, offset=2))
    assert names(kept, t) == keeps
    got = torch.autograd.grad(y, [t[k] for k in wanted], dy)
    mask = R.keep_mask(M, K, 0.25, 1, 2).double() / 0.75
    want = R.lora(*(t[k].detach().cpu() for k in "xwABb"), 0.5, mask, dy.cpu())
    for k, g in zip(wanted, got):
        R.check(g, want[{"x": "dx", "w": "dw", "A": "dA", "B": "dB", "b": "db"}[k]], k)


def test_operands_that_no_gradient_reads_may_change(gpu):
    """A frozen weight's x, a frozen input's weight: changed in place between forward and backward, the gradients are right."""
    t, dy = operands(gpu), rand(M, N, seed=9).to(gpu)
    want = R.linear(t["x"].cpu(), t["w"].cpu(), None, None, "none", None, dy.cpu())
    x = t["x"].clone().requires_grad_()
    y = ops.linear(x, t["w"])
    with torch.no_grad():
        x.mul_(3)
    R.check(torch.autograd.grad(y, x, dy)[0], want["dx"])
    w = t["w"].clone().requires_grad_()
    y = ops.linear(t["x"], w)
    with torch.no_grad():
        w.mul_(3)
    R.check(torch.autograd.grad(y, w, dy)[0], want["dw"])
    r, offset = t["r"].clone().requires_grad_(), torch.zeros(1, dtype=torch.int64, device=gpu)
    y = ops.linear(t["x"], t["w"], None, r, dropout_p=0.5, seed=1, offset=offset)
    offset += 1
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)


@pytest.mark.parametrize("call, draws, others", [
    (lambda t, off: ops.linear(t["x"], t["w"], t["b"], t["r"], activation="silu", dropout_p=0.5, seed=1, offset=off), "xwb", "r"),
    (lambda t, off: ops.dropout(t["x"], 0.5, seed=1, offset=off, residual=t["r2"]), "x", ["r2"]),
    (lambda t, off: ops.lora_linear(t["x"], t["w"], t["A"], t["B"], t["b"], dropout_p=0.5, seed=1, offset=off), "xA", "wBb")])
def test_changed_offset_stops_only_what_draws_the_mask(gpu, call, draws, others):
    """A gradient that does not draw the mask again is the same after the offset has changed; one that does is refused."""
    t, offset = operands(gpu), torch.zeros(1, dtype=torch.int64, device=gpu)
    t["r2"] = rand(M, K, seed=8).to(gpu)
    for leaf in t.values():
        leaf.requires_grad_()
    y = call(t, offset)
    dy = rand(*y.shape, seed=9).to(gpu)
    want = torch.autograd.grad(y, [t[k] for k in others], dy, retain_graph=True)
    offset += 1
    got = torch.autograd.grad(y, [t[k] for k in others], dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for k in draws:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, t[k], dy, retain_graph=True)
