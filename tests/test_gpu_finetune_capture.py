"""The guard against capturing a backward pass whose leaves belong to another stream's graph."""
import ctypes

import pytest
import torch

from interior_amd import _lib, ops

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def test_a_failing_capture_query_is_an_error(gpu):
    """A query that cannot say whether a capture is under way stops a forward that wants gradients, and no other."""
    m, table = ops._binding(), ops._entry_points()
    fails = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int))(lambda stream, status: 1)
    x, w = rand(40, 24).to(gpu), rand(16, 24, seed=1).to(gpu).requires_grad_()
    try:
        m.set_library(table | {"hipStreamIsCapturing": ctypes.cast(fails, ctypes.c_void_p).value}, _lib.ClipVitError)
        with pytest.raises(RuntimeError, match="capturing"):
            ops.linear(x, w)
        with torch.no_grad():
            ops.linear(x, w)
    finally:
        m.set_library(table, _lib.ClipVitError)
    ops.linear(x, w)


@pytest.mark.parametrize("make", [lambda x: x * 2, lambda x: (x.view(2, 20, 24) * 2).transpose(0, 1).reshape(40, 24).relu()])
def test_leaf_behind_other_operations(gpu, make):
    """The leaf is found behind torch's own operations on the capturing stream; once the eager graph is gone the capture
    works and its replays are right."""
    x, w, dy = rand(40, 24).to(gpu).requires_grad_(), rand(16, 24, seed=1).to(gpu), rand(40, 16, seed=2).to(gpu)

    def step():
        y = ops.linear(make(x), w, activation="silu")
        return y.detach(), *torch.autograd.grad(y, x, dy)

    want = [t.clone() for t in step()]
    eager = make(x)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.linear(make(x), w, activation="silu")
    del eager
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step()


def test_input_computed_before_the_capture(gpu):
    """An input that an eager graph made, differentiated only as far as itself, is no reason to refuse."""
    leaf, w, dy = rand(40, 24).to(gpu).requires_grad_(), rand(16, 24, seed=1).to(gpu), rand(40, 16, seed=2).to(gpu)
    x = leaf * 2
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        y0 = ops.linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h = torch.cuda.CUDAGraph()
        with torch.cuda.graph(h, stream=s):
            y = ops.linear(x, w)
    g.replay(), h.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, y0) and torch.equal(y, ops.linear(x.detach(), w))
