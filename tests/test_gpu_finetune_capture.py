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
