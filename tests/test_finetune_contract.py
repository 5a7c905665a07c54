"""What the fine-tuning operators ask of their callers and of the build, without a GPU."""
import ctypes

import pytest
import torch

from interior_amd import _lib, ops
from test_finetune import linear_grad_args, lora_grad_args


@pytest.mark.parametrize("args", [
    linear_grad_args(dw=None, x=None, x_row=0, x_col=0), linear_grad_args(dx=None, w=None, w_row=0, w_col=0),
    linear_grad_args(dx=None, dw=None, x=None, w=None, x_row=0, x_col=0, w_row=0, w_col=0)])
def test_linear_grad_needs_what_its_outputs_read(args):
    need = ctypes.c_size_t()
    assert _lib.lib().clipvit_linear_grad_workspace(ctypes.byref(args), ctypes.byref(need)) == 0


NO_X, NO_W = dict(x=None, x_stride=0), dict(w=None, w_row=0, w_col=0)
NO_A, NO_B, NO_U = dict(a=None, a_row=0, a_col=0), dict(b=None, b_row=0, b_col=0), dict(u=None)


@pytest.mark.parametrize("kw", [
    dict(dw=None, da=None, **NO_X),
    dict(dx=None, **NO_W, **NO_A),
    dict(dx=None, da=None, **NO_W, **NO_A, **NO_B),
    dict(db_factor=None, **NO_U),
    dict(dx=None, dw=None, da=None, db_factor=None, **NO_X, **NO_W, **NO_A, **NO_B, **NO_U)])
def test_lora_grad_needs_what_its_outputs_read(kw):
    need = ctypes.c_size_t()
    assert _lib.lib().clipvit_lora_linear_grad_workspace(ctypes.byref(lora_grad_args(**kw)), ctypes.byref(need)) == 0


@pytest.mark.parametrize("name", ["hipStreamIsCapturing", "clipvit_linear", "clipvit_last_error"])
def test_binding_refuses_a_library_without_an_entry(name):
    """A missing entry is an error when the binding is set up, not a check that is silently left out later."""
    m, table = ops._binding(), ops._entry_points()
    try:
        for bad in ({k: v for k, v in table.items() if k != name}, table | {name: 0}):
            with pytest.raises(RuntimeError, match=name):
                m.set_library(bad, _lib.ClipVitError)
    finally:
        m.set_library(table, _lib.ClipVitError)


def tracers():
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def fake(call, x):
        with FakeTensorMode(allow_non_fake_inputs=True):
            call(x)

    return {"jit.trace": lambda call, x: torch.jit.trace(call, x), "make_fx": lambda call, x: make_fx(call)(x),
            "make_fx symbolic": lambda call, x: make_fx(call, tracing_mode="symbolic")(x), "fake": fake}


@pytest.mark.parametrize("how", ["jit.trace", "make_fx", "make_fx symbolic", "fake"])
def test_binding_refuses_to_be_traced(how):
    """A trace would record the output's allocation and nothing that fills it. (The binding itself: it asks before it looks
    at the tensors' device.)"""
    m, w, A, B = ops._binding(), torch.zeros(5, 8), torch.zeros(8, 2), torch.zeros(2, 5)
    for call in (lambda x: m.linear(x, w, None, None, 0, 0.0, 0, 0, None), lambda x: m.dropout(x, None, 0.5, 0, 0, None),
                 lambda x: m.lora_linear(x, w, A, B, None, 1.0, 0.0, 0, 0, None)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            tracers()[how](call, torch.zeros(4, 8))
