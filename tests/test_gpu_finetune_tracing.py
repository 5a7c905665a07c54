"""Tracers and function transforms: refused, never a program that returns uninitialised memory; a compiler that runs the
calls as they are gets the same results."""
import pytest
import torch

from interior_amd import ops
from test_finetune_contract import tracers

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(BF)


@pytest.fixture
def calls(gpu):
    w, A, B = (rand(*s, seed=i).to(gpu) for i, s in enumerate(((16, 24), (24, 4), (4, 16))))
    return [lambda x: ops.linear(x, w, activation="silu"), lambda x: ops.dropout(x, 0.5, seed=1), lambda x: ops.lora_linear(x, w, A, B)]


@pytest.mark.parametrize("how", ["jit.trace", "make_fx", "make_fx symbolic", "fake"])
def test_tracing_is_refused(gpu, calls, how):
    x = rand(40, 24, seed=5).to(gpu)
    for call in calls:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            tracers()[how](call, x)


def test_function_transforms_raise(gpu, calls):
    x = rand(3, 40, 24, seed=5).to(gpu)
    for call in calls:
        for transform in (torch.func.vmap(call), torch.func.grad(lambda t: call(t).float().sum())):
            with pytest.raises(RuntimeError):
                transform(x)


def test_eager_compiler_and_counting_modes_run_them(gpu, calls):
    from torch.utils.flop_counter import FlopCounterMode
    x = rand(40, 24, seed=5).to(gpu)
    for call in calls:
        want = call(x)
        assert torch.equal(torch.compile(call, backend="eager")(x), want)
        with FlopCounterMode(display=False):
            assert torch.equal(call(x), want)
