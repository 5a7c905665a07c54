"""Fine-tuning operators without a GPU: refusals of the Python surface and of the C entry points (both check before
any device work), the mask generator's definition, and the reference formulas against differences."""
import ctypes

import pytest
import torch

import finetune_ref as R
from interior_amd import _lib, ops

BF, HF = torch.bfloat16, torch.float16


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def test_philox_known_answers():
    """The three published known-answer vectors of Philox4x32-10 (Random123 distribution, SC 2011)."""
    assert R.philox((0, 0, 0, 0), (0, 0)) == (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    f = 0xFFFFFFFF
    assert R.philox((f, f, f, f), (f, f)) == (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)
    assert R.philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == (
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)


def test_mask_rate_and_independence():
    a, b = R.keep_mask(256, 1024, 0.25, 3, 0), R.keep_mask(256, 1024, 0.25, 3, 1)
    n = a.numel()
    sd = (0.25 * 0.75 / n) ** 0.5
    assert abs(a.double().mean() - 0.75) < 6 * sd
    both = (a & b).double().mean()
    assert abs(both - 0.75 ** 2) < 6 * (0.5625 * 0.4375 / n) ** 0.5


@pytest.mark.parametrize("call, error", [
    (lambda: ops.linear(t(4, 8), t(5, 9)), ValueError),
    (lambda: ops.linear(t(4, 8), t(8)), ValueError),
    (lambda: ops.linear(t(4, 8, dtype=torch.float32), t(5, 8)), TypeError),
    (lambda: ops.linear(t(4, 8), t(5, 8, dtype=HF)), TypeError),
    (lambda: ops.linear(t(4, 8), t(5, 8), t(4)), ValueError),
    (lambda: ops.linear(t(4, 8), t(5, 8), t(5, dtype=HF)), TypeError),
    (lambda: ops.linear(t(4, 8), t(5, 8), None, t(4, 6)), ValueError),
    (lambda: ops.linear(t(4, 8), t(5, 8), None, t(1, 5)), ValueError),
    (lambda: ops.linear(t(4, 8), t(5, 8), activation="tanh"), ValueError),
    (lambda: ops.linear(t(4, 8), t(5, 8), dropout_p=1.5), ValueError),
    (lambda: ops.linear(t(4, 8), t(5, 8), dropout_p=float("nan")), ValueError),
    (lambda: ops.linear(t(4, 8), t(5, 8), dropout_p=0.5, seed=1.0), TypeError),
    (lambda: ops.linear(t(4, 8), t(5, 8), dropout_p=0.5, offset=torch.zeros(2, dtype=torch.int64)), TypeError),
    (lambda: ops.linear(t(4, 8), t(5, 8)), _lib.ClipVitError),  # CPU tensors: no fallback
    (lambda: ops.dropout(t(4, 8, dtype=torch.float64), 0.5, seed=0), TypeError),
    (lambda: ops.dropout(torch.zeros((), dtype=BF), 0.5, seed=0), ValueError),
    (lambda: ops.dropout(t(4, 8), -0.1, seed=0), ValueError),
    (lambda: ops.dropout(t(4, 8), 0.1, seed=0, residual=t(8)), ValueError),
    (lambda: ops.dropout(t(4, 8), 0.1, seed=0), _lib.ClipVitError),
    (lambda: ops.lora_linear(t(4, 8), t(5, 8), t(7, 2), t(2, 5)), ValueError),
    (lambda: ops.lora_linear(t(4, 8), t(5, 8), t(8, 2), t(3, 5)), ValueError),
    (lambda: ops.lora_linear(t(4, 8), t(5, 8), t(8, 0), t(0, 5)), ValueError),
    (lambda: ops.lora_linear(t(4, 8), t(5, 8), t(8, 2, dtype=torch.float32), t(2, 5)), TypeError),
    (lambda: ops.lora_linear(t(4, 8), t(5, 8), t(8, 2), t(2, 5)), _lib.ClipVitError),
])
def test_python_refusals(call, error):
    with pytest.raises(error):
        call()


FAKE = 4096  # never dereferenced: every call below is refused before a launch


def build(cls, base, kw):
    a = cls(**{k: v for k, v in base.items()})
    for k, v in kw.items():
        if k == "p":
            a.dropout.p = v
        else:
            setattr(a, k, v)
    return a


def linear_args(**kw):
    return build(_lib.LinearArgs, dict(dtype=_lib.BF16, bias_dtype=_lib.BF16, M=4, N=8, K=16, x=FAKE, w=FAKE, y=FAKE, x_row=16,
                                       x_col=1, w_row=16, w_col=1, y_stride=8), kw)


def linear_grad_args(**kw):
    return build(_lib.LinearGradArgs, dict(dtype=_lib.BF16, bias_dtype=_lib.BF16, M=4, N=8, K=16, dy=FAKE, dy_stride=8, x=FAKE,
                                           w=FAKE, x_row=16, x_col=1, w_row=16, w_col=1, dx=FAKE, dw=FAKE, db=FAKE), kw)


def lora_args(**kw):
    return build(_lib.LoraArgs, dict(dtype=_lib.F16, bias_dtype=_lib.F32, M=4, N=8, K=16, rank=4, x=FAKE, x_stride=16, w=FAKE, w_row=16,
                                     w_col=1, a=FAKE, a_row=4, a_col=1, b=FAKE, b_row=8, b_col=1, y=FAKE, u=FAKE, scaling=1.0), kw)


def lora_grad_args(**kw):
    return build(_lib.LoraGradArgs, dict(dtype=_lib.F16, bias_dtype=_lib.F32, M=4, N=8, K=16, rank=4, dy=FAKE, dy_stride=8, x=FAKE,
                                         x_stride=16, w=FAKE, w_row=16, w_col=1, a=FAKE, a_row=4, a_col=1, b=FAKE, b_row=8, b_col=1,
                                         u=FAKE, dx=FAKE, dw=FAKE, da=FAKE, db_factor=FAKE, dbias=FAKE, scaling=1.0), kw)


def refused(name, a):
    L, need = _lib.lib(), ctypes.c_size_t()
    assert getattr(L, f"clipvit_{name}_workspace")(ctypes.byref(a), ctypes.byref(need)) == _lib.E_INVALID
    assert getattr(L, f"clipvit_{name}")(None, ctypes.byref(a), None, 0) == _lib.E_INVALID
    assert L.clipvit_last_error()


COMMON = [{"dtype": _lib.F32}, {"dtype": 7}, {"bias_dtype": _lib.MXFP8}, {"M": -1}, {"N": -1}, {"K": 1 << 31}, {"p": 1.01}, {"p": -0.5},
          {"p": float("nan")}, {"w_row": 0}, {"w_row": 1 << 22}, {"w_row": 32, "w_col": 2}]


@pytest.mark.parametrize("kw", COMMON + [{"activation": 6}, {"activation": -1}, {"x": None}, {"w": None}, {"y": None}, {"y_stride": 7},
                                         {"x_row": 8}, {"x_row": 32, "x_col": 2}, {"residual": FAKE, "residual_stride": -8}])
def test_linear_entry_refuses(kw):
    refused("linear", linear_args(**kw))


@pytest.mark.parametrize("kw", COMMON + [{"dy": None}, {"x": None}, {"w": None}, {"dy_stride": 7}, {"dy_stride": 1 << 22}, {"x_row": 8}])
def test_linear_grad_entry_refuses(kw):
    refused("linear_grad", linear_grad_args(**kw))


@pytest.mark.parametrize("kw", COMMON + [{"rank": 0}, {"rank": 65537}, {"x": None}, {"w": None}, {"a": None}, {"b": None}, {"y": None},
                                         {"u": None}, {"u": FAKE + 8}, {"x_stride": 15}])
def test_lora_entry_refuses(kw):
    refused("lora_linear", lora_args(**kw))


@pytest.mark.parametrize("kw", COMMON + [{"rank": 0}, {"dy": None}, {"x": None}, {"w": None}, {"a": None}, {"b": None}, {"u": None},
                                         {"u": FAKE + 8}, {"dy_stride": 7}, {"x_stride": 15}])
def test_lora_grad_entry_refuses(kw):
    refused("lora_linear_grad", lora_grad_args(**kw))


@pytest.mark.parametrize("name, args", [
    ("linear", linear_args(K=17, x_row=17, w_row=17)),  # odd rows: both operands are copied first
    ("linear_grad", linear_grad_args(M=400)), ("lora_linear", lora_args()), ("lora_linear_grad", lora_grad_args())])
def test_workspace_rules(name, args):
    L, need = _lib.lib(), ctypes.c_size_t()
    size, call = getattr(L, f"clipvit_{name}_workspace"), getattr(L, f"clipvit_{name}")
    assert size(None, ctypes.byref(need)) == _lib.E_INVALID and size(ctypes.byref(args), None) == _lib.E_INVALID
    assert call(None, None, None, 0) == _lib.E_INVALID
    assert size(ctypes.byref(args), ctypes.byref(need)) == 0 and need.value > 0
    assert call(None, ctypes.byref(args), None, 0) == _lib.E_INVALID
    assert call(None, ctypes.byref(args), None, need.value) == _lib.E_INVALID
    assert call(None, ctypes.byref(args), FAKE + 16, need.value) == _lib.E_INVALID
    assert call(None, ctypes.byref(args), FAKE, need.value - 1) == _lib.E_INVALID


def test_empty_calls_launch_nothing():
    L = _lib.lib()
    for name, a in (("linear", linear_args(M=0, x=None, y=None)), ("linear", linear_args(N=0, w=None, y=None)),
                    ("linear_grad", linear_grad_args(dx=None, dw=None, db=None)), ("lora_linear", lora_args(M=0, x=None))):
        assert getattr(L, f"clipvit_{name}")(None, ctypes.byref(a), None, 0) == 0


def test_dropout_entry_refuses():
    L, d, bad = _lib.lib(), _lib.DropoutArgs(0.5, 1, 0, None), _lib.DropoutArgs(2.0, 1, 0, None)
    v, B = FAKE, ctypes.byref
    assert L.clipvit_dropout(None, _lib.BF16, v, 8, None, 0, v, 8, 4, 8, None) == _lib.E_INVALID
    assert L.clipvit_dropout(None, _lib.BF16, v, 8, None, 0, v, 8, 4, 8, B(bad)) == _lib.E_INVALID
    assert L.clipvit_dropout(None, _lib.MXFP8, v, 8, None, 0, v, 8, 4, 8, B(d)) == _lib.E_INVALID
    assert L.clipvit_dropout(None, _lib.BF16, None, 8, None, 0, v, 8, 4, 8, B(d)) == _lib.E_INVALID
    assert L.clipvit_dropout(None, _lib.BF16, v, 8, None, 0, v, 7, 4, 8, B(d)) == _lib.E_INVALID
    assert L.clipvit_dropout(None, _lib.BF16, v, 8, None, 0, v, 8, -1, 8, B(d)) == _lib.E_INVALID
    assert L.clipvit_dropout(None, _lib.BF16, None, 8, None, 0, None, 8, 0, 8, B(d)) == 0


def test_struct_layouts():
    assert ctypes.sizeof(_lib.DropoutArgs) == 32
    assert ctypes.sizeof(_lib.LinearArgs) == 16 + 24 + 2 * 24 + 8 + 16 + 16 + 8 + 32
    assert ctypes.sizeof(_lib.LinearGradArgs) == 8 + 24 + 16 + 2 * 24 + 8 + 24 + 32
    assert ctypes.sizeof(_lib.LoraArgs) == 8 + 32 + 16 + 3 * 24 + 3 * 8 + 8 + 32
    assert ctypes.sizeof(_lib.LoraGradArgs) == 8 + 32 + 2 * 16 + 3 * 24 + 8 + 5 * 8 + 8 + 32


@pytest.mark.parametrize("kind", ["none", "quick_gelu", "gelu", "gelu_tanh", "silu", "relu"])
def test_reference_gradients_against_differences(kind):
    """The formulas the GPU tests compare with, against central differences of their own forward."""
    g = torch.Generator().manual_seed(5)
    x, w, b = (torch.randn(s, generator=g).double() for s in ((3, 5), (4, 5), (4,)))
    r, dy = torch.randn(3, 4, generator=g).double(), torch.randn(3, 4, generator=g).double()
    mask = R.keep_mask(3, 4, 0.5, 9, 2).double() * 2

    def f(x, w, b, r):
        return ((r + mask * R.act(x @ w.t() + b, kind)[0]) * dy).sum()

    z = x @ w.t() + b
    dz = dy * mask * R.act(z, kind)[1]
    h = 1e-6
    for name, grad in (("x", dz @ w), ("w", dz.t() @ x), ("b", dz.sum(0)), ("r", dy)):
        base = {"x": x, "w": w, "b": b, "r": r}
        num = torch.zeros_like(base[name])
        for i in range(num.numel()):
            e = torch.zeros(num.numel(), dtype=torch.float64)
            e[i] = h
            e = e.view_as(num)
            num.view(-1)[i] = (f(**(base | {name: base[name] + e})) - f(**(base | {name: base[name] - e}))) / (2 * h)
        assert torch.allclose(num, grad, atol=1e-7, rtol=1e-7), name


def test_lora_reference_gradients_against_differences():
    g = torch.Generator().manual_seed(6)
    v = {"x": torch.randn(3, 8, generator=g), "w": torch.randn(4, 8, generator=g), "A": torch.randn(8, 2, generator=g),
         "B": torch.randn(2, 4, generator=g)}
    v = {k: a.double() for k, a in v.items()}
    dy, mask = torch.randn(3, 4, generator=g).double(), R.keep_mask(3, 8, 0.5, 1, 0).double() * 2

    def f(x, w, A, B):
        return ((x @ w.t() + 1.5 * (x * mask) @ A @ B) * dy).sum()

    leaves = {k: a.clone().requires_grad_() for k, a in v.items()}
    f(**leaves).backward()
    h = 1e-6
    for k in v:
        d = torch.randn(v[k].shape, generator=g).double()
        num = (f(**(v | {k: v[k] + h * d})) - f(**(v | {k: v[k] - h * d}))) / (2 * h)
        assert abs(num - (leaves[k].grad * d).sum()) < 1e-6 * (1 + abs(num))
