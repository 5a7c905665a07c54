"""Fine-tuning operators on 16-bit device tensors: a Linear with its epilogue, counter-based dropout and
the unmerged LoRA Linear, each differentiable.

The reference trains its adapters on ``LoRALinear`` modules (main.py:34-59, train_lora.py:62-100), which
:mod:`lora` only merges; these are that Linear's forward and gradients, in hand-written gfx950 kernels
(csrc/matmul.hip, csrc/finetune.hip, the ``clipvit_linear`` family of include/clipvit.h):

* ``linear(x, weight, bias, residual, activation=, dropout_p=, seed=, offset=)``
  = residual + dropout(act(x weight^T + bias));
* ``dropout(x, p, seed=, offset=, residual=)`` = residual + dropout(x), the mask never stored;
* ``lora_linear(x, weight, lora_A, lora_B, bias, scaling=, dropout_p=, ...)``
  = x weight^T + bias + scaling (dropout(x) lora_A) lora_B  (main.py:30-31, 42-43).

Matrix operands are bf16 or fp16 (one type per call), accumulated in fp32 and rounded once into the output;
a gradient that passes an activation or a dropout rounds dz to the operands' type before its products, as
the MFMA takes it. ``offset`` is an int, or a one-element int64 device tensor that the kernels read when they
run: under a captured graph, change it between replays and every replay draws its own mask. It must not
change between a forward and its backward (autograd raises if it does). ``seed`` and ``offset`` together
name the mask: calls that share both (and the row count) share their masks.

Every call runs on the current stream of the tensors' device and allocates its output and workspace from torch's
caching allocator. There is no CPU fallback: CPU tensors raise ``ClipVitError``. A backward may be captured
into a graph through ``torch.autograd.grad`` after the usual warm-up on a side stream, once no eager autograd graph of
the same leaves is alive (a capture that finds one raises). Matrices of more than one row hold fewer than 2^22 columns.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
ACTIVATIONS = {"none": 0, "quick_gelu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "relu": 5}
_byref = ctypes.byref
_MASK64 = (1 << 64) - 1


# ---------------------------------------------------------------- arguments
def _need_device(*tensors) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
    if dev.type != "cuda":
        raise _lib.ClipVitError(_lib.E_STATE, "the MI355X operators run on a HIP device ('cuda:N' in PyTorch-ROCm)")
    return dev


def _same16(name: str, dtype: torch.dtype, **tensors) -> None:
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name}: x must be bfloat16 or float16, got {dtype}")
    for key, t in tensors.items():
        if t is not None and t.dtype != dtype:
            raise TypeError(f"{name}: {key} must be {dtype} like x, got {t.dtype}")


def _check_bias(name: str, bias, n: int, dtype: torch.dtype) -> None:
    if bias is None:
        return
    if bias.dtype not in (dtype, torch.float32):
        raise TypeError(f"{name}: bias must be {dtype} or float32, got {bias.dtype}")
    if tuple(bias.shape) != (n,):
        raise ValueError(f"{name}: bias must be [{n}], got {tuple(bias.shape)}")


def _check_p(p) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    return p


def _check_counter(seed, offset, x: torch.Tensor) -> None:
    if not isinstance(seed, int):
        raise TypeError(f"seed must be an int, got {type(seed).__name__}")
    if torch.is_tensor(offset):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise TypeError("a tensor offset must hold one int64")
        if offset.device != x.device:
            raise ValueError(f"offset on {offset.device}, x on {x.device}")
    elif not isinstance(offset, int):
        raise TypeError(f"offset must be an int or an int64 tensor, got {type(offset).__name__}")


def _dropout_args(p: float, seed: int, offset) -> _lib.DropoutArgs:
    if torch.is_tensor(offset):
        return _lib.DropoutArgs(p, seed & _MASK64, 0, offset.data_ptr())
    return _lib.DropoutArgs(p, seed & _MASK64, offset & _MASK64, None)


_NO_DROPOUT = _lib.DropoutArgs(0.0, 0, 0, None)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., n] as [rows, n] with unit column stride and rows that do not overlap (a copy only where the
    strides are something else)."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


_MAX_LD = 1 << 22


def _rows_ld(t: torch.Tensor) -> torch.Tensor:
    """_rows with a row stride that the matrix products address (below 2^22, or one row)."""
    t = _rows(t)
    return t.contiguous() if t.shape[0] > 1 and t.stride(0) >= _MAX_LD else t


def _panel(t: torch.Tensor) -> torch.Tensor:
    """A matrix operand: one unit stride, rows (or columns) that do not overlap, the other stride below 2^22."""
    r, c = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or c == 1) and (r <= 1 or c <= s0 < _MAX_LD):
        return t
    if (s0 == 1 or r == 1) and (c <= 1 or r <= s1 < _MAX_LD):
        return t
    return t.contiguous()


def _stream(index: int):
    """The current stream of a device as the C entry points take it."""
    return torch._C._cuda_getCurrentRawStream(index)


class _On:
    """The tensors' device as the current one while kernels are launched; entered only where it is not already."""

    def __init__(self, index: int):
        self.index, self.prev = index, torch.cuda.current_device()

    def __enter__(self):
        torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        torch.cuda.set_device(self.prev)


def _launch(name: str, index: int, args, ws, nbytes: int) -> None:
    """One C call on the current stream of device `index`."""
    fn = getattr(_lib.lib(), name)
    ptr = ws.data_ptr() if nbytes else None
    if torch.cuda.current_device() == index:
        rc = fn(_stream(index), _byref(args), ptr, nbytes)
    else:
        with _On(index):
            rc = fn(_stream(index), _byref(args), ptr, nbytes)
    if rc:
        _lib.check(rc)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _bytes(name: str, args) -> int:
    need = ctypes.c_size_t()
    _lib.check(getattr(_lib.lib(), name)(_byref(args), _byref(need)))
    return need.value


# Workspace sizes by sizes, strides, alignments and wanted outputs, which is all they depend on (pointers are
# stand-ins of the same alignment).
@functools.lru_cache(maxsize=4096)
def _linear_bytes(dt, m, n, k, x0, x1, xa, w0, w1, wa) -> int:
    return _bytes("clipvit_linear_workspace", _lib.LinearArgs(
        dt, 0, dt, 0, m, n, k, 4096 + xa, x0, x1, 4096 + wa, w0, w1, None, None, 0, 4096, n, None, _NO_DROPOUT))


@functools.lru_cache(maxsize=4096)
def _linear_grad_bytes(dt, bdt, m, n, k, d0, da, x0, x1, xa, w0, w1, wa, slope, dx, dw, db, p) -> int:
    return _bytes("clipvit_linear_grad_workspace", _lib.LinearGradArgs(
        dt, bdt, m, n, k, 4096 + da, d0, 4096 + xa, x0, x1, 4096 + wa, w0, w1, 4096 if slope else None,
        4096 if dx else None, 4096 if dw else None, 4096 if db else None, _lib.DropoutArgs(p, 0, 0, None)))


@functools.lru_cache(maxsize=4096)
def _lora_bytes(dt, m, n, k, r, x0, xa, w0, w1, wa) -> int:
    return _bytes("clipvit_lora_linear_workspace", _lib.LoraArgs(
        dt, dt, m, n, k, r, 4096 + xa, x0, 4096 + wa, w0, w1, 4096, r, 1, 4096, n, 1, None, 4096, 4096, 1.0, 0.0, _NO_DROPOUT))


@functools.lru_cache(maxsize=4096)
def _lora_grad_bytes(dt, bdt, m, n, k, r, d0, da, x0, xa, w0, w1, wa, dx, dw, dA, dB, db, p) -> int:
    return _bytes("clipvit_lora_linear_grad_workspace", _lib.LoraGradArgs(
        dt, bdt, m, n, k, r, 4096 + da, d0, 4096 + xa, x0, 4096 + wa, w0, w1, 4096, r, 1, 4096, n, 1, 4096,
        4096 if dx else None, 4096 if dw else None, 4096 if dA else None, 4096 if dB else None, 4096 if db else None, 1.0, 0.0,
        _lib.DropoutArgs(p, 0, 0, None)))


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _differentiable(fn, args, leaves):
    """fn.apply(*args), with the stream noted at the gradient nodes of the leaves among `leaves`.

    A leaf's gradient node keeps the stream of the graph that it was made for, for as long as one of its graphs lives. A
    backward pass captured on another stream would draw that stream into the capture, which ends the process, so such
    a capture is refused here, before anything is recorded."""
    stream = _stream(args[0].device.index)
    if torch.cuda.is_current_stream_capturing():
        for t in leaves:
            if t is None or not t.requires_grad or not t.is_leaf:
                continue
            if torch.autograd.graph.get_gradient_edge(t).node.metadata.get("interior_amd", stream) != stream:
                raise RuntimeError("a graph capture would differentiate a leaf whose earlier autograd graph, made on another stream, "
                                   "is still alive: delete that graph's outputs (or run it on the capturing stream) first")
    y = fn.apply(*args)
    for node, _ in y.grad_fn.next_functions:  # (after the call: now the new graph holds the nodes)
        if node is not None:
            node.metadata.setdefault("interior_amd", stream)
    return y


# ---------------------------------------------------------------- linear
def _linear_forward(x2, w, bias, res2, act, drop, save):
    """(y [M, N], act'(z) or None, the operands' description) of x2 [M, K], w [N, K] as _panel gives them."""
    (m, k), n, dt, dev = x2.shape, w.shape[0], _DT[x2.dtype], x2.device
    (x0, x1), (w0, w1), xp, wp = x2.stride(), w.stride(), x2.data_ptr(), w.data_ptr()
    y = x2.new_empty((m, n))
    slope = torch.empty((m, n), dtype=torch.int16, device=dev) if save and act else None
    need = _linear_bytes(dt, m, n, k, x0, x1, xp & 15, w0, w1, wp & 15)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _launch("clipvit_linear", dev.index, _lib.LinearArgs(
        dt, act, dt if bias is None else _DT[bias.dtype], 0, m, n, k, xp, x0, x1, wp, w0, w1, _ptr(bias), _ptr(res2),
        0 if res2 is None else res2.stride(0), y.data_ptr(), n, _ptr(slope), drop), ws, need)
    return y, slope, (dt, m, n, k, x0, x1, w0, w1)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, p, seed, offset):
        needs = ctx.needs_input_grad
        drop = _dropout_args(p, seed, offset)
        x2, w = _panel(_rows(x)), _panel(weight)
        y, slope, ctx.meta = _linear_forward(x2, w, bias, None if residual is None else _rows(residual), act, drop,
                                             needs[0] or needs[1] or needs[2])
        # (the offset is saved so that autograd notices when it changes before the backward pass)
        ctx.save_for_backward(x2, w, slope, offset if torch.is_tensor(offset) else None)
        ctx.drop, ctx.bias_dtype, ctx.x_shape = drop, None if bias is None else bias.dtype, x.shape
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w, slope, _ = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if nx or nw or nb:
            dy2 = _rows_ld(dy)
            (dt, m, n, k, x0, x1, w0, w1), drop, dev = ctx.meta, ctx.drop, x2.device
            d0, xp, wp, dp = dy2.stride(0), x2.data_ptr(), w.data_ptr(), dy2.data_ptr()
            dx = x2.new_empty((m, k)) if nx else None
            dw = x2.new_empty((n, k)) if nw else None
            db = torch.empty(n, dtype=ctx.bias_dtype, device=dev) if nb else None
            bdt = _DT[ctx.bias_dtype] if nb else dt
            need = _linear_grad_bytes(dt, bdt, m, n, k, d0, dp & 15, x0, x1, xp & 15, w0, w1, wp & 15, slope is not None, nx, nw, nb, drop.p)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            _launch("clipvit_linear_grad", dev.index, _lib.LinearGradArgs(
                dt, bdt, m, n, k, dp, d0, xp, x0, x1, wp, w0, w1, _ptr(slope), _ptr(dx), _ptr(dw), _ptr(db), drop), ws, need)
            if nx:
                dx = dx.view(ctx.x_shape)
        return dx, dw, db, dy if nr else None, None, None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, *, activation: str = "none", dropout_p: float = 0.0,
           seed: int = 0, offset=0) -> torch.Tensor:
    """residual + dropout(act(x weight^T + bias)): x [..., K], weight [N, K] -> [..., N] of x's type.

    x, weight and residual are bf16 or fp16; bias is of that type or fp32. ``weight`` may be any view with one
    unit stride (a [K, N] factor is passed as ``factor.t()``). ``activation``: none, quick_gelu, gelu, gelu_tanh,
    silu or relu. The dropout mask is that of ``dropout`` on the [rows, N] output. Differentiable in x, weight,
    bias and residual (main.py:34-59 is the reference's Linear under training)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; one of {sorted(ACTIVATIONS)}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x [..., K] and weight [N, K] do not match: {tuple(x.shape)}, {tuple(weight.shape)}")
    n = weight.shape[0]
    _same16("linear", x.dtype, weight=weight, residual=residual)
    _check_bias("linear", bias, n, x.dtype)
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise ValueError(f"linear: residual must be {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
    p = _check_p(dropout_p)
    _check_counter(seed, offset, x)
    _need_device(x, weight, bias, residual)
    act = ACTIVATIONS[activation]
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    if _wants_grad(x, weight, bias, residual):
        return _differentiable(_Linear, (x, weight, bias, residual, act, p, seed, offset), (x, weight, bias, residual))
    y = _linear_forward(_panel(_rows(x)), _panel(weight), bias, None if residual is None else _rows(residual), act,
                        _dropout_args(p, seed, offset) if p else _NO_DROPOUT, False)[0]
    return y.view(*x.shape[:-1], n)


# ---------------------------------------------------------------- dropout
def _dropout_call(x, residual, drop):
    x2 = _rows(x)
    res2 = None if residual is None else _rows(residual)
    y, index = torch.empty(x2.shape, dtype=x.dtype, device=x.device), x.device.index
    args = (_DT[x.dtype], x2.data_ptr(), x2.stride(0), _ptr(res2), 0 if res2 is None else res2.stride(0), y.data_ptr(), y.stride(0),
            x2.shape[0], x2.shape[1], _byref(drop))
    if torch.cuda.current_device() == index:
        rc = _lib.lib().clipvit_dropout(_stream(index), *args)
    else:
        with _On(index):
            rc = _lib.lib().clipvit_dropout(_stream(index), *args)
    if rc:
        _lib.check(rc)
    return y.view(x.shape)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.drop = _dropout_args(p, seed, offset)
        ctx.save_for_backward(offset if torch.is_tensor(offset) else None)
        return _dropout_call(x, residual, ctx.drop)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ctx.saved_tensors  # raises where a tensor offset changed since the forward pass
        dx = _dropout_call(dy, None, ctx.drop) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, *, seed: int, offset=0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """residual + dropout(x): fp32, bf16 or fp16 of any shape; the last dimension is the mask's column, the others
    together its row. Kept elements are scaled by 1 / (1 - p), dropped ones are exactly 0 (NaN included). The
    backward pass computes the mask again from (seed, offset). Differentiable in x and residual."""
    if x.dtype not in _DT:
        raise TypeError(f"dropout: x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("dropout: x needs at least one dimension")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError(f"dropout: residual must be {tuple(x.shape)} of {x.dtype}, got {tuple(residual.shape)} of {residual.dtype}")
    p = _check_p(p)
    _check_counter(seed, offset, x)
    _need_device(x, residual)
    if _wants_grad(x, residual):
        return _differentiable(_Dropout, (x, residual, p, seed, offset), (x, residual))
    return _dropout_call(x, residual, _dropout_args(p, seed, offset))


# ---------------------------------------------------------------- LoRA linear
def _lora_forward(x2, w, A, B, bias, scaling, drop):
    """(y [M, N], u [M, rank rounded up to 32], the operands' description) of x2 [M, K] rows, w [N, K] as _panel gives it."""
    (m, k), n, r, dt, dev = x2.shape, w.shape[0], A.shape[1], _DT[x2.dtype], x2.device
    x0, (w0, w1), xp, wp = x2.stride(0), w.stride(), x2.data_ptr(), w.data_ptr()
    y, u = x2.new_empty((m, n)), x2.new_empty((m, (r + 31) // 32 * 32))
    need = _lora_bytes(dt, m, n, k, r, x0, xp & 15, w0, w1, wp & 15)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _launch("clipvit_lora_linear", dev.index, _lib.LoraArgs(
        dt, dt if bias is None else _DT[bias.dtype], m, n, k, r, xp, x0, wp, w0, w1, A.data_ptr(), A.stride(0), A.stride(1),
        B.data_ptr(), B.stride(0), B.stride(1), _ptr(bias), y.data_ptr(), u.data_ptr(), scaling, 0.0, drop), ws, need)
    return y, u, (dt, m, n, k, r, x0, w0, w1)


class _LoraLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, A, B, bias, scaling, p, seed, offset):
        drop = _dropout_args(p, seed, offset)
        x2, w = _rows_ld(x), _panel(weight)
        y, u, ctx.meta = _lora_forward(x2, w, A, B, bias, scaling, drop)
        ctx.save_for_backward(x2, w, A, B, u, offset if torch.is_tensor(offset) else None)
        ctx.drop, ctx.scaling, ctx.bias_dtype, ctx.x_shape = drop, scaling, None if bias is None else bias.dtype, x.shape
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w, A, B, u, _ = ctx.saved_tensors
        nx, nw, nA, nB, nb = ctx.needs_input_grad[:5]
        dy2 = _rows_ld(dy)
        (dt, m, n, k, r, x0, w0, w1), drop, dev = ctx.meta, ctx.drop, x2.device
        d0, xp, wp, dp = dy2.stride(0), x2.data_ptr(), w.data_ptr(), dy2.data_ptr()
        dx = x2.new_empty((m, k)) if nx else None
        dw = x2.new_empty((n, k)) if nw else None
        dA = x2.new_empty((k, r)) if nA else None
        dB = x2.new_empty((r, n)) if nB else None
        db = torch.empty(n, dtype=ctx.bias_dtype, device=dev) if nb else None
        bdt = _DT[ctx.bias_dtype] if nb else dt
        need = _lora_grad_bytes(dt, bdt, m, n, k, r, d0, dp & 15, x0, xp & 15, w0, w1, wp & 15, nx, nw, nA, nB, nb, drop.p)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _launch("clipvit_lora_linear_grad", dev.index, _lib.LoraGradArgs(
            dt, bdt, m, n, k, r, dp, d0, xp, x0, wp, w0, w1, A.data_ptr(), A.stride(0), A.stride(1), B.data_ptr(), B.stride(0),
            B.stride(1), u.data_ptr(), _ptr(dx), _ptr(dw), _ptr(dA), _ptr(dB), _ptr(db), ctx.scaling, 0.0, drop), ws, need)
        return dx if dx is None else dx.view(ctx.x_shape), dw, dA, dB, db, None, None, None, None


def lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_A: torch.Tensor, lora_B: torch.Tensor,
                bias: torch.Tensor | None = None, *, scaling: float = 1.0, dropout_p: float = 0.0, seed: int = 0,
                offset=0) -> torch.Tensor:
    """x weight^T + bias + scaling (dropout(x) lora_A) lora_B: the reference's LoRALinear (main.py:30-31, 42-43), unmerged.

    x [..., K], weight [N, K], lora_A [K, r], lora_B [r, N] (the checkpoint layout), all bf16 or fp16 of one type;
    scaling = alpha / r (main.py:28). The thin product dropout(x) lora_A is rounded to that type once (it is an
    MFMA operand), the adapter's term is added in fp32 before the output's rounding. Differentiable in x, weight,
    lora_A, lora_B and bias."""
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"lora_linear: x [..., K] and weight [N, K] do not match: {tuple(x.shape)}, {tuple(weight.shape)}")
    n, k = weight.shape
    if lora_A.dim() != 2 or lora_B.dim() != 2 or lora_A.shape[0] != k or lora_B.shape[1] != n or lora_A.shape[1] != lora_B.shape[0]:
        raise ValueError(f"lora_linear: lora_A [{k}, r] and lora_B [r, {n}] expected, got {tuple(lora_A.shape)}, {tuple(lora_B.shape)}")
    if not 1 <= lora_A.shape[1] <= 65536:
        raise ValueError(f"lora_linear: rank must lie in [1, 65536], got {lora_A.shape[1]}")
    _same16("lora_linear", x.dtype, weight=weight, lora_A=lora_A, lora_B=lora_B)
    _check_bias("lora_linear", bias, n, x.dtype)
    p = _check_p(dropout_p)
    _check_counter(seed, offset, x)
    _need_device(x, weight, lora_A, lora_B, bias)
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    if _wants_grad(x, weight, lora_A, lora_B, bias):
        return _differentiable(_LoraLinear, (x, weight, lora_A, lora_B, bias, float(scaling), p, seed, offset),
                               (x, weight, lora_A, lora_B, bias))
    return _lora_forward(_rows_ld(x), _panel(weight), lora_A, lora_B, bias, float(scaling), _dropout_args(p, seed, offset))[0].view(
        *x.shape[:-1], n)
