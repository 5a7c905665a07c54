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
into a graph through ``torch.autograd.grad`` after the usual warm-up on a side stream.
"""
from __future__ import annotations

import ctypes
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


def _panel(t: torch.Tensor) -> torch.Tensor:
    """A matrix operand: one unit stride, rows (or columns) that do not overlap, the other stride below 2^22."""
    r, c = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or c == 1) and (r <= 1 or c <= s0 < _MAX_LD):
        return t
    if (s0 == 1 or r == 1) and (c <= 1 or r <= s1 < _MAX_LD):
        return t
    return t.contiguous()


class _On:
    """The tensors' device as the current one (a no-op where it is already), and its current stream."""

    def __init__(self, dev: torch.device):
        self.index = dev.index
        self.prev = torch.cuda.current_device()

    def __enter__(self):
        if self.prev != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)


def _workspace(nbytes: int, dev: torch.device):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------- calls of the C entry points
def _matmul(stream, x, w, *, bias=None, residual=None, act=0, slope=None, low=None, low_mask=False,
            drop=_NO_DROPOUT) -> torch.Tensor:
    """[M, N] of x [M, K] and w [N, K] views through clipvit_linear."""
    L = _lib.lib()
    x, w = _panel(x), _panel(w)
    M, K = x.shape
    N = w.shape[0]
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    a = _lib.LinearArgs()
    a.dtype, a.activation, a.low_mask = _DT[x.dtype], act, int(low_mask)
    a.bias_dtype = a.dtype if bias is None else _DT[bias.dtype]
    a.M, a.N, a.K = M, N, K
    a.x, a.w, a.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
    a.x_stride[0], a.x_stride[1] = x.stride()
    a.w_stride[0], a.w_stride[1] = w.stride()
    a.y_stride = N
    a.bias = _ptr(bias)
    if residual is not None:
        a.residual, a.residual_stride = residual.data_ptr(), residual.stride(0)
    a.slope = _ptr(slope)
    if low is not None:
        u, v = low
        a.R, a.low_u, a.low_v = u.shape[1], u.data_ptr(), v.data_ptr()
    a.dropout = drop
    need = ctypes.c_size_t()
    _lib.check(L.clipvit_linear_workspace(_byref(a), _byref(need)))
    ws = _workspace(need.value, x.device)
    _lib.check(L.clipvit_linear(stream, _byref(a), _ptr(ws), need.value))
    return y


def _dz(stream, dy, slope, drop, want_dz: bool, db_dtype):
    """(dz or None, db or None) of dy [M, N] through clipvit_linear_dz."""
    M, N = dy.shape
    ld = (N + 7) // 8 * 8  # rows that 16-byte loads can address, whatever N is
    dz = torch.empty((M, ld), dtype=dy.dtype, device=dy.device)[:, :N] if want_dz else None
    db = torch.empty(N, dtype=db_dtype, device=dy.device) if db_dtype is not None else None
    a = _lib.DzArgs()
    a.dtype = _DT[dy.dtype]
    a.db_dtype = a.dtype if db is None else _DT[db_dtype]
    a.M, a.N, a.dy, a.dy_stride = M, N, dy.data_ptr(), dy.stride(0)
    a.slope, a.dz, a.dz_stride, a.db, a.dropout = _ptr(slope), _ptr(dz), ld, _ptr(db), drop
    need = 4 * N * min(512, (M + 63) // 64) if db is not None else 0
    ws = _workspace(need, dy.device)
    _lib.check(_lib.lib().clipvit_linear_dz(stream, _byref(a), _ptr(ws), need))
    return dz, db


def _pad(stream, *factors):
    """Zero-padded contiguous copies of one or two 16-bit factors: (view, rows, cols) each."""
    out, args = [], []
    for t, rows, cols in factors:
        d = torch.empty((rows, cols), dtype=t.dtype, device=t.device)
        out.append(d)
        args.append(_lib.PadArgs(t.data_ptr(), t.stride(0), t.stride(1), t.shape[0], t.shape[1], rows, cols, d.data_ptr()))
    _lib.check(_lib.lib().clipvit_lora_pad(stream, _byref(args[0]), _byref(args[1]) if len(args) > 1 else None))
    return out


def _down(stream, x, f, alpha: float, drop) -> torch.Tensor:
    """u [M, R] = alpha mask(x) f^T."""
    M, K = x.shape
    u = torch.empty((M, f.shape[0]), dtype=x.dtype, device=x.device)
    _lib.check(_lib.lib().clipvit_lora_down(stream, _DT[x.dtype], x.data_ptr(), x.stride(0), f.data_ptr(), f.stride(0),
                                            u.data_ptr(), M, K, f.shape[0], alpha, _byref(drop)))
    return u


def _low_grad(stream, x, u, rank: int, transposed: bool, drop) -> torch.Tensor:
    """[C, rank] (or [rank, C]) = mask(x)^T u."""
    L = _lib.lib()
    M, C = x.shape
    R = u.shape[1]
    out = torch.empty((rank, C) if transposed else (C, rank), dtype=x.dtype, device=x.device)
    need = ctypes.c_size_t()
    _lib.check(L.clipvit_lora_grad_workspace(M, C, R, _byref(need)))
    ws = _workspace(need.value, x.device)
    sc, sr = (1, C) if transposed else (rank, 1)
    _lib.check(L.clipvit_lora_grad(stream, _DT[x.dtype], x.data_ptr(), x.stride(0), u.data_ptr(), out.data_ptr(), sc, sr,
                                   M, C, R, rank, _byref(drop), _ptr(ws), need.value))
    return out


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------- linear
def _linear_forward(x2, weight, bias, res2, act, p, seed, offset, save):
    with _On(x2.device) as stream:
        slope = None
        if save and act:
            slope = torch.empty((x2.shape[0], weight.shape[0]), dtype=torch.int16, device=x2.device)
        y = _matmul(stream, x2, weight, bias=bias, residual=res2, act=act, slope=slope,
                    drop=_dropout_args(p, seed, offset))
    return y, slope


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, p, seed, offset):
        x2 = _rows(x)
        res2 = None if residual is None else _rows(residual)
        save = ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        y, slope = _linear_forward(x2, weight, bias, res2, act, p, seed, offset, save)
        ctx.save_for_backward(x, weight, slope, offset if torch.is_tensor(offset) else None)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.p, ctx.seed, ctx.offset = p, seed, None if torch.is_tensor(offset) else offset
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, slope, off = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if nx or nw or nb:
            x2, dy2 = _rows(x), _rows(dy)
            drop = _dropout_args(ctx.p, ctx.seed, ctx.offset if off is None else off)
            with _On(x.device) as stream:
                dz = dy2
                changed = slope is not None or ctx.p > 0.0
                if nb or changed:
                    dz, db = _dz(stream, dy2, slope, drop, changed and (nx or nw), ctx.bias_dtype if nb else None)
                    dz = dy2 if dz is None else dz
                if nx:
                    dx = _matmul(stream, dz, weight.t()).view(x.shape)
                if nw:
                    dw = _matmul(stream, dz.t(), x2.t())
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
        return _Linear.apply(x, weight, bias, residual, act, p, seed, offset)
    y, _ = _linear_forward(_rows(x), weight, bias, None if residual is None else _rows(residual), act, p, seed, offset, False)
    return y.view(*x.shape[:-1], n)


# ---------------------------------------------------------------- dropout
def _dropout_call(x, residual, p, seed, offset):
    x2 = _rows(x)
    res2 = None if residual is None else _rows(residual)
    y = torch.empty(x2.shape, dtype=x.dtype, device=x.device)
    with _On(x.device) as stream:
        _lib.check(_lib.lib().clipvit_dropout(
            stream, _DT[x.dtype], x2.data_ptr(), x2.stride(0), _ptr(res2), 0 if res2 is None else res2.stride(0), y.data_ptr(),
            y.stride(0), x2.shape[0], x2.shape[1], _byref(_dropout_args(p, seed, offset))))
    return y.view(x.shape)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.save_for_backward(offset if torch.is_tensor(offset) else None)
        ctx.p, ctx.seed, ctx.offset = p, seed, None if torch.is_tensor(offset) else offset
        return _dropout_call(x, residual, p, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (off,) = ctx.saved_tensors
        dx = _dropout_call(dy, None, ctx.p, ctx.seed, ctx.offset if off is None else off) if ctx.needs_input_grad[0] else None
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
        return _Dropout.apply(x, residual, p, seed, offset)
    return _dropout_call(x, residual, p, seed, offset)


# ---------------------------------------------------------------- LoRA linear
def _up32(n: int) -> int:
    return (n + 31) // 32 * 32


def _lora_forward(x2, weight, A, B, bias, scaling, p, seed, offset):
    R = _up32(A.shape[1])
    with _On(x2.device) as stream:
        f, v = _pad(stream, (A.t(), R, _up32(A.shape[0])), (B.t(), B.shape[1], R))
        keep = 1.0 / (1.0 - p) if p < 1.0 else 0.0
        u = _down(stream, x2, f, scaling * keep, _dropout_args(p, seed, offset))
        y = _matmul(stream, x2, weight, bias=bias, low=(u, v))
    return y, u


class _LoraLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, A, B, bias, scaling, p, seed, offset):
        y, u = _lora_forward(_rows(x), weight, A, B, bias, scaling, p, seed, offset)
        ctx.save_for_backward(x, weight, A, B, u, offset if torch.is_tensor(offset) else None)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.scaling, ctx.p, ctx.seed, ctx.offset = scaling, p, seed, None if torch.is_tensor(offset) else offset
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, A, B, u, off = ctx.saved_tensors
        nx, nw, nA, nB, nb = ctx.needs_input_grad[:5]
        dx = dw = dA = dB = db = None
        x2, dy2 = _rows(x), _rows(dy)
        (K, rank), N, R = A.shape, weight.shape[0], u.shape[1]
        drop = _dropout_args(ctx.p, ctx.seed, ctx.offset if off is None else off)
        with _On(x.device) as stream:
            if nx or nA:
                f, v = _pad(stream, (B, R, _up32(N)), (A, K, R))
                keep = 1.0 / (1.0 - ctx.p) if ctx.p < 1.0 else 0.0
                du = _down(stream, dy2, f, ctx.scaling * keep, _NO_DROPOUT)
                if nx:
                    dx = _matmul(stream, dy2, weight.t(), low=(du, v), low_mask=True, drop=drop).view(x.shape)
                if nA:
                    dA = _low_grad(stream, x2, du, rank, False, drop)
            if nB:
                dB = _low_grad(stream, dy2, u, rank, True, _NO_DROPOUT)
            if nw:
                dw = _matmul(stream, dy2.t(), x2.t())
            if nb:
                _, db = _dz(stream, dy2, None, _NO_DROPOUT, False, ctx.bias_dtype)
        return dx, dw, dA, dB, db, None, None, None, None


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
        return _LoraLinear.apply(x, weight, lora_A, lora_B, bias, float(scaling), p, seed, offset)
    return _lora_forward(_rows(x), weight, lora_A, lora_B, bias, float(scaling), p, seed, offset)[0].view(*x.shape[:-1], n)
