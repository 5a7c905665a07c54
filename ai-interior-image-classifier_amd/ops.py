"""Fine-tuning operators on 16-bit device tensors: a Linear with its epilogue, counter-based dropout and
the unmerged LoRA Linear, each differentiable.

The reference trains its adapters on ``LoRALinear`` modules (main.py:34-59, train_lora.py:62-100), which
:mod:`lora` only merges; these are that Linear's forward and gradients, in hand-written gfx950 kernels
(csrc/matmul.hip, csrc/finetune.hip, the ``clipvit_linear`` family of include/clipvit.h) behind native autograd
nodes (csrc/ops_torch.cpp):

* ``linear(x, weight, bias, residual, activation=, dropout_p=, seed=, offset=)``
  = residual + dropout(act(x weight^T + bias));
* ``dropout(x, p, seed=, offset=, residual=)`` = residual + dropout(x), the mask never stored;
* ``lora_linear(x, weight, lora_A, lora_B, bias, scaling=, dropout_p=, ...)``
  = x weight^T + bias + scaling (dropout(x) lora_A) lora_B  (main.py:30-31, 42-43).

Matrix operands are bf16 or fp16 (one type per call), accumulated in fp32 and rounded once into the output;
a gradient that passes an activation or a dropout rounds dz to the operands' type before its products, as
the MFMA takes it. ``offset`` is an int, or a one-element int64 device tensor that the kernels read when they
run: under a captured graph, change it between replays and every replay draws its own mask. It must not
change between a forward and a backward that draws the mask again (autograd raises if it does). ``seed`` and ``offset`` together
name the mask: calls that share both (and the row count) share their masks.

Every call runs on the current stream of the tensors' device and allocates its output and workspace from torch's
caching allocator. There is no CPU fallback: CPU tensors raise ``ClipVitError``. A backward may be captured
into a graph through ``torch.autograd.grad`` after the usual warm-up on a side stream, once no eager autograd graph of
the same leaves is alive (a capture that finds one raises). They are differentiable once (no ``create_graph``), and
keep for the backward pass only what the wanted gradients read: a frozen weight's x, or a frozen x's weight, may change
or be freed after the forward. They run eagerly or in a captured graph and refuse to be traced (``torch.jit.trace``,
``make_fx``). Matrices of more than one row hold fewer than 2^22 columns.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
ACTIVATIONS = {"none": 0, "quick_gelu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "relu": 5}
_MASK64 = (1 << 64) - 1
_binding_module = None


def _binding():
    """The native autograd binding (csrc/ops_torch.cpp), given this process's build of the library."""
    global _binding_module
    if _binding_module is None:
        try:
            from . import _ops_torch as m
        except ImportError as e:
            raise _lib.ClipVitError(_lib.E_STATE, f"_ops_torch.so is not built (run __graft_entry__.build()): {e}") from e
        m.set_library(_entry_points(), _lib.ClipVitError)
        _binding_module = m
    return _binding_module


def _entry_points() -> dict[str, int]:
    """Addresses of what the binding calls: the library's entry points and the capture query of the runtime it is linked to."""
    L = _lib.lib()
    names = [f"clipvit_{n}{w}" for n in ("linear", "linear_grad", "lora_linear", "lora_linear_grad") for w in ("", "_workspace")]
    return {n: ctypes.cast(getattr(L, n), ctypes.c_void_p).value
            for n in (*names, "clipvit_dropout", "clipvit_last_error", "hipStreamIsCapturing")}


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


def _counter(seed: int, offset):
    """(seed, offset, offset tensor or None) as 64-bit words."""
    if torch.is_tensor(offset):
        return seed & _MASK64, 0, offset
    return seed & _MASK64, offset & _MASK64, None


# ---------------------------------------------------------------- linear
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
    return _binding().linear(x, weight, bias, residual, ACTIVATIONS[activation], p, *_counter(seed, offset))


# ---------------------------------------------------------------- dropout
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
    return _binding().dropout(x, residual, p, *_counter(seed, offset))


# ---------------------------------------------------------------- LoRA linear
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
    return _binding().lora_linear(x, weight, lora_A, lora_B, bias, float(scaling), p, *_counter(seed, offset))
