"""Operators of a layer with FP8 weights, around and of its matrix products:
the root-mean-square norm with the residual's addition and an 8-bit output,
the rounding of rows to 8 bits, and the product of 8-bit rows with FP8 weights
with bias, activation, gate and residual in its epilogue.  No counterpart in
the reference.

8-bit values are E4M3FN bytes (uint8) with one float32 scale per row.  These
are inference operators: they have no backward, and inputs that require a
gradient are refused.  Errors raise RuntimeError.  Kernels run on the current
torch stream of the inputs' device; scratch memory comes from torch's caching
allocator.
"""
from __future__ import annotations

import ctypes

import torch

from ._C import _check_dev, _on, _ptr, _require, _stream
from ._lib import check, lib

__all__ = ["ACTIVATIONS", "fp8_linear", "fp8_quantize_rows", "fp8_rmsnorm"]

# name -> TANS_ACT_*
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _check_in(name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    _check_dev(name, t, dtype)
    _require(not (t.requires_grad and torch.is_grad_enabled()),
             f"{name} requires a gradient; the layer operators have no backward")


def _rows(name: str, x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """x [D] or [M, D] -> x [M, D]."""
    _check_in(name, x, dtype)
    _require(x.dim() in (1, 2), f"{name} must be [D] or [M, D]")
    x2 = x.view(1, -1) if x.dim() == 1 else x
    _require(x2.shape[1] >= 16 and x2.shape[1] % 16 == 0,
             f"the columns of {name} must be a multiple of 16")
    return x2


def _opt(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def fp8_rmsnorm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                eps: float = 1e-6):
    """h = x + residual, y = h * weight / sqrt(mean(h^2) + eps), rounded to 8
    bits -> (q uint8 like x, scale float32 [M] or [], h bf16 like x).

    x, residual: bf16 [D] or [M, D], D a multiple of 16; weight bf16 [D].
    scale = max(max |y| of the row, 2^-100) / 448 and q = E4M3FN(y / scale).
    The norm is taken of the sum in 32 bits; h is that sum as bf16 (without
    residual: x itself)."""
    x2 = _rows("x", x, torch.bfloat16)
    M, D = x2.shape
    _check_in("weight", weight, torch.bfloat16)
    _require(weight.dim() == 1 and weight.numel() == D, f"weight must be [{D}]")
    dev = x.device
    _require(weight.device == dev, "all tensors must be on one device")
    _require(eps >= 0.0, "eps must not be negative")
    h = x
    if residual is not None:
        _check_in("residual", residual, torch.bfloat16)
        _require(residual.shape == x.shape, "residual must have the shape of x")
        _require(residual.device == dev, "all tensors must be on one device")
        h = torch.empty_like(x)
    q = torch.empty(x.shape, dtype=torch.uint8, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    with _on(dev):
        check(lib.tans_fp8_rmsnorm(_ptr(x), _opt(residual), _ptr(weight), M, D, float(eps), _ptr(q),
                                   _ptr(scale), _ptr(h), _stream(dev)), "fp8_rmsnorm")
    return q, scale, h


def fp8_quantize_rows(x: torch.Tensor):
    """Rows of bf16 x [D] or [M, D] to 8 bits -> (q uint8 like x, scale float32
    [M] or []): scale = max(max |x| of the row, 2^-100) / 448, q =
    E4M3FN(x / scale).  D a multiple of 16."""
    x2 = _rows("x", x, torch.bfloat16)
    M, D = x2.shape
    dev = x.device
    q = torch.empty(x.shape, dtype=torch.uint8, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    with _on(dev):
        check(lib.tans_fp8_quantize_rows(_ptr(x), M, D, _ptr(q), _ptr(scale), _stream(dev)),
              "fp8_quantize_rows")
    return q, scale


def fp8_linear(a: torch.Tensor, a_scale: torch.Tensor | None, w: torch.Tensor,
               w_scale: torch.Tensor | float = 1.0, *, bias: torch.Tensor | None = None,
               activation: str = "none", residual: torch.Tensor | None = None,
               gated: bool = False) -> torch.Tensor:
    """y = act(a_scale * w_scale * (a @ w^T) + bias) + residual as bf16, from
    E4M3FN bytes on both sides; one kernel does the product and its epilogue.

    a uint8 [C] or [M, C] (any M), C a multiple of 16; a_scale float32 [M] (or
    []) or None; w uint8 [R, C]; w_scale float32 [R] or a number; bias bf16 [R];
    activation one of "none", "relu", "silu", "gelu" (x Phi(x)), "gelu_tanh".
    gated: w's first R / 2 rows are the gate's, the others the value's, and
    y = act(gate) * value + residual.  residual bf16 and y are [M, R], gated
    [M, R / 2] ([R], [R / 2] for a [C]).  32-bit accumulation in a fixed order,
    one rounding."""
    a2 = _rows("a", a, torch.uint8)
    M, C = a2.shape
    _check_in("w", w, torch.uint8)
    _require(w.dim() == 2 and w.shape[0] >= 1 and w.shape[1] == C, f"w must be [R, C] with C = {C}")
    R = w.shape[0]
    _require(activation in ACTIVATIONS, f"activation must be one of {sorted(ACTIVATIONS)}")
    _require(not gated or R % 2 == 0, "a gated product needs an even number of rows of w")
    N = R // 2 if gated else R
    shape = a.shape[:-1] + (N,)
    dev = a.device
    scale = 1.0
    if isinstance(w_scale, torch.Tensor):
        _check_in("w_scale", w_scale, torch.float32)
        _require(w_scale.shape == (R,), f"w_scale must be a number or [{R}]")
    else:
        scale, w_scale = float(w_scale), None
    if a_scale is not None:
        _check_in("a_scale", a_scale, torch.float32)
        _require(a_scale.shape == a.shape[:-1], "a_scale must hold one scale per row of a")
    if bias is not None:
        _check_in("bias", bias, torch.bfloat16)
        _require(bias.shape == (R,), f"bias must be [{R}]")
    if residual is not None:
        _check_in("residual", residual, torch.bfloat16)
        _require(residual.shape == shape, f"residual must be {list(shape)}")
    for t in (w, a_scale, w_scale, bias, residual):
        _require(t is None or t.device == dev, "all tensors must be on one device")
    y = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    with _on(dev):
        need = ctypes.c_int64()
        check(lib.tans_fp8_linear_workspace(M, R, C, int(gated), ctypes.byref(need)), "fp8_linear")
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
        check(lib.tans_fp8_linear(_ptr(a), _opt(a_scale), _ptr(w), _opt(w_scale), scale, _opt(bias),
                                  _opt(residual), ACTIVATIONS[activation], int(gated), M, R, C,
                                  _opt(ws), need.value, _ptr(y), _stream(dev)), "fp8_linear")
    return y
