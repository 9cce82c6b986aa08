"""Operators of a layer with FP8 weights, around and of its matrix products:
the root-mean-square norm with the residual's addition and an 8-bit output,
the rounding of rows to 8 bits, and the product of 8-bit rows with FP8 weights
with bias, activation, gate and residual in its epilogue.  No counterpart in
the reference.

8-bit values are E4M3FN bytes (uint8) with one float32 scale per row.  These
are inference operators: they have no backward and no forward-mode derivative,
and inputs that require a gradient or carry a tangent are refused.  Errors raise RuntimeError.  Kernels run on the current
torch stream of the inputs' device; scratch memory comes from torch's caching
allocator.

One row's norm takes the GPU about 4 us, less than Python takes for the call,
so each function tests its arguments in one expression and names what is wrong
only where that fails.
"""
from __future__ import annotations

import ctypes
import functools
import types

import torch
from torch.autograd import forward_ad

from ._C import _check_dev, _on, _require
from ._lib import check, lib

__all__ = ["ACTIVATIONS", "fp8_linear", "fp8_quantize_rows", "fp8_rmsnorm"]

# name -> TANS_ACT_*
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}

_BF16, _U8, _F32 = torch.bfloat16, torch.uint8, torch.float32

# the current stream's handle, 0.1 us in place of the 2 us of a Stream object
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

# the level is -1 outside of dual_level; asking for a tangent takes 0.4 us there
_forward = (forward_ad if hasattr(forward_ad, "_current_level")
            else types.SimpleNamespace(_current_level=0))


def _no_tangents(**tensors) -> None:
    """Raise for the first that forward-mode differentiation follows (no_grad does
    not end it).  Called within a dual level only."""
    for name, t in tensors.items():
        _require(not isinstance(t, torch.Tensor) or forward_ad.unpack_dual(t).tangent is None,
                 f"{name} carries a tangent; the layer operators have no forward-mode derivative")


def _ok(t: torch.Tensor, dtype: torch.dtype, dev: torch.device) -> bool:
    try:
        return (t.dtype is dtype and t.device == dev and t.is_contiguous()
                and not (t.requires_grad and torch.is_grad_enabled()))
    except AttributeError:   # no tensor
        return False


def _explain(name: str, t: torch.Tensor, dtype: torch.dtype, dev: torch.device) -> None:
    """Raise for the first thing that keeps t from being _ok."""
    _require(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _check_dev(name, t, dtype)
    _require(not (t.requires_grad and torch.is_grad_enabled()),
             f"{name} requires a gradient; the layer operators have no backward")
    _require(t.device == dev, "all tensors must be on one device")


def _rows(name: str, x: torch.Tensor, dtype: torch.dtype):
    """(M, D) of x [D] or [M, D]."""
    try:
        shape = x.shape
        fine = (x.is_cuda and _ok(x, dtype, x.device) and 1 <= len(shape) <= 2
                and shape[-1] >= 16 and shape[-1] % 16 == 0)
    except AttributeError:   # no tensor
        fine = False
    if not fine:
        _explain(name, x, dtype, getattr(x, "device", None))
        _require(x.dim() in (1, 2), f"{name} must be [D] or [M, D]")
        _require(False, f"the columns of {name} must be a multiple of 16")
    return (1, shape[0]) if len(shape) == 1 else shape


def _number(name: str, v) -> float:
    try:
        return float(v)
    except (TypeError, ValueError, OverflowError):
        raise RuntimeError(f"{name} must be a number") from None


def _call(dev: torch.device, what: str, fn, *args) -> None:
    """fn(*args, stream) on dev's current stream."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(dev.index))
    else:
        with _on(dev):
            rc = fn(*args, _raw_stream(dev.index))
    if rc:
        check(rc, what)


def fp8_rmsnorm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                eps: float = 1e-6):
    """h = x + residual, y = h * weight / sqrt(mean(h^2) + eps), rounded to 8
    bits -> (q uint8 like x, scale float32 [M] or [], h bf16 like x).

    x, residual: bf16 [D] or [M, D], D a multiple of 16; weight bf16 [D].
    scale = max(max |y| of the row, 2^-100) / 448 and q = E4M3FN(y / scale).
    The norm is taken of the sum in 32 bits, of whatever finite size; h is that
    sum as bf16 (without residual: x itself)."""
    M, D = _rows("x", x, _BF16)
    dev, shape = x.device, x.shape
    if _forward._current_level >= 0:
        _no_tangents(x=x, weight=weight, residual=residual)
    if type(eps) is not float:
        eps = _number("eps", eps)
    if not (_ok(weight, _BF16, dev) and weight.shape == (D,) and eps >= 0.0):
        _explain("weight", weight, _BF16, dev)
        _require(weight.shape == (D,), f"weight must be [{D}]")
        _require(False, "eps must not be negative")
    if residual is None:
        h = x
    else:
        if not (_ok(residual, _BF16, dev) and residual.shape == shape):
            _explain("residual", residual, _BF16, dev)
            _require(False, "residual must have the shape of x")
        h = torch.empty_like(x)
    q = torch.empty_like(x, dtype=_U8)
    scale = torch.empty(M if len(shape) == 2 else (), dtype=_F32, device=dev)
    _call(dev, "fp8_rmsnorm", lib.tans_fp8_rmsnorm, x.data_ptr(),
          None if residual is None else residual.data_ptr(), weight.data_ptr(), M, D, eps,
          q.data_ptr(), scale.data_ptr(), h.data_ptr())
    return q, scale, h


def fp8_quantize_rows(x: torch.Tensor):
    """Rows of bf16 x [D] or [M, D] to 8 bits -> (q uint8 like x, scale float32
    [M] or []): scale = max(max |x| of the row, 2^-100) / 448, q =
    E4M3FN(x / scale).  D a multiple of 16."""
    M, D = _rows("x", x, _BF16)
    dev = x.device
    if _forward._current_level >= 0:
        _no_tangents(x=x)
    q = torch.empty_like(x, dtype=_U8)
    scale = torch.empty(M if x.dim() == 2 else (), dtype=_F32, device=dev)
    _call(dev, "fp8_quantize_rows", lib.tans_fp8_quantize_rows, x.data_ptr(), M, D, q.data_ptr(),
          scale.data_ptr())
    return q, scale


@functools.lru_cache(maxsize=4096)
def _workspace(M: int, R: int, C: int, gated: bool, index: int) -> int:
    """Bytes of scratch of a product of these sizes on this device."""
    need = ctypes.c_int64()
    with _on(torch.device("cuda", index)):
        check(lib.tans_fp8_linear_workspace(M, R, C, gated, ctypes.byref(need)), "fp8_linear")
    return need.value


def fp8_linear(a: torch.Tensor, a_scale: torch.Tensor | None, w: torch.Tensor,
               w_scale: torch.Tensor | float = 1.0, *, bias: torch.Tensor | None = None,
               activation: str = "none", residual: torch.Tensor | None = None,
               gated: bool = False) -> torch.Tensor:
    """y = act(a_scale * w_scale * (a @ w^T) + bias) + residual as bf16, from
    E4M3FN bytes on both sides; one kernel does the product and its epilogue
    (two where a product of few tiles is split along its columns).

    a uint8 [C] or [M, C] (any M), C a multiple of 16; a_scale float32 [M] (or
    []) or None; w uint8 [R, C]; w_scale float32 [R] or a number; bias bf16 [R];
    activation one of "none", "relu", "silu", "gelu" (x Phi(x)), "gelu_tanh".
    gated: w's first R / 2 rows are the gate's, the others the value's, and
    y = act(gate) * value + residual.  residual bf16 and y are [M, R], gated
    [M, R / 2] ([R], [R / 2] for a [C]).

    Accumulation in a fixed order, one rounding.  The FP8 matrix instructions
    add products in groups of 8 columns, each cut off at 2^-13 of the largest of
    its group, and the groups in 32 bits."""
    M, C = _rows("a", a, _U8)
    dev = a.device
    if _forward._current_level >= 0:
        _no_tangents(a_scale=a_scale, w_scale=w_scale, bias=bias, residual=residual)
    if not (_ok(w, _U8, dev) and w.dim() == 2 and w.shape[0] >= 1 and w.shape[1] == C
            and isinstance(activation, str) and activation in ACTIVATIONS
            and not (gated and w.shape[0] % 2)):
        _explain("w", w, _U8, dev)
        _require(w.dim() == 2 and w.shape[0] >= 1 and w.shape[1] == C,
                 f"w must be [R, C] with C = {C}")
        _require(isinstance(activation, str) and activation in ACTIVATIONS,
                 f"activation must be one of {sorted(ACTIVATIONS)}")
        _require(False, "a gated product needs an even number of rows of w")
    R = w.shape[0]
    rows = a.shape[:-1]
    shape = (*rows, R // 2 if gated else R)
    scale, sw, sa, b, res = 1.0, None, None, None, None
    if isinstance(w_scale, torch.Tensor):
        if not (_ok(w_scale, _F32, dev) and w_scale.shape == (R,)):
            _explain("w_scale", w_scale, _F32, dev)
            _require(False, f"w_scale must be a number or [{R}]")
        sw = w_scale.data_ptr()
    else:
        scale = _number("w_scale", w_scale)
    if a_scale is not None:
        if not (_ok(a_scale, _F32, dev) and a_scale.shape == rows):
            _explain("a_scale", a_scale, _F32, dev)
            _require(False, "a_scale must hold one scale per row of a")
        sa = a_scale.data_ptr()
    if bias is not None:
        if not (_ok(bias, _BF16, dev) and bias.shape == (R,)):
            _explain("bias", bias, _BF16, dev)
            _require(False, f"bias must be [{R}]")
        b = bias.data_ptr()
    if residual is not None:
        if not (_ok(residual, _BF16, dev) and residual.shape == shape):
            _explain("residual", residual, _BF16, dev)
            _require(False, f"residual must be {list(shape)}")
        res = residual.data_ptr()
    y = torch.empty(*shape, dtype=_BF16, device=dev)
    need = _workspace(M, R, C, bool(gated), dev.index)
    ws = torch.empty(need, dtype=_U8, device=dev) if need else None
    _call(dev, "fp8_linear", lib.tans_fp8_linear, a.data_ptr(), sa, w.data_ptr(), sw, scale, b, res,
          ACTIVATIONS[activation], bool(gated), M, R, C, None if ws is None else ws.data_ptr(), need,
          y.data_ptr())
    return y
