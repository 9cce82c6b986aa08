"""Operators of a layer's attention: rotary positions, rotary positions with the
writing of keys and values into a paged cache, and attention of each sequence's new
tokens (a tree of drafted tokens, or a chain) over that cache.  No counterpart in the
reference.

A batch is packed: of N tokens, rows starts[b] .. starts[b + 1] - 1 are sequence b's.
Its new tokens have the slots lens[b], lens[b] + 1, ... of the sequence, after the
lens[b] that the cache holds already; slot s is row s % page of the cache's page
pages[b, s // page].  These numbers are int32 tensors on the GPU.  They are not read on
the host: no value makes an access leave the tensors, but a wrong one gives a wrong
result.

  * a negative length counts as 0, starts as if clamped to 0 .. N;
  * slots past the table's pages, and those whose entry is no page of the cache, are
    neither written nor seen;
  * rows of q that belong to no sequence (behind the last, say) are left as they were
    in the output.

These are inference operators, as the other layer operators: they have no backward and
no forward-mode derivative, and inputs that require a gradient or carry a tangent are
refused (rotary's gradient is the inverse rotation, inverse=True).  Errors raise
RuntimeError.  Kernels run on the current torch stream of the inputs' device; scratch
memory comes from torch's caching allocator.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import torch

from ._C import _on, _require
from ._lib import check, lib
from .layer import _BF16, _F32, _U8, _call, _explain, _forward, _no_tangents, _number, _ok

__all__ = ["KvCache", "rotary", "rotary_append", "rotary_frequencies", "tree_attention"]

_I32, _F64 = torch.int32, torch.float64

# Marks tensors that a kernel wrote to as changed, for those who saved them for a backward
# pass: 0.2 us, and 0.9 through the public function's own checks.
_changed = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version


class KvCache(NamedTuple):
    """k, v: bf16 [pages, heads, page, D], or uint8 (E4M3FN bytes) with a float32
    scale for each row, k_scale and v_scale [pages, heads, page].  D is 64, 128 or
    256; a page holds any number of rows."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, heads: int, page: int, dim: int, fp8: bool = False, device="cuda"):
        """A cache whose rows hold nothing yet."""
        shape = (pages, heads, page, dim)
        k, v = (torch.empty(shape, dtype=_U8 if fp8 else _BF16, device=device) for _ in range(2))
        if not fp8:
            return cls(k, v)
        return cls(k, v, *(torch.empty(shape[:3], dtype=_F32, device=device) for _ in range(2)))


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 4096, fast: float = 32.0, slow: float = 1.0,
                       device="cuda"):
    """(frequencies float64 [dim / 2] in radians a position, magnitude): what rotary
    takes.  Without scaling, frequency i is base ** (-2 i / dim).  For contexts that
    are `factor` times the trained ones, `scaling` is

      "linear"  all frequencies divided by factor;
      "ntk"     a larger base, so that the slowest frequency is divided by factor and
                the fastest is kept;
      "yarn"    frequencies that turn at least `fast` times within original_length
                positions are kept, those that turn at most `slow` times divided by
                factor, between them a blend over the pair's number; magnitude
                0.1 ln(factor) + 1."""
    _require(isinstance(dim, int) and dim >= 16 and dim % 16 == 0, "dim must be a multiple of 16")
    _require(scaling in ("none", "linear", "ntk", "yarn"),
             "scaling must be one of 'linear', 'none', 'ntk', 'yarn'")
    base, factor = _number("base", base), _number("factor", factor)
    _require(1.0 < base < math.inf and 1.0 <= factor < math.inf, "base must be above 1 and factor at least 1")
    i = torch.arange(dim // 2, dtype=_F64)
    if scaling == "ntk":
        try:
            base *= factor ** (dim / (dim - 2))
        except OverflowError:
            base = math.inf
        _require(base < math.inf, "the base, enlarged by the factor, is out of range")
    f = base ** (-2.0 * i / dim)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        fast, slow = _number("fast", fast), _number("slow", slow)
        original_length = _number("original_length", original_length)
        _require(fast > slow > 0.0 and original_length >= 1, "yarn needs fast > slow > 0 and an original length")
        _require(slow > 1e-100 and max(fast, original_length) < 1e100,
                 "yarn needs fast, slow and an original length within 1e-100 .. 1e100")

        def pair(turns):   # the pair that turns so often within the trained length
            return dim * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
        stretch = ((i - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        f = f / factor * stretch + f * (1.0 - stretch)
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.to(device), magnitude


def _vector(name: str, t, dtype: torch.dtype, dev: torch.device, n: int, what: str) -> int:
    if not (_ok(t, dtype, dev) and t.shape == (n,)):
        _explain(name, t, dtype, dev)
        _require(False, f"{name} must be [{what}]")
    return t.data_ptr()


def _heads(name: str, x, dev: Optional[torch.device] = None):
    """(N, H, D, elements from a token to the next) of x [N, H, D], whose tokens may
    be parts of longer rows."""
    try:
        N, H, D = x.shape
        a, b, c = x.stride()
        row = H * D
        if N < 2:
            a = max(row, 8)
        fine = (x.dtype is _BF16 and x.is_cuda and (dev is None or x.device == dev)
                and not (x.requires_grad and torch.is_grad_enabled())
                and (c == 1 or D < 2) and (b == D or H < 2) and a >= row and a % 8 == 0)
    except (AttributeError, TypeError, ValueError, RuntimeError):   # no tensor of three dimensions
        fine = False
    if not fine:
        _require(isinstance(x, torch.Tensor), f"{name} must be a tensor")
        _require(x.is_cuda, f"{name} must be a CUDA tensor")
        _require(x.dtype is _BF16, f"{name} must be {_BF16}")
        _require(dev is None or x.device == dev, "all tensors must be on one device")
        _require(not (x.requires_grad and torch.is_grad_enabled()),
                 f"{name} requires a gradient; the attention operators have no backward")
        _require(x.dim() == 3, f"{name} must be [N, H, D]")
        _require(False, f"the heads of {name} must be contiguous, its tokens a multiple of 8 elements apart")
    return N, H, D, a


def _factor(name: str, v) -> float:
    _require(not (isinstance(v, torch.Tensor) and v.requires_grad and torch.is_grad_enabled()),
             f"{name} requires a gradient; the attention operators have no backward")
    return _number(name, v)


def _out(out, q, N: int, H: int, D: int):
    if out is None:
        return torch.empty(N, H, D, dtype=_BF16, device=q.device)
    if _forward._current_level >= 0:   # (it would keep the tangent of what is written over)
        _no_tangents(out=out)
    if not (_ok(out, _BF16, q.device) and out.shape == (N, H, D)):
        _explain("out", out, _BF16, q.device)
        _require(False, f"out must be {[N, H, D]}")
    return out


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
           interleaved: bool = False, magnitude: float = 1.0, inverse: bool = False,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions: the first rot = 2 * len(frequencies) dimensions of every head
    of x bf16 [N, H, D] are turned, pair i of token n by positions[n] * frequencies[i]
    radians, and multiplied by magnitude; the others are copied.  A pair is dimensions
    i and i + rot / 2, or 2 i and 2 i + 1 if interleaved.  positions int32 [N],
    frequencies float64 [rot / 2] (rotary_frequencies).  D and rot are multiples of 16,
    D at most 1024.

    x's tokens may be parts of longer rows (a multiple of 8 elements apart), its start
    16-byte aligned; out [N, H, D] is contiguous, and may be x itself where x is (else
    they must not overlap).
    inverse: by the negative angle.  Angles are exact to the frequencies' last bit at
    any position; one rounding, to bf16."""
    N, H, D, stride = _heads("x", x)
    dev = x.device
    if _forward._current_level >= 0:
        _no_tangents(x=x, frequencies=frequencies, magnitude=magnitude)
    half = frequencies.numel() if isinstance(frequencies, torch.Tensor) else 0
    f = _vector("frequencies", frequencies, _F64, dev, half, "rot / 2")
    p = _vector("positions", positions, _I32, dev, N, "N")
    if type(magnitude) is not float:
        magnitude = _factor("magnitude", magnitude)
    y = _out(out, x, N, H, D)
    _call(dev, "rotary", lib.tans_rotary, x.data_ptr(), stride, p, f, N, H, D, 2 * half,
          bool(interleaved), bool(inverse), magnitude, y.data_ptr(), H * D)
    if out is not None:
        _changed((out,))
    return y


def _cache(cache, dev: torch.device):
    """((k, v, scales' addresses, pages, heads, page, D), its tensors) of a cache."""
    try:
        k, v, ks, vs = cache
    except (TypeError, ValueError):
        raise RuntimeError("cache must be a KvCache") from None
    if _forward._current_level >= 0:
        _no_tangents(**{"the cache's k": k, "the cache's v": v, "the cache's k_scale": ks,
                        "the cache's v_scale": vs})
    dtype = _BF16 if ks is None and vs is None else _U8
    if not (_ok(k, dtype, dev) and _ok(v, dtype, dev) and k.dim() == 4 and v.shape == k.shape):
        _explain("the cache's k", k, dtype, dev)
        _explain("the cache's v", v, dtype, dev)
        _require(k.dim() == 4 and v.shape == k.shape, "the cache's k and v must be [pages, heads, page, D]")
    pages, heads, page, D = k.shape
    if dtype is _U8 and not (_ok(ks, _F32, dev) and _ok(vs, _F32, dev) and ks.shape == vs.shape == k.shape[:3]):
        _explain("the cache's k_scale", ks, _F32, dev)
        _explain("the cache's v_scale", vs, _F32, dev)
        _require(False, "the cache's scales must be [pages, heads, page]")
    if ks is None:
        return (k.data_ptr(), v.data_ptr(), None, None, pages, heads, page, D), (k, v)
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, page, D), (k, v, ks, vs)


def _batch(pages, starts, lens, dev: torch.device):
    """(pages' address, columns, starts, lens, sequences)."""
    if not (_ok(pages, _I32, dev) and pages.dim() == 2):
        _explain("pages", pages, _I32, dev)
        _require(False, "pages must be [B, pages of a sequence]")
    B, per = pages.shape
    s = _vector("starts", starts, _I32, dev, B + 1, "B + 1")
    n = _vector("lens", lens, _I32, dev, B, "B")
    return pages.data_ptr(), per, s, n, B


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                  frequencies: torch.Tensor, cache: KvCache, pages: torch.Tensor,
                  starts: torch.Tensor, lens: torch.Tensor, *, interleaved: bool = False,
                  magnitude: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """rotary of q bf16 [N, Hq, D] (returned) and of k [N, heads, D], and k's and v's
    rows written into the cache: token t of sequence b into its slot lens[b] + t.  An
    8-bit cache gets each row as fp8_quantize_rows would round it, from 32 bits.

    pages int32 [B, pages of a sequence], starts int32 [B + 1], lens int32 [B] (the
    slots that the cache holds before these tokens).  out may be q where q is contiguous,
    and must overlap nothing else.  Every slot must belong to one token: of sequences that
    share a page, one at most may write to it.  positions are the tokens' own (in a tree
    those of its levels), and need not be their slots."""
    N, Hq, D, sq = _heads("q", q)
    dev = q.device
    nk, hk, dk, sk = _heads("k", k, dev)
    nv, hv, dv, sv = _heads("v", v, dev)
    if _forward._current_level >= 0:
        _no_tangents(q=q, k=k, v=v, frequencies=frequencies, magnitude=magnitude)
    kc, held = _cache(cache, dev)
    bt = _batch(pages, starts, lens, dev)
    if not (nk == nv == N and hk == hv == kc[5] and D == dk == dv == kc[7]):
        _require(False, f"q, k, v must be [N, Hq, {kc[7]}] and [N, {kc[5]}, {kc[7]}] as the cache's rows")
    half = frequencies.numel() if isinstance(frequencies, torch.Tensor) else 0
    f = _vector("frequencies", frequencies, _F64, dev, half, "rot / 2")
    p = _vector("positions", positions, _I32, dev, N, "N")
    if type(magnitude) is not float:
        magnitude = _factor("magnitude", magnitude)
    y = _out(out, q, N, Hq, D)
    _call(dev, "rotary_append", lib.tans_rotary_append, q.data_ptr(), sq, k.data_ptr(), sk,
          v.data_ptr(), sv, p, f, 2 * half, bool(interleaved), magnitude, *kc, *bt, N, Hq,
          y.data_ptr())
    _changed(held)
    if out is not None:
        _changed((out,))
    return y


@functools.lru_cache(maxsize=4096)
def _workspace(N: int, B: int, Hq: int, heads: int, D: int, slots: int, most: int, index: int) -> int:
    """Bytes, by the sizes and the device's CU count."""
    need = ctypes.c_int64()
    with _on(torch.device("cuda", index)):
        check(lib.tans_tree_attention_workspace(N, B, Hq, heads, D, slots, most, ctypes.byref(need)),
              "tree_attention workspace")
    return need.value


def tree_attention(q: torch.Tensor, cache: KvCache, pages: torch.Tensor, starts: torch.Tensor,
                   lens: torch.Tensor, mask: Optional[torch.Tensor] = None, *,
                   scale: Optional[float] = None, max_tokens: Optional[int] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q bf16 [N, Hq, D], the new tokens, over the cache, which holds
    their own keys and values too (rotary_append) -> bf16 [N, Hq, D].  Hq is a
    multiple of the cache's heads: query head h reads the cache's h // (Hq / heads).

    Every token sees the lens[b] slots before the new ones.  Of the new ones it sees
    those that mask bool [N, W] names: mask[n, i] for the i-th new token of n's
    sequence (columns that W lacks are False); in a tree of drafted tokens itself and
    its ancestors.  Without a mask it sees those up to itself: one token a sequence,
    a piece of a prompt.  A token that sees nothing gets zeros.  What a token does not
    see does not reach it, be it infinite or NaN.

    pages, starts and lens as for rotary_append.  scale (default D ** -0.5) is positive.
    max_tokens: the most new tokens of a sequence (default: the mask's columns, or the
    tokens of a sequence on average); it chooses the kernel, and any value is right.  out
    may be q where q is contiguous, and must overlap nothing else.

    Scores, maxima and sums are held in 32 bits; the probabilities are rounded to bf16
    for the product with the values (of 8-bit rows after the values' scales), or held in
    16 bits: of a bf16 cache where a sequence's new tokens, times the query heads of a
    cache head, are 32 rows at most and their slots are shared by workgroups.  A call's
    result is the same bits every time."""
    N, Hq, D, stride = _heads("q", q)
    dev = q.device
    if _forward._current_level >= 0:
        _no_tangents(q=q, scale=scale)
    kc, _ = _cache(cache, dev)
    bt = _batch(pages, starts, lens, dev)
    if D != kc[7]:
        _require(False, f"q must be [N, Hq, {kc[7]}] as the cache's rows")
    m, W = None, 0
    if mask is not None:
        if not (_ok(mask, torch.bool, dev) and mask.dim() == 2 and mask.shape[0] == N):
            _explain("mask", mask, torch.bool, dev)
            _require(False, f"mask must be [{N}, new tokens]")
        if mask.shape[1] == 0:   # (a tensor without elements has no address)
            mask = torch.zeros(N, 1, dtype=torch.bool, device=dev)
        m, W = mask.data_ptr(), mask.shape[1]
    scale = D ** -0.5 if scale is None else scale if type(scale) is float else _factor("scale", scale)
    if max_tokens is None:
        # N would be a long prompt's kernel for a batch of single tokens (96 of them over 100 ..
        # 16000 slots 338 us, so 225, in 8 bits 379 / 138; 255 beside a prompt of 512 647 / 429);
        # worse is the average where one prompt has nearly all of the work (255 over 100 slots
        # beside 2048 tokens over 14000 979 / 1246)
        most = W or -(-N // max(bt[4], 1))
    else:
        _require(isinstance(max_tokens, int) and max_tokens >= 0, "max_tokens must be a whole number")
        most = min(max_tokens, N)
    y = _out(out, q, N, Hq, D)
    need = _workspace(N, bt[4], Hq, kc[5], D, bt[1] * kc[6], most, dev.index)
    ws = torch.empty(need, dtype=_U8, device=dev) if need else None
    _call(dev, "tree_attention", lib.tans_tree_attention, q.data_ptr(), stride, *kc, *bt, m, W, N, Hq,
          scale, most, None if ws is None else ws.data_ptr(), need, y.data_ptr())
    if out is not None:
        _changed((out,))
    return y
