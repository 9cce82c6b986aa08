"""Refusals of the layer operators (fp8_rmsnorm, fp8_quantize_rows,
fp8_linear), CPU only: the C entry points return TANS_EINVAL before any GPU
work, the Python wrappers raise RuntimeError."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
D16 = P(1 << 12)
F = ctypes.c_float


def _lib():
    from rans_vectoradd._lib import lib
    return lib


def _says(text):
    return text in _lib().tans_last_error()


def test_rmsnorm_refuses():
    lib = _lib()

    def call(x=D16, res=None, w=D16, M=4, D=64, eps=1e-6, q=D16, s=D16, h=None):
        return lib.tans_fp8_rmsnorm(x, res, w, M, D, F(eps), q, s, h, None)

    for kw in ({"x": None}, {"w": None}, {"q": None}, {"s": None}, {"res": D16}):
        assert call(**kw) == -1 and _says(b"null"), kw
    for D in (0, 8, 24, -16, (1 << 24) + 16):
        assert call(D=D) == -1 and _says(b"multiple of 16"), D
    for M in (-1, 1 << 31):
        assert call(M=M) == -1 and _says(b"M must"), M
    for kw in ({"x": P(8)}, {"w": P(4104)}, {"q": P(4100)}, {"s": P(4098)},
               {"res": P(4104), "h": D16}, {"res": D16, "h": P(4104)}):
        assert call(**kw) == -1 and _says(b"misaligned"), kw
    for eps in (-1e-6, float("nan")):
        assert call(eps=eps) == -1 and _says(b"eps"), eps
    assert call(M=0, x=None, q=None, s=None) == 0


def test_quantize_rows_refuses():
    lib = _lib()
    assert lib.tans_fp8_quantize_rows(None, 1, 64, D16, D16, None) == -1
    assert lib.tans_fp8_quantize_rows(D16, 1, 40, D16, D16, None) == -1
    assert lib.tans_fp8_quantize_rows(D16, -1, 64, D16, D16, None) == -1
    assert lib.tans_fp8_quantize_rows(P(4104), 1, 64, D16, D16, None) == -1
    assert lib.tans_fp8_quantize_rows(None, 0, 64, None, None, None) == 0


def test_linear_refuses():
    lib = _lib()

    def call(a=D16, sa=None, w=D16, sw=None, bias=None, res=None, act=0, gated=0, M=4, R=64, C=64,
             ws=D16, ws_bytes=1 << 40, y=D16):
        return lib.tans_fp8_linear(a, sa, w, sw, F(1.0), bias, res, act, gated, M, R, C, ws,
                                   ws_bytes, y, None)

    for kw in ({"a": None}, {"w": None}, {"y": None}):
        assert call(**kw) == -1 and _says(b"null"), kw
    for C in (0, 8, 40, -16, (1 << 22) + 16):
        assert call(C=C) == -1 and _says(b"C must"), C
    for kw in ({"M": -1}, {"R": 0}, {"R": -4}, {"R": 63, "gated": 1}, {"M": 1 << 31},
               {"R": 1 << 31}):
        assert call(**kw) == -1 and _says(b"linear: need"), kw
    for act in (-1, 5):
        assert call(act=act) == -1 and _says(b"activation"), act
    for kw in ({"a": P(4104)}, {"w": P(4104)}, {"y": P(4104)}, {"sa": P(4098)}, {"sw": P(4098)}):
        assert call(**kw) == -1 and _says(b"misaligned"), kw
    assert call(M=0, a=None, y=None) == 0
    n = ctypes.c_int64(-1)
    assert lib.tans_fp8_linear_workspace(4, 64, 64, 0, None) == -1
    assert lib.tans_fp8_linear_workspace(4, 64, 60, 0, ctypes.byref(n)) == -1
    assert lib.tans_fp8_linear_workspace(4, 64, 64, 0, ctypes.byref(n)) == 0 and n.value >= 0


def test_wrappers_refuse_what_they_cannot_take():
    import rans_vectoradd as R
    x = torch.ones(2, 64, dtype=torch.bfloat16)
    u = torch.ones(2, 64, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        R.fp8_rmsnorm(x, x[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        R.fp8_quantize_rows(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        R.fp8_linear(u, None, u)


def test_every_activation_has_its_number():
    """The names of ACTIVATIONS against the header's TANS_ACT_*."""
    import os
    import re
    from rans_vectoradd.layer import ACTIVATIONS
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "tans_amd.h")).read()
    found = {k.lower(): int(v) for k, v in re.findall(r"TANS_ACT_(\w+) = (\d+)", text)}
    assert found == ACTIVATIONS
