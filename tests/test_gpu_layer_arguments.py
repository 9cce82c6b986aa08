"""The layer operators' other arguments: what is no tensor, number or name raises
RuntimeError with the argument's name."""
import numpy as np
import pytest
import torch

import test_gpu_layer as L

pytestmark = pytest.mark.gpu


def test_what_is_no_tensor_or_number_is_refused_by_name():
    import rans_vectoradd as R
    g = L._gen(1)
    x, w = L._bf16(g, 4, 64), L._bf16(g, 64)
    a, wq = L._fp8(g, 4, 64), L._fp8(g, 32, 64)
    s = torch.ones(4, device="cuda")

    def refuses(match, f, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)

    for bad in (None, 2.0, [1.0] * 64, np.ones(64, dtype=np.float32)):
        refuses("weight must be a tensor", R.fp8_rmsnorm, x, bad)
        refuses("w must be a tensor", R.fp8_linear, a, s, bad)
    for bad in (2.0, [1.0] * 64, np.ones(64, dtype=np.float32)):
        refuses("residual must be a tensor", R.fp8_rmsnorm, x, w, bad)
        refuses("a_scale must be a tensor", R.fp8_linear, a, bad, wq)
        refuses("bias must be a tensor", R.fp8_linear, a, s, wq, bias=bad)
        refuses("residual must be a tensor", R.fp8_linear, a, s, wq, residual=bad)
    for bad in (None, "small", [1.0, 2.0], 10 ** 400, 1j):
        refuses("eps must be a number", R.fp8_rmsnorm, x, w, eps=bad)
        refuses("w_scale must be a number", R.fp8_linear, a, s, wq, bad)
    for bad in (None, 1, ["silu"], {"silu": 1}):
        refuses("activation must be one of", R.fp8_linear, a, s, wq, activation=bad)


def test_numbers_of_other_types_are_taken():
    import rans_vectoradd as R
    g = L._gen(1)
    x, w = L._bf16(g, 4, 64), L._bf16(g, 64)
    a, wq = L._fp8(g, 4, 64), L._fp8(g, 32, 64)
    want = R.fp8_rmsnorm(x, w, eps=1.0)
    for one in (1, True, np.float32(1), np.float64(1), np.int64(1), torch.tensor(1.0)):
        for got, ref in zip(R.fp8_rmsnorm(x, w, eps=one), want):
            assert torch.equal(got, ref)
        if not isinstance(one, torch.Tensor):   # (scales in a tensor are one for each row of w)
            assert torch.equal(R.fp8_linear(a, None, wq, one), R.fp8_linear(a, None, wq))
