"""Outputs that the C entry points may write over an input: the product's y over
its residual, the norm's h over x or over the residual.  The same bits as with
buffers of their own, in every kernel."""
import ctypes

import pytest
import torch

import test_gpu_layer as L

pytestmark = pytest.mark.gpu

# (rows of a, rows of w, columns, gated, kernel): outputs that fill no tile, odd
# numbers of them, and ones that fill every tile
CASES = [
    (5, 1035, 1296, False, "few"), (9, 20002, 528, True, "stream"), (16, 17408, 512, False, "stream"),
    (100, 1035, 17408, False, "mid split"), (300, 1034, 17408, True, "mid split"),
    (256, 5120, 17408, False, "mid split"), (1003, 2187, 1296, False, "mid"),
    (4241, 646, 3824, True, "mid"), (2047, 4354, 144, True, "pairs"), (2048, 4352, 272, False, "pairs"),
    (2540, 13051, 2064, False, "tiles 256"), (2500, 10202, 2064, True, "tiles 256"),
    (4101, 4501, 912, False, "tiles 192"), (2048, 5120, 17408, False, "tiles 192")]


@pytest.mark.parametrize("M,R_,C,gated,kernel", CASES)
def test_product_over_its_residual(M, R_, C, gated, kernel):
    import rans_vectoradd as R
    from rans_vectoradd._lib import lib
    L._say(f"case: linear in place {M}x{R_}x{C} gated={gated} ({kernel})")
    g = L._gen(M + C)
    a, w = L._fp8(g, M, C), L._fp8(g, R_, C)
    N = R_ // 2 if gated else R_
    res = L._bf16(g, M, N)
    want = R.fp8_linear(a, None, w, 1e-3, activation="silu", residual=res, gated=gated)
    need = ctypes.c_int64()
    assert lib.tans_fp8_linear_workspace(M, R_, C, gated, ctypes.byref(need)) == 0
    ws = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    y = res.clone()
    assert lib.tans_fp8_linear(a.data_ptr(), None, w.data_ptr(), None, 1e-3, None, y.data_ptr(), 2,
                               gated, M, R_, C, ws.data_ptr(), need.value, y.data_ptr(),
                               torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, want)


# one wave a row, several, and the three passes of the longest rows (five where
# the squares overflow)
@pytest.mark.parametrize("D", [272, 1296, 5120, 65552])
@pytest.mark.parametrize("over", ["x", "residual"])
@pytest.mark.parametrize("std", [1.0, 1e30])
def test_norm_over_x_or_the_residual(D, over, std):
    import rans_vectoradd as R
    from rans_vectoradd._lib import lib
    L._say(f"case: rmsnorm in place 12x{D} over {over} std={std}")
    g = L._gen(D)
    x, res, w = L._bf16(g, 12, D, std=std), L._bf16(g, 12, D, std=std), L._bf16(g, D)
    q, s, h = R.fp8_rmsnorm(x, w, res)
    x2, res2 = x.clone(), res.clone()
    h2 = x2 if over == "x" else res2
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    assert lib.tans_fp8_rmsnorm(x2.data_ptr(), res2.data_ptr(), w.data_ptr(), 12, D, 1e-6,
                                q2.data_ptr(), s2.data_ptr(), h2.data_ptr(),
                                torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(h2, h) and torch.equal(q2, q) and torch.equal(s2, s)
    other, was = (res2, res) if over == "x" else (x2, x)
    assert torch.equal(other, was)
