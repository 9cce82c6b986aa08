"""fp8_linear takes bias and residual at any element of a larger buffer (a slice
of a fused bias, rows of a matrix with an odd number of columns) and gives the
bits that it gives with copies of their own."""
import pytest
import torch

import test_gpu_layer as L

pytestmark = pytest.mark.gpu


# few rows, tiles whole and split along the columns, pairs of workgroups, large
# tiles of 256 and 192 rows of w; outputs that fill the tiles and that do not
@pytest.mark.parametrize("M,R_,C,gated", [
    (1, 530, 272, False), (20, 512, 272, True), (97, 1024, 656, False), (100, 1030, 656, True),
    (64, 640, 4096, False), (66, 642, 4096, True), (2047, 4354, 144, True), (2048, 4352, 272, False),
    (1500, 5120, 2576, False), (2500, 6160, 1296, False), (1060, 11000, 656, True)])
@pytest.mark.parametrize("shift", [1, 2, 3, 5, 7])
def test_bias_and_residual_at_any_element(M, R_, C, gated, shift):
    import rans_vectoradd as R
    L._say(f"case: linear alignment {M}x{R_}x{C} gated={gated} shift={shift}")
    g = L._gen(M + shift)
    a, w = L._fp8(g, M, C), L._fp8(g, R_, C)
    N = R_ // 2 if gated else R_
    bias_buf, res_buf = L._bf16(g, R_ + 8), L._bf16(g, M * N + 8)
    bias, res = bias_buf[shift:shift + R_], res_buf[shift:shift + M * N].view(M, N)
    assert bias.data_ptr() % 16 and res.data_ptr() % 16
    y = R.fp8_linear(a, None, w, 1e-3, bias=bias, activation="silu", residual=res, gated=gated)
    want = R.fp8_linear(a, None, w, 1e-3, bias=bias.clone(), activation="silu", residual=res.clone(),
                        gated=gated)
    assert torch.equal(y, want)
