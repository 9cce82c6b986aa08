"""fp8_rmsnorm of rows whose squares leave the range of 32 bits: the norm of a
finite row is what the formula gives, however large or small its elements are
(eps included: it is compared with the mean square of the row as it is).
Against 64 bits, with the bounds of tests/test_gpu_layer.py."""
import pytest
import torch

import test_gpu_layer as L

pytestmark = pytest.mark.gpu

# one wave a row, several, and the three passes of the longest rows
WIDTHS = [16, 272, 1040, 5120, 65552]


def _rows(g, D, kind):
    x = torch.randn(8, D, generator=g, device="cuda")
    if kind == "huge":
        x[0] *= 1e25
        x[1, 5] = 3.0e38                     # among ordinary values
        x[2] = -1.0e30
        x[3] = 2.0 ** 62                     # squares that are finite, their sum is not
        x[4] *= 3.0e37
        x[5, D - 1] = -2.0 ** 64             # the smallest power whose square is infinite
    else:
        x[0] *= 2.0 ** -45
        x[1] *= 2.0 ** -70
        x[2] *= 2.0 ** -120
        x[3] *= 2.0 ** -130                  # subnormal
        x[4] = 0.0
        x[4, 3] = 2.0 ** -133                # the smallest bf16
        x[5] *= 2.0 ** -62                   # squares at the border of subnormals
        x[5, D - 2] = 2.0 ** -50
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("kind,eps", [("huge", 1e-6), ("huge", 0.0), ("huge", 1e30), ("tiny", 0.0),
                                      ("tiny", 1e-36), ("tiny", 1e-30), ("tiny", 1e-6)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_of_rows_out_of_the_squares_range(D, kind, eps, with_residual):
    import rans_vectoradd as R
    L._say(f"case: rmsnorm range 8x{D} {kind} eps={eps} residual={with_residual}")
    g = L._gen(D)
    x = _rows(g, D, kind)
    w = L._bf16(g, D)
    res = None
    if with_residual:   # of x's size, so that the sum is what has to be scaled
        res = (x.float() * 0.25).to(torch.bfloat16)
        x = (x.float() * 0.75).to(torch.bfloat16)
    q, scale, _ = R.fp8_rmsnorm(x, w, res, eps=eps)
    # 32 bits are what eps is passed in
    want = L._norm64(x, w, res, torch.tensor(eps, dtype=torch.float32).double().item())
    assert torch.isfinite(scale).all()
    L._check_q(q, scale, want)


@pytest.mark.parametrize("D", WIDTHS)
def test_rows_out_of_range_leave_the_others_alone(D):
    import rans_vectoradd as R
    g = L._gen(D + 1)
    x, w = L._bf16(g, 12, D), L._bf16(g, D)
    clean = R.fp8_rmsnorm(x, w)
    y = x.clone()
    y[3] *= 1e30
    y[7, D // 2] = float("nan")
    y[8, 0] = float("inf")
    y[9] = 0.0
    got = R.fp8_rmsnorm(y, w)
    keep = [0, 1, 2, 4, 5, 6, 10, 11]
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
    L._check_q(got[0][3], got[1][3], L._norm64(y[3], w, None, 1e-6))
    assert not torch.isfinite(got[1][7]) and not torch.isfinite(got[1][8])
    assert (got[0][9] & 0x7F == 0).all()
