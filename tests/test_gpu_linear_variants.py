"""fp8_linear at products that take each of its kernels (streaming with either
workgroup, every tile, with and without splits along the columns, the large
tiles), outputs that fill no tile and columns that end inside a step, plain and
gated; seeded products of random sizes; rows of w past 4 GiB; and weights whose
products cancel.  Against 64 bits, with the bounds of tests/test_gpu_layer.py."""
import random

import pytest
import torch

import test_gpu_layer as L

pytestmark = pytest.mark.gpu

# (rows of a, rows of w, columns, gated)
VARIANTS = [
    (5, 1035, 1296, False), (16, 4215, 528, False), (17, 4215, 400, False), (9, 38, 2064, True),
    (18, 2, 16, True), (31, 8870, 272, True),
    (33, 1, 16, False), (33, 2, 16, True), (36, 1, 1904, False), (36, 2, 1808, True),
    (2842, 153, 16, False), (2793, 130, 16, True), (1062, 70, 2272, False), (676, 66, 4160, True),
    (2734, 358, 288, False), (2470, 418, 272, True), (1448, 67, 5248, False),
    (2115, 66, 3808, True), (2410, 837, 144, False), (1480, 1284, 160, True),
    (1832, 132, 4880, False), (2795, 140, 2912, True), (2800, 866, 144, False),
    (1160, 2138, 144, True), (2730, 1, 3984, False), (2771, 2, 3888, True),
    (2750, 1045, 160, False), (1433, 2214, 144, True), (2069, 1, 7568, False),
    (2841, 2, 8384, True), (302, 11315, 1200, False), (149, 17162, 1184, True),
    (2202, 271, 8832, False), (2752, 270, 8000, True), (535, 6809, 272, False),
    (290, 10986, 288, True), (68, 10894, 5456, False), (155, 5432, 6048, True),
    (2086, 2001, 16, False), (1665, 2436, 16, True), (137, 6258, 9568, False),
    (67, 17438, 5872, True), (1576, 7625, 672, False), (1060, 11000, 656, True),
    (1500, 5120, 2576, False), (1801, 4099, 1040, False), (1537, 5115, 3216, False),
    (2500, 6160, 1296, False)]


@pytest.mark.parametrize("M,R_,C,gated", VARIANTS)
def test_linear_variants(M, R_, C, gated):
    L._say(f"case: linear variant {M}x{R_}x{C} gated={gated}")
    L._run_linear(M, R_, C, "silu" if gated else "none", gated, bias=True, residual=True)
    L._run_linear(M, R_, C, "gelu", gated, seed=1)


def _random_products(n, seed):
    rng = random.Random(seed)

    def size(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))
    out = []
    for _ in range(n):
        C = 16 * size(1, 1088)
        R_ = min(size(1, 20000), 30_000_000 // C)
        gated = rng.random() < 0.4
        R_ = max(2, R_ - R_ % 2) if gated else R_
        M = min(size(1, 5000), max(1, 400_000_000 // (R_ * 40)))
        out.append((M, R_, C, gated, rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    rng.random() < 0.5, rng.random() < 0.5))
    return out


@pytest.mark.parametrize("M,R_,C,gated,act,bias,residual", _random_products(60, 17))
def test_linear_random_products(M, R_, C, gated, act, bias, residual):
    L._say(f"case: linear random {M}x{R_}x{C} {act} gated={gated} {bias} {residual}")
    L._run_linear(M, R_, C, act, gated, bias, residual, seed=3)


@pytest.mark.parametrize("M", [2, 40, 600])
def test_linear_weights_past_4_gib(M):
    """Rows of w beyond 2^32 bytes give what they give as a matrix of their own."""
    import rans_vectoradd as R
    R_, C = 1_100_003, 4096           # 4.5 GB
    g = L._gen(2)
    w = torch.randint(0, 120, (R_, C), generator=g, device="cuda", dtype=torch.uint8)
    a = L._fp8(g, M, C)
    y = R.fp8_linear(a, None, w, 1e-5)
    for lo in (0, 1_048_448, R_ - 515):
        part = w[lo:lo + 515].contiguous()
        want, off, _ = L._linear64(a, None, part, 1e-5, None, "none", None, False)
        err = (y[:, lo:lo + 515].double() - want).abs()
        assert (err <= off + (want.abs() + off) * 2.0 ** -8 + 2.0 ** -130).all()


def test_linear_many_rows_past_4_gib_of_output():
    """y of more than 2^32 bytes."""
    import rans_vectoradd as R
    M, R_, C = 70_001, 34816, 32
    g = L._gen(6)
    a, w = L._fp8(g, M, C), L._fp8(g, R_, C)
    y = R.fp8_linear(a, None, w, 1e-3)
    for lo in (0, 61_600, M - 300):
        want, off, _ = L._linear64(a[lo:lo + 300].contiguous(), None, w, 1e-3, None, "none", None,
                                   False)
        err = (y[lo:lo + 300].double() - want).abs()
        assert (err <= off + (want.abs() + off) * 2.0 ** -8 + 2.0 ** -130).all()


@pytest.mark.parametrize("M", [1, 20, 100, 700])
@pytest.mark.parametrize("C", [128, 272, 4096])
def test_linear_sums_that_cancel_exactly(M, C):
    """Every second weight row is the negative of the one before, a constant
    along the columns: products of equal size cancel to zero exactly in any
    order, and the rows themselves sum to C times one product."""
    import rans_vectoradd as R
    a = torch.full((M, C), 0x38, dtype=torch.uint8, device="cuda")         # 1.0
    w = torch.full((514, C), 0x40, dtype=torch.uint8, device="cuda")       # 2.0
    w[1::2, ::2] = 0xC0                                                    # -2.0
    y = R.fp8_linear(a, None, w)
    assert (y[:, 0::2] == 2.0 * C).all() and (y[:, 1::2] == 0.0).all()


# tiles of 192 x 160 rows and gated ones of 256 x 256
@pytest.mark.parametrize("M,R_,C,gated", [
    (190, 34838, 272, False), (191, 34818, 272, True), (557, 13136, 16, True),
    (136, 17968, 6128, False), (131, 16398, 6096, True), (290, 32730, 1376, True),
    (643, 17400, 656, False)])
def test_linear_wide_tiles(M, R_, C, gated):
    L._say(f"case: linear {M}x{R_}x{C} gated={gated}")
    L._run_linear(M, R_, C, "silu" if gated else "none", gated, bias=True, residual=True)
    L._run_linear(M, R_, C, "gelu", gated, seed=1)


# few steps and many tiles: 128 x 128, two workgroups a CU
@pytest.mark.parametrize("M,R_,C,gated", [
    (2049, 4099, 16, False), (2047, 4354, 144, True), (4225, 2049, 272, False),
    (1151, 7938, 384, True), (363, 22017, 528, False), (1537, 5633, 768, False)])
@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
def test_linear_two_workgroups_a_cu(M, R_, C, gated, act):
    L._say(f"case: linear pairs {M}x{R_}x{C} {act} gated={gated}")
    L._run_linear(M, R_, C, act, gated, bias=True, residual=True)
