"""fp8_linear bit for bit: operands are small whole numbers and scales powers of
two, so that every product, sum and epilogue is exact in 32 bits (the FP8 matrix
instructions cut a product off at 2^-13 of the largest of its group of 8: of at
most 16 that is less than the smallest, 1) and y is the exact value, rounded
once to bf16.  One wrong output anywhere fails, also in rows of 17408 columns.

Each case names the kernel that it is meant for (on 256 CUs; which one it takes
is checked on the CPU in test_linear_choices.py); among them products of which a
persistent workgroup takes several tiles, of either width, plain and gated."""
import pytest
import torch

import test_gpu_layer as L

pytestmark = pytest.mark.gpu

# (rows of a, rows of w, columns, gated, kernel)
CASES = [
    (1, 5121, 17408, False, "stream"), (7, 534, 17408, True, "stream"), (13, 2187, 1296, False, "few"),
    (20, 1035, 17408, False, "few"), (31, 9002, 4000, True, "stream"),
    (47, 31, 17408, False, "mid split"), (100, 1035, 17408, False, "mid split"),
    (300, 1034, 17408, True, "mid split"), (256, 5120, 17408, False, "mid split"),
    (700, 5121, 17408, False, "mid split"), (97, 34816, 5120, True, "mid"),
    (4241, 644, 3824, True, "mid"), (1003, 2187, 1296, False, "mid"),
    (2049, 4099, 16, False, "pairs"), (2047, 4354, 144, True, "pairs"), (4389, 29417, 304, False, "pairs"),
    (1537, 5633, 768, False, "pairs"),
    (2048, 5120, 17408, False, "tiles 192"), (3001, 5121, 17408, False, "tiles 256"),
    (1500, 10242, 5120, True, "tiles 256")]

# several tiles a workgroup
MANY = [
    (2500, 10202, 2064, True, "tiles 256"), (4090, 8102, 3088, True, "tiles 256"),
    (2540, 13050, 2064, False, "tiles 256"), (3001, 10243, 17408, False, "tiles 256"),
    (4101, 4500, 912, False, "tiles 192"), (1100, 24000, 912, False, "tiles 192"),
    (5003, 15001, 1040, False, "tiles 192"),
    # one step to seven of 128 columns, the last one partly filled
    (130, 92292, 48, False, "tiles 192"), (129, 70849, 160, False, "tiles 192"),
    (133, 69693, 336, False, "tiles 192"), (137, 65823, 464, False, "tiles 192"),
    (130, 65671, 608, False, "tiles 192"), (136, 66789, 688, False, "tiles 192"),
    (130, 67008, 816, False, "tiles 192")]

# y of more than 2^32 bytes
PAST_4_GIB = (70_001, 34816, 784, False, "tiles 192")


def _whole(g, most, *shape):
    """E4M3FN bytes of whole numbers -most .. most, and their values."""
    v = torch.randint(-most, most + 1, shape, generator=g, device="cuda").float()
    return v.to(torch.float8_e4m3fn).view(torch.uint8), v


def _powers(g, lo, hi, n):
    return torch.exp2(torch.randint(lo, hi + 1, (n,), generator=g, device="cuda").float())


def _product(M, R_, C, gated, seed, relu=True):
    """(the call, the exact result as a function of rows lo .. hi)."""
    import rans_vectoradd as R
    g = L._gen(seed)
    a, av = _whole(g, 2 if gated else 4, M, C)
    w, wv = _whole(g, 2 if gated else 4, R_, C)
    N = R_ // 2 if gated else R_
    # gated: gate times value has twice the bits
    sa, sw = _powers(g, -1, 0, M), _powers(g, 0 if gated else -2, 0, R_)
    bias = torch.randint(-8, 9, (R_,), generator=g, device="cuda").to(torch.bfloat16)
    res = torch.randint(-8, 9, (M, N), generator=g, device="cuda").to(torch.bfloat16)
    wt = wv.double().t().contiguous()

    def exact(lo, hi):
        v = (av[lo:hi].double() @ wt) * sa[lo:hi, None].double() * sw.double() + bias.double()
        act = v.clamp(min=0.0) if relu else v
        y = act[:, :N] * v[:, N:] if gated else act
        y = y + res[lo:hi].double()
        f = y.float()
        assert (f.double() == y).all()       # 32 bits hold it
        return f.to(torch.bfloat16)

    y = R.fp8_linear(a, sa, w, sw, bias=bias, activation="relu" if relu else "none", residual=res,
                     gated=gated)
    return y, exact


@pytest.mark.parametrize("M,R_,C,gated,kernel", CASES + MANY)
def test_linear_is_exact(M, R_, C, gated, kernel):
    L._say(f"case: linear exact {M}x{R_}x{C} gated={gated} ({kernel})")
    for relu in (False, True):
        y, exact = _product(M, R_, C, gated, M + R_ + C, relu)
        for lo in range(0, M, 4096):
            assert torch.equal(y[lo:lo + 4096], exact(lo, min(M, lo + 4096)))


def test_linear_is_exact_past_4_gib_of_output():
    M, R_, C, gated, kernel = PAST_4_GIB
    L._say(f"case: linear exact {M}x{R_}x{C} ({kernel})")
    y, exact = _product(M, R_, C, gated, 1)
    for lo in range(0, M, 4096):
        assert torch.equal(y[lo:lo + 4096], exact(lo, min(M, lo + 4096))), lo
