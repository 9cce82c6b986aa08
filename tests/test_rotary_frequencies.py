"""rotary_frequencies refuses with RuntimeError what it has no frequencies for."""
import math

import pytest
import torch

from rans_vectoradd import rotary_frequencies


@pytest.mark.parametrize("kw", [
    {"dim": 24}, {"dim": 0}, {"dim": 64.0}, {"scaling": "other"}, {"scaling": []}, {"base": "x"}, {"base": 1.0},
    {"base": math.inf}, {"base": math.nan}, {"factor": 0.5}, {"factor": math.inf}, {"factor": None},
    {"base": 1e300, "factor": 1e300, "scaling": "ntk"}, {"base": 1e300, "factor": 1e9, "scaling": "ntk"},
    *({"scaling": "yarn", **kw} for kw in (
        {"original_length": "x"}, {"original_length": math.inf}, {"original_length": math.nan},
        {"original_length": 10 ** 400}, {"original_length": 0}, {"fast": math.inf}, {"fast": math.nan}, {"fast": "x"},
        {"fast": 1e308, "slow": 1e-320}, {"fast": 1.0, "slow": 1.0}, {"slow": 0.0}, {"slow": -1.0}, {"slow": 1e-300}))])
def test_refusals(kw):
    with pytest.raises(RuntimeError):
        rotary_frequencies(**{"dim": 64, "device": "cpu", **kw})


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("dim,base,factor,kw", [
    (16, 1e30, 1e9, {}), (64, 1 + 2.0 ** -52, 2.0, {}), (1024, 1e4, 1.0, {"original_length": 1}),
    (128, 5e5, 8, {"original_length": 1e99, "fast": 1e99, "slow": 1e-99})])
def test_the_ends_of_the_ranges(dim, base, factor, kw, scaling):
    f, magnitude = rotary_frequencies(dim, base, scaling, factor, **kw, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (dim // 2,)
    assert torch.isfinite(f).all() and (f >= 0).all() and (f <= 1).all() and magnitude >= 1.0
