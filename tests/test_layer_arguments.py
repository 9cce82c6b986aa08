"""What is no tensor, number or name raises RuntimeError in the layer operators,
with the argument's name, like everything else that they refuse.  Arguments that
are looked at after a CUDA tensor are in test_gpu_layer_arguments.py."""
import numpy as np
import pytest
import torch


@pytest.mark.parametrize("bad", [None, 1, 1.0, "x", [1.0] * 16, np.ones(16, dtype=np.float32)])
def test_rows_that_are_no_tensor(bad):
    import rans_vectoradd as R
    w = torch.ones(16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="x must be a tensor"):
        R.fp8_quantize_rows(bad)
    with pytest.raises(RuntimeError, match="x must be a tensor"):
        R.fp8_rmsnorm(bad, w)
    with pytest.raises(RuntimeError, match="a must be a tensor"):
        R.fp8_linear(bad, None, w)
