"""The layer operators have no derivative: inputs that forward-mode
differentiation follows are refused, as those that require a gradient are."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import test_gpu_layer as L

pytestmark = pytest.mark.gpu


def _calls():
    """(name of the input, that input, a call with it)"""
    import rans_vectoradd as R
    g = L._gen(2)
    x, res, w = L._bf16(g, 4, 64), L._bf16(g, 4, 64), L._bf16(g, 64)
    a, wq = L._fp8(g, 4, 64), L._fp8(g, 32, 64)
    s, ws, b, r = torch.ones(4, device="cuda"), torch.ones(32, device="cuda"), L._bf16(g, 32), L._bf16(g, 4, 32)
    return [("x", x, lambda t: R.fp8_rmsnorm(t, w, res)),
            ("weight", w, lambda t: R.fp8_rmsnorm(x, t, res)),
            ("residual", res, lambda t: R.fp8_rmsnorm(x, w, t)),
            ("x", x, R.fp8_quantize_rows),
            ("a_scale", s, lambda t: R.fp8_linear(a, t, wq, ws)),
            ("w_scale", ws, lambda t: R.fp8_linear(a, s, wq, t)),
            ("bias", b, lambda t: R.fp8_linear(a, s, wq, ws, bias=t)),
            ("residual", r, lambda t: R.fp8_linear(a, s, wq, ws, residual=t))]


@pytest.mark.parametrize("which", range(8))
def test_inputs_with_a_tangent_are_refused(which):
    name, t, call = _calls()[which]
    with fwd.dual_level():
        dual = fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):   # torch's own follow it here
            call(dual)
        call(t)                          # others are taken
        call(fwd.unpack_dual(dual).primal)
        with torch.inference_mode():     # which ends forward mode too
            call(dual)
    call(t)


def test_function_transforms_are_refused():
    _, t, call = _calls()[3]
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: call(x)[1], (t,), (torch.ones_like(t),))
