"""What the attention operators write to counts as changed: a backward pass that saved it
fails by name where it would take the new values."""
import pytest
import torch

from test_gpu_tree_attention import _gen, _randn, make_cache

pytestmark = pytest.mark.gpu


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _case(fp8):
    import rans_vectoradd as R
    g = _gen(5)
    q, k, v = (_randn(g, 4, h, 64).to(torch.bfloat16) for h in (4, 2, 2))
    return q, k, v, _i32(0, 1, 2, 3), R.rotary_frequencies(64)[0], make_cache(g, 2, 2, 16, 64, fp8), \
        (_i32(1).view(1, 1), _i32(0, 4), _i32(0))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_outputs_and_caches_count_as_changed(grad, fp8):
    import rans_vectoradd as R
    q, k, v, p, f, cache, batch = _case(fp8)
    with torch.set_grad_enabled(grad):
        for call, written in (
                (lambda o: R.rotary(q, p, f, out=o), ()),
                (lambda o: R.rotary_append(q, k, v, p, f, cache, *batch, out=o), [x for x in cache if x is not None]),
                (lambda o: R.tree_attention(q, cache, *batch, out=o), ())):
            out = torch.empty_like(q)
            inputs = [x for x in (q, k, v, p, f, *cache, *batch) if x is not None]
            before = [x._version for x in inputs]
            at = out._version
            assert call(out) is out and out._version > at
            for x, was in zip(inputs, before):
                assert (x._version > was) == any(x is w for w in written)
            call(None)


def test_a_saved_cache_is_missed():
    import rans_vectoradd as R
    q, k, v, p, f, cache, batch = _case(False)
    w = torch.ones_like(cache.v).requires_grad_()
    y = (cache.v * w).sum()   # (saves the cache's values for w's gradient)
    with torch.no_grad():
        R.rotary_append(q, k, v, p, f, cache, *batch)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    (cache.v * w).sum().backward()
    assert torch.equal(w.grad, cache.v)


@pytest.mark.parametrize("fp8", [False, True])
def test_in_inference_mode(fp8):
    import rans_vectoradd as R
    with torch.inference_mode():
        q, k, v, p, f, cache, batch = _case(fp8)
        out = torch.empty_like(q)
        R.rotary_append(q, k, v, p, f, cache, *batch, out=out)
        o = R.tree_attention(out, cache, *batch, out=torch.empty_like(q))
    # and of its tensors outside of it
    assert torch.equal(R.rotary(q, p, f, out=torch.empty_like(q)), out)
    R.rotary_append(q, k, v, p, f, cache, *batch, out=out)
    assert torch.equal(R.tree_attention(out, cache, *batch, out=o), o)
