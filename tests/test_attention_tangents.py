"""Forward-mode tangents and gradients of what the attention operators take besides
their first tensor: refused by name, where they would be dropped without a word."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from rans_vectoradd import attention as A


def _cache(fp8):
    return A.KvCache.empty(2, 2, 16, 64, fp8=fp8, device="cpu")


@pytest.mark.parametrize("fp8,field", [(False, "k"), (False, "v"), (True, "k_scale"), (True, "v_scale")])
def test_a_cache_with_a_tangent(fp8, field):
    cpu = torch.device("cpu")
    with fwd.dual_level():
        c = _cache(fp8)
        A._cache(c, cpu)
        t = getattr(c, field).zero_()
        c = c._replace(**{field: fwd.make_dual(t, torch.ones_like(t))})
        with pytest.raises(RuntimeError, match=f"the cache's {field} carries a tangent"):
            A._cache(c, cpu)


def test_an_output_with_a_tangent():
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with fwd.dual_level():
        assert A._out(q, q, 3, 2, 64) is q
        with pytest.raises(RuntimeError, match="out carries a tangent"):
            A._out(fwd.make_dual(q, torch.ones_like(q)), q, 3, 2, 64)


def test_factors_that_require_a_gradient():
    x = torch.tensor(2.0, requires_grad=True)
    with pytest.raises(RuntimeError, match="scale requires a gradient"):
        A._factor("scale", x)
    with torch.no_grad():
        assert A._factor("scale", x) == 2.0
    assert A._factor("scale", torch.tensor(3.0)) == 3.0 and A._factor("scale", 4) == 4.0


# -- the public calls -------------------------------------------------------------


def _case(fp8):
    from test_gpu_tree_attention import _gen, _randn, make_cache
    g = _gen(5)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    c = {"q": _randn(g, 4, 4, 64).to(torch.bfloat16), "k": _randn(g, 4, 2, 64).to(torch.bfloat16),
         "v": _randn(g, 4, 2, 64).to(torch.bfloat16), "positions": i32(0, 1, 2, 3),
         "frequencies": A.rotary_frequencies(64)[0], "magnitude": torch.tensor(1.0), "scale": torch.tensor(0.125),
         "out": torch.empty(4, 4, 64, dtype=torch.bfloat16, device="cuda"),
         "pages": i32(1).view(1, 1), "starts": i32(0, 4), "lens": i32(0)}
    return {**c, **{f"cache.{n}": x for n, x in make_cache(g, 2, 2, 16, 64, fp8)._asdict().items()}}


def _call(op, c):
    cache = A.KvCache(*(c[f"cache.{n}"] for n in A.KvCache._fields))
    batch = (cache, c["pages"], c["starts"], c["lens"])
    if op == "rotary":
        return A.rotary(c["q"], c["positions"], c["frequencies"], magnitude=c["magnitude"], out=c["out"])
    if op == "append":
        return A.rotary_append(c["q"], c["k"], c["v"], c["positions"], c["frequencies"], *batch,
                               magnitude=c["magnitude"], out=c["out"])
    return A.tree_attention(c["q"], *batch, scale=c["scale"], out=c["out"])


TAKES = {"rotary": ("q", "frequencies", "magnitude", "out"),
         "append": ("q", "k", "v", "frequencies", "magnitude", "out"), "attend": ("q", "scale", "out")}


@pytest.mark.gpu
@pytest.mark.parametrize("op", list(TAKES))
@pytest.mark.parametrize("fp8", [False, True])
def test_every_floating_input(op, fp8):
    names = TAKES[op]
    if op != "rotary":
        names += ("cache.k_scale", "cache.v_scale") if fp8 else ("cache.k", "cache.v")
    for name in names:
        print(f"case: {op}, fp8={fp8}, {name}", flush=True)
        with fwd.dual_level():
            c = _case(fp8)
            _call(op, c)
            dual = {**c, name: fwd.make_dual(c[name], torch.ones_like(c[name]))}
            with pytest.raises(RuntimeError, match="carries a tangent"):
                _call(op, dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="carries a tangent"):
                _call(op, dual)
        c = _case(fp8)
        c[name] = c[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="requires a gradient"):
            _call(op, c)
        with torch.no_grad():
            _call(op, c)
