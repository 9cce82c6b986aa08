"""tree_attention of single tokens over long contexts of a bf16 cache, whose probabilities
are held in 16 bits for the product with the values."""
import random

import pytest
import torch

from attention_reference import attention
from test_gpu_tree_attention import _gen, _randn, make_batch, make_cache, make_tree, run

pytestmark = pytest.mark.gpu


def close(got, want, spread, off, D):
    """attention_reference.check's bounds with another rounding of the probabilities: cut to
    bf16, of which less than 2^-7 is left; that is rounded to bf16 (2^-8 of it), or is 2^-17 of
    the probability where it is less."""
    lim = (2.0 ** -8 * want.abs() * (1 + 2.0 ** -7)
           + spread * (2.0 ** -15 + 2.0 ** -17 + 2.0 ** -16 + 2 * (2 * D + 8) * 2.0 ** -24 * off[..., None]) * (1 + 2.0 ** -7)
           + 2.0 ** -126)
    bad = (got.double() - want).abs() > lim
    assert not bad.any(), (f"{bad.sum().item()} outputs are off, the first at {torch.nonzero(bad)[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}")


@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("lens,counts,Hq,heads,D,page", [
    ([5000], [1], 5, 1, 64, 16), ([30000], [1], 40, 8, 128, 64), ([9000], [1], 4, 4, 256, 48),
    ([900, 4000, 33], [2, 1, 3], 10, 1, 128, 16), ([2000] * 300, [1] * 300, 2, 2, 64, 16),
    ([2500, 31, 700], [16, 4, 1], 4, 2, 64, 7), ([1100], [32], 3, 3, 256, 16)])
def test_shared_items_of_few_rows(lens, counts, Hq, heads, D, page, tree, flat):
    print(f"case: {lens[:4]} and {counts[:4]}, {Hq} heads over {heads}, D = {D}, tree={tree}, flat={flat}", flush=True)
    g, rng = _gen(sum(lens) + D), random.Random(D)
    pages, starts, ctx, total = make_batch(rng, lens, counts, page)
    cache = make_cache(g, total, heads, page, D, False)
    q = (_randn(g, sum(counts), Hq, D) * (0.1 if flat else 2.0)).to(torch.bfloat16)
    mask = make_tree(rng, counts, max(counts)) if tree else None
    want, spread, off = attention(q, cache, pages, starts, ctx, mask, D ** -0.5)
    close(run(q, cache, pages, starts, ctx, mask, max_tokens=max(counts)), want, spread, off, D)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_infinite_values_beside_probabilities_of_any_bits(D):
    """Probabilities that are bf16 numbers (no rest) and others, times an infinite value."""
    import rans_vectoradd as R
    cache = R.KvCache(torch.zeros(300, 1, 16, D, dtype=torch.bfloat16, device="cuda"),
                      torch.ones(300, 1, 16, D, dtype=torch.bfloat16, device="cuda"))
    pages = torch.arange(300, dtype=torch.int32).cuda().view(1, 300)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    q = torch.ones(1, 2, D, dtype=torch.bfloat16, device="cuda")
    for k in (0.0, 1.0, 0.3):
        cache.k[100:, :, :, 0] = k
        cache.v[7, 0, 3, 5], cache.v[200, 0, 9, 6], cache.v[250, 0, 1, 7] = torch.inf, -torch.inf, torch.nan
        o = R.tree_attention(q, cache, pages, i32(0, 1), i32(4799))
        assert (o[..., 5] == torch.inf).all() and (o[..., 6] == -torch.inf).all() and o[..., 7].isnan().all()
        assert (o[..., :5] == 1).all() and (o[..., 8:] == 1).all()
