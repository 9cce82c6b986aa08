"""tree_attention where its kernels change: items whole or shared, two workgroups a CU,
tiles of 128 and 256 rows with many units and any number left over, maxima that rise
slowly and in steps, pages missing in the middle, against 64 bits
(attention_reference.py)."""
import random

import pytest
import torch

from attention_reference import attention, check
from test_gpu_tree_attention import _gen, _randn, _say, compare, make_batch, make_cache, make_tree, run

pytestmark = pytest.mark.gpu


def _case(seed, lens, counts, Hq, heads, D, page, fp8, tree=False):
    rng, g = random.Random(seed), _gen(seed)
    pages, starts, ctx, total = make_batch(rng, lens, counts, page)
    cache = make_cache(g, total, heads, page, D, fp8)
    q = (_randn(g, sum(counts), Hq, D) * 2.0).to(torch.bfloat16)
    return q, cache, pages, starts, ctx, make_tree(rng, counts, max(counts)) if tree else None


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G,most", [(1, 128), (1, 256), (4, 32), (4, 64), (3, 43), (1, 20), (2, 32)])
def test_every_number_of_units(D, G, most, fp8):
    """Contexts of 0 .. 13 units and some slots, so that each count of rounds and of units
    left over occurs in every tile size (20 and 2 x 32 rows: the waves share the units)."""
    rng = random.Random(D + G)
    lens = [32 * i + rng.choice((0, 1, 17, 31)) for i in range(14)]
    counts = [rng.choice((1, most, most - 1, max(1, most // 2))) for _ in lens]
    counts[3] = most
    for tree in (False, True):
        case = _case(D + G, lens, counts, 2 * G, 2, D, 16, fp8, tree)
        compare(*case)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("count", [1, 40, 90])
def test_many_items(D, count, fp8):
    """More items than four a CU: 40 tokens of 32 heads and 90 of 8 give tiles of 256 and 128
    rows (D = 256: 128) and an item a workgroup; single tokens over contexts of all lengths share them."""
    B = 160 if count == 1 else 90
    lens = [(37 * i) % 600 for i in range(B)]
    _say(f"case: {B} sequences of {count} tokens, D={D} fp8={fp8}")
    q, cache, pages, starts, ctx, _ = _case(count, lens, [count] * B, 32 if count == 40 else 8, 8, D, 16, fp8)
    got = compare(q, cache, pages, starts, ctx, max_tokens=count)
    assert torch.equal(got, run(q, cache, pages, starts, ctx, max_tokens=count))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D,Hq,heads,tokens", [(128, 10, 2, 1), (128, 5, 1, 13), (64, 16, 2, 30), (128, 4, 1, 50),
                                              (256, 4, 1, 20), (64, 2, 2, 500)])
def test_long_contexts_in_many_parts(D, Hq, heads, tokens, fp8):
    case = _case(tokens, [30011], [tokens], Hq, heads, D, 64, fp8, tree=tokens in (13, 30, 20))
    got = compare(*case, max_tokens=tokens)
    assert torch.equal(got, run(*case, max_tokens=tokens))


@pytest.mark.parametrize("tokens", [1, 9, 40])
@pytest.mark.parametrize("rise", [0.02, 0.3, 40.0, -0.3])
def test_maxima_that_rise(rise, tokens):
    """Scores that grow (or fall) along the context, by less and by more than the kernels
    let a score exceed the maximum that they refer to."""
    D, n = 64, 1500
    g = _gen(3)
    q, cache, pages, starts, ctx, _ = _case(5, [n], [tokens], 5, 1, D, 16, False)
    q.zero_()
    q[..., 0] = 8.0
    q[..., 1:] = (_randn(g, tokens, 5, D - 1) * 0.25).to(torch.bfloat16)
    for s in range(n):   # the score's leading part: rise * s / 32 in the exponent of e
        cache.k[int(pages[0, s // 16]), 0, s % 16, 0] = rise * s / 32
    compare(q, cache, pages, starts, ctx, scale=0.125, max_tokens=tokens)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tokens", [1, 12, 30, 70])
def test_pages_that_do_not_exist_in_the_middle(tokens, fp8):
    """The plain units are then computed slot by slot."""
    q, cache, pages, starts, ctx, mask = _case(tokens, [2000, 300], [tokens, 3], 4, 1, 128, 16, fp8, tree=True)
    pages[0, 40:43] = -1
    pages[0, 90] = cache[0].shape[0]
    pages[1, 0] = 1 << 30
    compare(q, cache, pages, starts, ctx, mask)
    pages[0] = -1   # none at all: the row sees nothing
    assert (compare(q, cache, pages, starts, ctx, mask)[:tokens] == 0).all()


def test_one_page_over_and_over():
    """Sequences that share their pages (a common beginning) read the same rows."""
    g = _gen(8)
    cache = make_cache(g, 5, 2, 32, 64, True)
    pages = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 1, 4]], dtype=torch.int32).cuda()
    i = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    q = _randn(g, 6, 4, 64).to(torch.bfloat16)
    compare(q, cache, pages, i(0, 2, 4, 6), i(64, 70, 90))
    # a long table of one page
    pages = torch.zeros(1, 3000, dtype=torch.int32).cuda()
    want, spread, off = attention(q, cache, pages, i(0, 6), i(95000), None, 0.125)
    check(run(q, cache, pages, i(0, 6), i(95000)), want, spread, off, 64)


def test_strides_of_longer_rows_in_every_kernel():
    """q as the first heads of a wider row, for few, some and many rows."""
    for tokens in (1, 12, 30, 70):
        q, cache, pages, starts, ctx, _ = _case(tokens, [500], [tokens], 4, 1, 128, 16, False)
        wide = _randn(_gen(1), tokens, 9, 128).to(torch.bfloat16)
        wide[:, 2:6] = q
        assert torch.equal(run(wide[:, 2:6], cache, pages, starts, ctx), run(q, cache, pages, starts, ctx))
