"""tree_attention with infinities and NaN among the keys, values and scales: each output
is the infinity, the NaN or the number that the formula gives over the slots that its
token sees, in 64 bits."""
import math
import random

import pytest
import torch

from attention_reference import check, rows_of
from test_gpu_tree_attention import _gen, _randn, make_batch, make_cache, make_tree, run

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def formula(q, cache, pages, starts, lens, mask):
    """(o, spread, off) as attention_reference.attention's, each sum over the seen slots
    alone, so that what is infinite or NaN takes its way by itself."""
    N, Hq, D = q.shape
    heads = cache[0].shape[1]
    scale = D ** -0.5
    o = torch.full((N, Hq, D), NAN, dtype=torch.float64, device=q.device)
    spread, off = torch.zeros_like(o), torch.zeros(N, Hq, dtype=torch.float64, device=q.device)
    for b, c in enumerate(lens.tolist()):
        n0, n1 = starts[b].item(), starts[b + 1].item()
        K, V, ok = rows_of(cache, pages[b], c + n1 - n0)
        assert ok.all()
        for n in range(n0, n1):
            new = mask[n, :n1 - n0] if mask is not None else torch.arange(n1 - n0, device=q.device) <= n - n0
            at = torch.cat((torch.arange(c, device=q.device), c + torch.nonzero(new).flatten()))
            k, v = (x[at].transpose(0, 1).repeat_interleave(Hq // heads, dim=0) for x in (K, V))   # [Hq, seen, D]
            products = q[n].double()[:, None, :] * k
            s = products.sum(dim=2) * scale
            p = torch.exp(s - s.amax(dim=1, keepdim=True))
            w = (p / p.sum(dim=1, keepdim=True))[..., None]
            o[n] = (w * v).sum(dim=1)
            spread[n] = (w * torch.nan_to_num(v, 0.0, 0.0, 0.0).abs()).sum(dim=1)
            off[n] = torch.nan_to_num(products, 0.0, 0.0, 0.0).abs().sum(dim=2).amax(dim=1) * scale
    return o, spread, off


def same(got, want, spread, off, D):
    g = got.double()
    for name, kind in (("NaN", torch.isnan), ("inf", torch.isposinf), ("-inf", torch.isneginf)):
        wrong = kind(g) != kind(want)
        assert not wrong.any(), (f"{name}: {int(wrong.sum())} outputs, the first at {torch.nonzero(wrong)[0].tolist()}: "
                                 f"{g[wrong][0].item()} for {want[wrong][0].item()}")
    fine = torch.isfinite(want)
    check(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), spread, off, D)


# (contexts, tokens): single tokens, 32 rows, 64, 128, 256; whole items and shared ones
SHAPES = [([300], [1]), ([3000], [1]), ([200, 37], [5, 9]), ([2100], [13]), ([70, 500], [33, 20]), ([1700], [70])]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 48), (256, 16), (256, 9)])
def test_infinities_take_their_way(D, page, tree, fp8):
    for lens, counts in SHAPES:
        print(f"case: D = {D}, page {page}, {lens} and {counts}, tree={tree}, fp8={fp8}", flush=True)
        g, rng = _gen(D + sum(lens)), random.Random(sum(counts) + page)
        pages, starts, ctx, total = make_batch(rng, lens, counts, page)
        cache = make_cache(g, total, 2, page, D, fp8)
        q = _randn(g, sum(counts), 8, D).to(torch.bfloat16)
        mask = make_tree(rng, counts, max(counts)) if tree else None
        for c, t, b in zip(lens, counts, range(len(lens))):
            # of the context the first slot, one inside and the last; of the new ones two
            for i, slot in enumerate((0, c // 2, c - 1, c + t // 2, c + t - 1)):
                at = (int(pages[b, slot // page]), i % 2, slot % page)
                d = rng.randrange(D)
                if not fp8:
                    cache.v[at][d] = (INF, -INF, NAN, INF, -INF)[i]
                    cache.v[at][(d + 5) % D] = (-INF, NAN, INF, NAN, INF)[i]
                elif i % 2:
                    cache.v[at][d] = (0x7F, 0xFF)[i // 2]
                else:
                    cache.v_scale[at] = (NAN, INF, -INF)[i // 2]
        want, spread, off = formula(q, cache, pages, starts, ctx, mask)
        assert torch.isfinite(want).any() and not torch.isfinite(want).all()
        same(run(q, cache, pages, starts, ctx, mask), want, spread, off, D)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 48), (256, 16), (256, 9)])
def test_scores_that_are_infinite(D, page, tree, fp8):
    """A key's infinity makes a score of either sign: the row is NaN, or does not have the
    slot.  (8 bits: NaN alone, as byte or scale.)"""
    for lens, counts in SHAPES:
        print(f"case: D = {D}, page {page}, {lens} and {counts}, tree={tree}, fp8={fp8}", flush=True)
        g, rng = _gen(D + sum(lens)), random.Random(sum(counts) + page)
        pages, starts, ctx, total = make_batch(rng, lens, counts, page)
        cache = make_cache(g, total, 2, page, D, fp8)
        q = _randn(g, sum(counts), 8, D).to(torch.bfloat16)
        q = torch.where(q == 0, 1.0, q)
        mask = make_tree(rng, counts, max(counts)) if tree else None
        c, t = lens[0], counts[0]
        for i, slot in enumerate((c // 3, c + t // 2)):
            at = (int(pages[0, slot // page]), i, slot % page)
            if not fp8:
                cache.k[at][rng.randrange(D)] = (INF, -INF)[i]
            elif i:
                cache.k[at][rng.randrange(D)] = 0x7F
            else:
                cache.k_scale[at] = NAN
        want, spread, off = formula(q, cache, pages, starts, ctx, mask)
        assert fp8 is False or torch.isnan(want).any()   # (a single token's rows may all be NaN)
        same(run(q, cache, pages, starts, ctx, mask), want, spread, off, D)
