"""tree_attention (no counterpart in the reference) against attention in 64 bits
(attention_reference.py, whose check() derives the tolerances)."""
import math
import random

import pytest
import torch

from attention_reference import attention, check

pytestmark = pytest.mark.gpu


def _say(msg):
    print(msg, flush=True)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def make_cache(g, pages, heads, page, D, fp8):
    import rans_vectoradd as R
    c = R.KvCache.empty(pages, heads, page, D, fp8=fp8)
    if not fp8:
        c.k.copy_(_randn(g, *c.k.shape))
        c.v.copy_(_randn(g, *c.v.shape))
        return c
    for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        q, scale = R.fp8_quantize_rows(_randn(g, x[..., 0].numel(), D).to(torch.bfloat16))
        x.copy_(q.view(x.shape))
        s.copy_(scale.view(s.shape))
    return c


def make_tree(rng, counts, W):
    """A random tree for each sequence: a token sees itself and its ancestors."""
    rows = []
    for n in counts:
        mine = []
        for t in range(n):
            parent = rng.randrange(-1, t) if t else -1
            row = list(mine[parent]) if parent >= 0 else [False] * W
            row[t] = True
            mine.append(row)
        rows += mine
    return torch.tensor(rows, dtype=torch.bool).view(len(rows), W).cuda()


def make_batch(rng, lens, counts, page, spare=3):
    """(pages, starts, lens, pages of the cache), in no order."""
    need = [-(-(c + t) // page) for c, t in zip(lens, counts)]
    order = list(range(sum(need) + spare))
    rng.shuffle(order)
    per = max(need + [1])
    table, at = [], 0
    for k in need:
        table.append(order[at:at + k] + [order[-1]] * (per - k))
        at += k
    starts = [0]
    for t in counts:
        starts.append(starts[-1] + t)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    return i32(table), i32(starts), i32(lens), len(order)


def run(q, cache, pages, starts, lens, mask=None, **kw):
    import rans_vectoradd as R
    return R.tree_attention(q, cache, pages, starts, lens, mask, **kw)


def compare(q, cache, pages, starts, lens, mask=None, scale=None, **kw):
    got = run(q, cache, pages, starts, lens, mask, scale=scale, **kw)
    want, spread, off = attention(q, cache, pages, starts, lens, mask,
                                  q.shape[2] ** -0.5 if scale is None else scale)
    check(got, want, spread, off, q.shape[2])
    return got


# contexts and new tokens around the units' 32 slots, the row tiles' 32 .. 256 rows
# (tokens times query heads of a cache head) and the split's borders; odd pages
CASES = [
    # lens, counts, Hq, heads, D, page
    ([0], [1], 1, 1, 64, 16),
    ([1], [1], 5, 1, 128, 1),
    ([31], [1], 8, 8, 256, 7),
    ([32], [1], 40, 8, 128, 16),
    ([63], [2], 4, 2, 64, 64),
    ([700], [1], 40, 8, 128, 16),
    ([1000], [7], 10, 2, 128, 48),
    ([4097], [1], 16, 1, 64, 256),
    ([4097], [1], 16, 1, 256, 100),
    ([333], [13], 5, 1, 128, 33),
    ([333], [13], 5, 1, 64, 33),
    ([333], [13], 5, 1, 256, 33),
    ([2050], [33], 8, 2, 128, 64),
    ([2050], [33], 8, 2, 256, 64),
    ([2050], [33], 8, 2, 64, 64),
    ([900], [100], 8, 1, 128, 16),
    ([900], [100], 8, 1, 64, 16),
    ([900], [100], 8, 1, 256, 16),
    ([0], [300], 6, 3, 128, 20),
    ([5, 100, 0, 31, 2000], [3, 1, 2, 9, 4], 6, 2, 128, 16),
    ([5, 100, 0, 31, 2000], [1, 1, 1, 1, 1], 20, 4, 64, 16),
    ([0, 0, 40], [64, 1, 65], 4, 4, 64, 32),
    ([70, 300, 8], [0, 4, 0], 4, 2, 128, 16),
    ([1500] * 3 + [7] * 70, [2] * 73, 2, 2, 64, 24),
    ([10 * i for i in range(130)], [1 + i % 3 for i in range(130)], 4, 1, 128, 16),
    ([600, 20, 1300], [40, 129, 1], 16, 2, 256, 16),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("lens,counts,Hq,heads,D,page", CASES)
def test_matches_64_bits(lens, counts, Hq, heads, D, page, tree, fp8):
    _say(f"case: attention {lens[:4]} {counts[:4]} {Hq}/{heads} x {D} page={page} tree={tree} fp8={fp8}")
    rng, g = random.Random(len(lens) * 7 + D + page), _gen(sum(lens) + D + Hq)
    pages, starts, ctx, total = make_batch(rng, lens, counts, page)
    cache = make_cache(g, total, heads, page, D, fp8)
    q = (_randn(g, sum(counts), Hq, D) * 2.0).to(torch.bfloat16)
    mask = make_tree(rng, counts, max(counts)) if tree else None
    got = compare(q, cache, pages, starts, ctx, mask)
    # every kernel gives the same to rounding, and the same bits every time
    for most in (1, 8, 20, 100, 10000):
        compare(q, cache, pages, starts, ctx, mask, max_tokens=most)
    assert torch.equal(got, run(q, cache, pages, starts, ctx, mask))


@pytest.mark.parametrize("seed", range(12))
def test_random_batches(seed):
    rng, g = random.Random(seed), _gen(seed)
    D, fp8 = rng.choice((64, 128, 256)), rng.random() < 0.5
    heads = rng.choice((1, 2, 3, 8))
    Hq = heads * rng.randint(1, 9)
    page = rng.choice((16, 32, rng.randint(1, 70)))
    B = rng.randint(1, 9)
    lens = [rng.choice((0, rng.randint(1, 100), rng.randint(1, 5000))) for _ in range(B)]
    counts = [rng.choice((0, 1, rng.randint(1, 40), rng.randint(1, 200))) for _ in range(B)]
    counts[0] = max(1, counts[0])
    _say(f"case: random {seed}: {lens} {counts} {Hq}/{heads} x {D} page={page} fp8={fp8}")
    pages, starts, ctx, total = make_batch(rng, lens, counts, page)
    cache = make_cache(g, total, heads, page, D, fp8)
    q = (_randn(g, sum(counts), Hq, D) * 3.0).to(torch.bfloat16)
    W = max(counts)
    mask = [None, make_tree(rng, counts, W), torch.rand(sum(counts), W, generator=g, device="cuda") < 0.3][seed % 3]
    compare(q, cache, pages, starts, ctx, mask, scale=rng.choice((None, 0.02, 1.0)),
            max_tokens=rng.choice((None, 1, W)))


@pytest.mark.parametrize("most", [1, 12, 30, 200])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_rows_that_see_nothing_are_zero(D, fp8, most):
    """No context and an empty row of the mask; a mask narrower than the tree, or
    without any column."""
    _say(f"case: empty rows D={D} fp8={fp8} most={most}")
    rng, g = random.Random(1), _gen(D)
    pages, starts, ctx, total = make_batch(rng, [0, 0, 50], [5, 40, 3], 16)
    cache = make_cache(g, total, 2, 16, D, fp8)
    q = _randn(g, 48, 4, D).to(torch.bfloat16)
    mask = torch.rand(48, 40, generator=g, device="cuda") < 0.5
    mask[[0, 3, 7, 44, 47]] = False
    got = compare(q, cache, pages, starts, ctx, mask, max_tokens=most)
    assert (got[[0, 3, 7, 44]] == 0).all() and (got[47] != 0).any()
    assert torch.equal(run(q, cache, pages, starts, ctx, mask[:, :2].contiguous(), max_tokens=most),
                       run(q, cache, pages, starts, ctx, mask & (torch.arange(40).cuda() < 2), max_tokens=most))
    none = run(q, cache, pages, starts, ctx, torch.zeros(48, 0, dtype=torch.bool).cuda(), max_tokens=most)
    assert (none[:45] == 0).all() and torch.equal(none, run(q, cache, pages, starts, ctx, mask & False, max_tokens=most))


@pytest.mark.parametrize("most", [1, 12, 30, 200])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_does_not_reach(D, fp8, bad, most):
    """NaN and infinities in every row of the cache that a token does not see: behind
    the last slot, in unused pages, in drafted tokens of other branches."""
    _say(f"case: unseen {bad} D={D} fp8={fp8} most={most}")
    rng, g = random.Random(3), _gen(D + 1)
    lens, counts, page = [70, 0, 33], [21, 40, 1], 16
    pages, starts, ctx, total = make_batch(rng, lens, counts, page)
    cache = make_cache(g, total, 2, page, D, fp8)
    q = _randn(g, sum(counts), 6, D).to(torch.bfloat16)
    mask = make_tree(rng, counts, 40)
    clean = compare(q, cache, pages, starts, ctx, mask, max_tokens=most)
    used = torch.zeros(total, page, dtype=torch.bool, device="cuda")
    for b in range(3):
        for s in range(lens[b] + counts[b]):
            used[pages[b, s // page].long(), s % page] = True
    # one branch of each tree is dropped: its tokens are no longer seen by the others
    dropped = [5, 9, 21 + 3, 21 + 30]
    first = [0, 0, 21, 21]
    for n, f in zip(dropped, first):
        mask[:, n - f] &= torch.arange(len(mask)).cuda() == n
        mask[n] = False
    want = compare(q, cache, pages, starts, ctx, mask, max_tokens=most)

    def spoil(at_pages, at_rows):
        if fp8:
            cache.k[at_pages, :, at_rows] = 0x7F
            cache.v[at_pages, :, at_rows] = 0xFF
            cache.k_scale[at_pages, :, at_rows] = bad
            cache.v_scale[at_pages, :, at_rows] = bad
        else:
            cache.k[at_pages, :, at_rows] = bad
            cache.v[at_pages, :, at_rows] = bad
    for n, f in zip(dropped, first):
        b = 0 if f == 0 else 1
        s = lens[b] + n - f
        spoil(pages[b, s // page].long(), s % page)
    p, r = torch.nonzero(~used, as_tuple=True)
    spoil(p, r)
    assert torch.equal(run(q, cache, pages, starts, ctx, mask, max_tokens=most), want)
    assert torch.isfinite(clean.float()).all()


@pytest.mark.parametrize("most", [1, 12, 30, 200])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_is_seen_reaches_its_rows_only(D, most):
    """An infinite or NaN value (bf16) that some tokens of a tree see makes their
    outputs infinite or NaN, and no others."""
    _say(f"case: seen infinities D={D} most={most}")
    rng, g = random.Random(5), _gen(D + 2)
    pages, starts, ctx, total = make_batch(rng, [50], [30], 16)
    cache = make_cache(g, total, 1, 16, D, False)
    q = _randn(g, 30, 2, D).to(torch.bfloat16)
    mask = make_tree(rng, [30], 30)
    for slot, d, v in ((50 + 4, 3, math.inf), (50 + 4, D - 1, math.nan), (50 + 11, 17, -math.inf)):
        cache.v[pages[0, slot // 16].long(), 0, slot % 16, d] = v
    compare(q, cache, pages, starts, ctx, mask, max_tokens=most)
    cache.v[pages[0, 0].long(), 0, 3, 5] = math.inf    # the context: all rows see it
    got = compare(q, cache, pages, starts, ctx, mask, max_tokens=most)
    assert not torch.isfinite(got[:, :, 5].float()).any()
    cache.k[pages[0, 0].long(), 0, 4, 7] = math.nan
    assert torch.isnan(run(q, cache, pages, starts, ctx, mask, max_tokens=most).float()).all()


@pytest.mark.parametrize("most", [1, 12, 30, 200])
def test_rows_of_no_sequence_are_left_as_they_were(most):
    g = _gen(7)
    pages, starts, ctx, total = make_batch(random.Random(7), [40, 90], [6, 5], 16)
    cache = make_cache(g, total, 2, 16, 128, False)
    q = _randn(g, 20, 4, 128).to(torch.bfloat16)
    starts = starts + 2                      # rows 0, 1 and those from 13 on are nobody's
    out = torch.full_like(q, 7.0)
    got = run(q, cache, pages, starts, ctx, max_tokens=most, out=out)
    assert got is out and (out[:2] == 7).all() and (out[13:] == 7).all()
    want, spread, off = attention(q, cache, pages, starts, ctx, None, 128 ** -0.5)
    check(out[2:13], want[2:13], spread[2:13], off[2:13], 128)


@pytest.mark.parametrize("most", [1, 12, 30, 200])
@pytest.mark.parametrize("fp8", [False, True])
def test_numbers_out_of_range_stay_in_the_buffers(fp8, most):
    """Pages that are none, lengths below zero and past the table, starts outside of
    the rows: their slots are not seen, the rest is right."""
    _say(f"case: out of range fp8={fp8} most={most}")
    g = _gen(8)
    pages, starts, ctx, total = make_batch(random.Random(8), [400, 90, 30, 77], [6, 5, 1, 3], 16)
    cache = make_cache(g, total, 2, 16, 64, fp8)
    q = _randn(g, 15, 4, 64).to(torch.bfloat16)
    pages[0, 3], pages[0, 24], pages[1, 0] = -1, total, 2 ** 31 - 1
    pages[1, 2] = -2 ** 31
    compare(q, cache, pages, starts, ctx, max_tokens=most)
    for lens in ([-5, 90, 30, 77], [400, 2 ** 31 - 1, -2 ** 31, 77], [10 ** 6, 90, 10 ** 9, 415]):
        ctx.copy_(torch.tensor(lens, dtype=torch.int32))
        compare(q, cache, pages, starts, ctx, max_tokens=most)
    for st in ([0, 6, 11, 12, 2 ** 31 - 1], [-2 ** 31, 6, 11, 12, 15], [-3, -2, 0, 4, 99], [0, 0, 0, 0, 0],
               [20, 30, 40, 50, 60]):
        starts.copy_(torch.tensor(st, dtype=torch.int32))
        got = run(q, cache, pages, starts, ctx, max_tokens=most, out=torch.full_like(q, 5.0))
        want, spread, off = attention(q, cache, pages, starts, ctx, None, 0.125)
        mine = torch.isfinite(want).all(dim=2).all(dim=1)
        assert (got[~mine] == 5).all()
        check(got[mine], want[mine], spread[mine], off[mine], 64)


def test_pages_none_at_all():
    """A table without columns, batches without sequences or tokens."""
    import rans_vectoradd as R
    g = _gen(9)
    cache = make_cache(g, 2, 2, 16, 64, False)
    q = _randn(g, 3, 4, 64).to(torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    none = torch.empty(1, 0, dtype=torch.int32).cuda()
    assert (run(q, cache, none, i32(0, 3), i32(5)) == 0).all()
    out = torch.full_like(q, 3.0)
    run(q, cache, none[:0], i32(0), i32(), out=out)
    assert (out == 3).all()
    assert R.tree_attention(q[:0], cache, torch.zeros(1, 1, dtype=torch.int32).cuda(), i32(0, 0), i32(5)).shape == (0, 4, 64)


def test_queries_in_longer_rows():
    g = _gen(10)
    pages, starts, ctx, total = make_batch(random.Random(10), [100, 7], [9, 4], 16)
    cache = make_cache(g, total, 2, 16, 128, True)
    qkv = _randn(g, 13, 8, 128).to(torch.bfloat16)
    q = qkv[:, 1:5]
    assert not q.is_contiguous()
    assert torch.equal(run(q, cache, pages, starts, ctx), run(q.contiguous(), cache, pages, starts, ctx))
    wide = torch.zeros(13, 4 * 128 + 24, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + 512] = q.reshape(13, 512)
    v = wide[:, 8:8 + 512].view(13, 4, 128)
    assert torch.equal(run(v, cache, pages, starts, ctx), run(q.contiguous(), cache, pages, starts, ctx))


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_past_4_gib(fp8):
    """Pages whose rows lie more than 2^32 bytes and, in elements, past 2^31 into the
    cache, at both ends of it."""
    D, heads, page = 128, 2, 64
    total = (2 ** 33 // (heads * page * D * (1 if fp8 else 2))) + 5
    _say(f"case: {total} pages fp8={fp8}")
    import rans_vectoradd as R
    g = _gen(11)
    cache = R.KvCache.empty(total, heads, page, D, fp8=fp8)
    for x in cache:
        if x is not None:
            x.view(torch.uint8).zero_()
    ids = [total - 1, 0, total - 2, total // 2, 1, total - 3]
    small = make_cache(g, len(ids), heads, page, D, fp8)
    for x, y in zip(cache, small):
        if x is not None:
            x[torch.tensor(ids).cuda()] = y
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    q = _randn(g, 5, 8, D).to(torch.bfloat16)
    for most in (1, 30):
        a = run(q, cache, i32([ids]), i32([0, 5]), i32([6 * page - 9]), max_tokens=most)
        b = run(q, small, i32([list(range(6))]), i32([0, 5]), i32([6 * page - 9]), max_tokens=most)
        assert torch.equal(a, b)
    compare(q, small, i32([list(range(6))]), i32([0, 5]), i32([6 * page - 9]))


@pytest.mark.parametrize("Hq,heads,most", [(8, 2, 1), (8, 2, 40)])
def test_a_long_context_split_over_all_workgroups(Hq, heads, most):
    _say("case: long context")
    g = _gen(12)
    pages, starts, ctx, total = make_batch(random.Random(12), [70001], [4], 128)
    cache = make_cache(g, total, heads, 128, 128, False)
    q = (_randn(g, 4, Hq, 128) * 3).to(torch.bfloat16)
    compare(q, cache, pages, starts, ctx, max_tokens=most)


def test_large_scores():
    """Scores of thousands either way: the running maximum rises and falls."""
    g = _gen(13)
    pages, starts, ctx, total = make_batch(random.Random(13), [2000], [3], 16)
    cache = make_cache(g, total, 1, 16, 64, False)
    cache.k.mul_(20.0)
    q = (_randn(g, 3, 2, 64) * 20).to(torch.bfloat16)
    got = run(q, cache, pages, starts, ctx, scale=1.0)
    want, spread, off = attention(q, cache, pages, starts, ctx, None, 1.0)
    check(got, want, spread, off, 64)


def test_other_streams_and_graphs():
    """On a stream of the caller's, captured and replayed on new inputs and lengths, two
    captures side by side, with eager calls between the replays."""
    import rans_vectoradd as R
    g = _gen(14)
    pages, starts, ctx, total = make_batch(random.Random(14), [3000, 50], [4, 9], 16)
    cache = make_cache(g, total, 2, 16, 128, True)
    q = _randn(g, 13, 10, 128).to(torch.bfloat16)
    mask = make_tree(random.Random(14), [4, 9], 9)
    want = run(q, cache, pages, starts, ctx, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, cache, pages, starts, ctx, mask)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for most in (1, 9):
        run(q, cache, pages, starts, ctx, mask, max_tokens=most)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = R.tree_attention(q, cache, pages, starts, ctx, mask, max_tokens=most)
        graphs.append((gr, o, most))
    for i in range(4):
        q.copy_(_randn(g, 13, 10, 128))
        ctx.copy_(torch.tensor([[3000, 50], [1, 0], [777, 64], [2999, 49]][i], dtype=torch.int32))
        for gr, o, most in graphs:
            gr.replay()
        for gr, o, most in graphs:
            eager = run(q, cache, pages, starts, ctx, mask, max_tokens=most)
            torch.cuda.synchronize()
            assert torch.equal(o, eager), f"replay {i}, {most}"
    # at once, on two streams
    main = torch.cuda.current_stream()
    other = torch.cuda.Stream()
    other.wait_stream(main)
    for _ in range(5):
        a = run(q, cache, pages, starts, ctx, mask)
        with torch.cuda.stream(other):
            b = run(q, cache, pages, starts, ctx, mask)
        torch.cuda.synchronize()
        assert torch.equal(a, b)
