"""The kernel that tree_attention takes where the caller does not say how many tokens a
sequence has at most: the one that their average would choose."""
import random

import pytest
import torch

from test_gpu_tree_attention import _gen, _randn, compare, make_batch, make_cache, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens,counts,average", [
    ([2000 + 31 * b for b in range(40)], [1] * 40, 1), ([900] * 7, [1] * 7, 1), ([3000, 1000], [9, 7], 8),
    ([1500] * 9 + [40], [1] * 9 + [300], 31), ([2500], [70], 70), ([300, 500, 900], [0, 0, 2], 1)])
def test_the_average_chooses(lens, counts, average, fp8):
    """The same bits as with it, and no other kernel's where N would choose one."""
    print(f"case: {lens[:3]} and {counts[:3]}, fp8={fp8}", flush=True)
    g = _gen(sum(lens))
    pages, starts, ctx, total = make_batch(random.Random(sum(counts)), lens, counts, 16)
    cache = make_cache(g, total, 2, 16, 128, fp8)
    q = _randn(g, sum(counts), 10, 128).to(torch.bfloat16)
    got = compare(q, cache, pages, starts, ctx)
    assert torch.equal(got, run(q, cache, pages, starts, ctx, max_tokens=average))
    if len(lens) == 40:
        assert not torch.equal(got, run(q, cache, pages, starts, ctx, max_tokens=sum(counts)))


def test_no_sequences():
    g = _gen(1)
    cache = make_cache(g, 2, 2, 16, 64, False)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    q = _randn(g, 3, 2, 64).to(torch.bfloat16)
    out = torch.full_like(q, 2.0)
    run(q, cache, torch.empty(0, 4, dtype=torch.int32, device="cuda"), i32(0), i32(), out=out)
    assert (out == 2).all()
