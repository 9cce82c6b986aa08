"""tree_attention where the batch's starts go back, so that sequences overlap and hold more
work together than any proper batch: it ends in a proper batch's time, and nothing beside
the output is written."""
import pytest
import torch

from test_gpu_tree_attention import _gen, _randn, compare, make_cache, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D,Hq,heads", [(64, 8, 2), (128, 5, 1), (256, 4, 4)])
def test_sequences_that_overlap(D, Hq, heads, fp8):
    g = _gen(D)
    cache = make_cache(g, 30, heads, 16, D, fp8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    for B, N, columns in ((2, 9, 40), (65, 40, 40), (301, 100, 3), (301, 33, 70)):
        print(f"case: {B} sequences of the same {N} tokens, D = {D}, fp8={fp8}", flush=True)
        pages = torch.randint(-1, 31, (B, columns), generator=g, device="cuda").to(torch.int32)
        starts = i32([N * (b % 2) for b in range(B + 1)])
        q = _randn(g, N, Hq, D).to(torch.bfloat16)
        for most in (1, 4, 20, N):
            out = torch.full((N + 2, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda")
            run(q, cache, pages, starts, i32([2 ** 31 - 1] * B), max_tokens=most, out=out[1:-1])
            torch.cuda.synchronize()
            assert (out[0] == 3).all() and (out[-1] == 3).all()
    # and proper ones after it
    starts = i32([0, 3, 3, 40])
    q = _randn(g, 40, Hq, D).to(torch.bfloat16)
    compare(q, cache, pages[:3].contiguous(), starts, i32([500, 1, 900]))
