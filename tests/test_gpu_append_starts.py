"""rotary_append where the batch's starts go back: only rows that lie in their sequence
are written, and nothing beside the cache."""
import pytest
import torch

from test_gpu_tree_attention import _gen, _randn

pytestmark = pytest.mark.gpu


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_before_their_sequence_are_left(D, fp8):
    import rans_vectoradd as R
    print(f"case: starts 5, 6, 0, 8, D = {D}, fp8={fp8}", flush=True)
    g = _gen(D)
    q, k, v = (_randn(g, 8, h, D).to(torch.bfloat16) for h in (4, 2, 2))
    f, _ = R.rotary_frequencies(D)
    pos = torch.arange(8, dtype=torch.int32).cuda()
    # the cache is pages 1 .. 4 of larger buffers
    whole = R.KvCache.empty(6, 2, 16, D, fp8=fp8)
    for x in whole:
        if x is not None:
            x.view(torch.uint8).fill_(7)
    cache = R.KvCache(*(x if x is None else x[1:5] for x in whole))
    before = [x if x is None else x.clone() for x in whole]
    pages = _i32(*range(4), *range(4), 3, 1, 0, 2).view(3, 4)
    out = torch.full((10, 4, D), 3.0, dtype=torch.bfloat16, device="cuda")
    R.rotary_append(q, k, v, pos, f, cache, pages, _i32(5, 6, 0, 8), _i32(0, 0, 0), out=out[1:9])
    torch.cuda.synchronize()
    # rows 6 and 7 are found in the last sequence (rows 0 .. 7, slots of the same numbers)
    want = R.rotary(q, pos, f)
    assert torch.equal(out[7:9], want[6:]) and (out[:7] == 3).all() and (out[9] == 3).all()
    for x, y in zip(whole, before):
        if x is not None:
            changed = (x.view(torch.uint8) != y.view(torch.uint8)).view(6, 2, 16, -1).any(dim=3)
            at = torch.zeros_like(changed)
            at[4, :, 6:8] = True   # page 3 of the cache
            assert torch.equal(changed, at)
