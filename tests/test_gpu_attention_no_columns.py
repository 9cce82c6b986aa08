"""tree_attention over page tables that have no column, or fewer than the tokens need, in
every kernel."""
import pytest
import torch

from test_gpu_tree_attention import _gen, _randn, compare, make_cache, run

pytestmark = pytest.mark.gpu


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tables_without_columns(D, page, fp8):
    g = _gen(D + page)
    cache = make_cache(g, 3, 2, page, D, fp8)
    none = torch.empty(2, 0, dtype=torch.int32).cuda()
    for tokens in (1, 3, 16, 65, 129, 200, 700):
        for Hq in (2, 6):
            print(f"case: no columns, D = {D}, page {page}, fp8={fp8}, {tokens} tokens, {Hq} heads", flush=True)
            q = _randn(g, tokens + 2, Hq, D).to(torch.bfloat16)
            a = (q, cache, none, _i32(0, tokens // 2, tokens), _i32(40, 0))
            for mask in (None, torch.ones(tokens + 2, 5, dtype=torch.bool, device="cuda")):
                for most in (None, 1, tokens):
                    out = run(*a, mask, max_tokens=most, out=torch.full_like(q, 3.0))
                    assert (out[:tokens] == 0).all() and (out[tokens:] == 3).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tables_shorter_than_the_tokens(D, fp8):
    g = _gen(D)
    cache = make_cache(g, 40, 2, 16, D, fp8)
    for columns, tokens, contexts in ((1, 300, (0, 5)), (3, 200, (47, 48)), (20, 400, (0, 311)), (20, 150, (300, 1000))):
        print(f"case: {columns} columns, D = {D}, fp8={fp8}, {tokens} tokens after {contexts}", flush=True)
        pages = torch.randint(0, 40, (2, columns), generator=g, device="cuda").to(torch.int32)
        q = _randn(g, tokens, 4, D).to(torch.bfloat16)
        compare(q, cache, pages, _i32(0, tokens // 3, tokens), _i32(*contexts))
