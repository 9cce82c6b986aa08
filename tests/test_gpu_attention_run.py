"""The attention operators one after the other, as a program that serves a model calls
them: a prompt in pieces, single tokens, a tree of drafted tokens of which some are
accepted, against attention in 64 bits over everything that was appended; and a layer's
half with fp8_rmsnorm and fp8_linear around them.  And what the wrappers refuse."""
import math
import random

import pytest
import torch
import torch.autograd.forward_ad as fwd

from attention_reference import e4m3, rotated
from test_gpu_tree_attention import _gen, _randn, compare, make_cache, make_tree

pytestmark = pytest.mark.gpu


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,Hq,heads,page", [(64, 6, 2, 16), (128, 5, 1, 48), (256, 4, 4, 7)])
def test_prompt_tokens_and_trees(D, Hq, heads, page, interleaved, fp8):
    """Each step's attention against 64 bits over the cache, and the cache against the keys
    and values that went into it."""
    import rans_vectoradd as R
    g, rng = _gen(D + page), random.Random(D)
    B, most = 3, 200
    per = -(-most // page)
    cache = R.KvCache.empty(B * per, heads, page, D, fp8=fp8)
    order = list(range(B * per))
    rng.shuffle(order)
    pages = _i32(*order).view(B, per)
    f, m = R.rotary_frequencies(D, scaling="yarn", factor=4.0)
    lens = [0] * B
    kept = [[] for _ in range(B)]   # (k row turned, v row) of each slot, in 64 bits

    def step(counts, tree=False):
        nonlocal lens
        N = sum(counts)
        qkv = _randn(g, N, Hq + 2 * heads, D).to(torch.bfloat16)
        q, k, v = qkv.split((Hq, heads, heads), dim=1)
        starts = [0]
        for t in counts:
            starts.append(starts[-1] + t)
        mask = make_tree(rng, counts, max(counts)) if tree else None
        if tree:   # a token's position is its slot's context and the tokens above it
            depth = mask.sum(dim=1).tolist()
            pos = [lens[b] + depth[n] - 1 for b in range(B) for n in range(starts[b], starts[b + 1])]
        else:
            pos = [lens[b] + t for b in range(B) for t in range(counts[b])]
        pos, st, ctx = _i32(*pos), _i32(*starts), _i32(*lens)
        turned = R.rotary_append(q, k, v, pos, f, cache, pages, st, ctx, interleaved=interleaved, magnitude=m)
        o = compare(turned, cache, pages, st, ctx, mask)
        kt = rotated(k, pos, f, interleaved, m)
        for b in range(B):
            del kept[b][lens[b]:]
            kept[b] += [(kt[n], v[n].double()) for n in range(starts[b], starts[b + 1])]
        return o, [lens[b] + counts[b] for b in range(B)]

    _, lens = step([100, 7, 0])        # pieces of prompts
    _, lens = step([1, 60, 33])
    for _ in range(3):                 # tokens
        _, lens = step([1, 1, 1])
    for _ in range(2):                 # drafted ones, of which the first few are accepted
        step([9, 4, 17], tree=True)
        _, lens = step([2, 1, 3])
    k, v, ks, vs = cache
    for b in range(B):
        for s, (kw, vw) in enumerate(kept[b][:lens[b]]):
            at = (int(pages[b, s // page]), slice(None), s % page)
            for x, scale, want in ((k, ks, kw), (v, vs, vw)):
                got = x[at].double() if scale is None else e4m3(x[at]) * scale[at].double()[:, None]
                # (bf16: half a step; 8 bits: half a step of the value or of the smallest, 2^-10 of the
                # scale; and what 32 bits lose of the turned pairs)
                top = want.abs().amax(dim=1, keepdim=True)
                lim = want.abs() * (2.0 ** -8 if scale is None else 2.0 ** -4) * (1 + 2.0 ** -12) + top * 2.0 ** -17
                if scale is not None:
                    lim = lim + top / 448.0 * 2.0 ** -10
                assert ((got - want).abs() <= lim).all(), (b, s)


def test_half_a_layer():
    """Norm, qkv product, positions into the cache, attention, output product with the
    residual: every step's output goes into the next one, and a graph of the five calls
    gives the same bits."""
    import rans_vectoradd as R
    g = _gen(21)
    N, H, Hq, heads, D = 12, 256, 8, 2, 64
    x = _randn(g, N, H).to(torch.bfloat16)
    w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    wqkv, sqkv = R.fp8_quantize_rows((_randn(g, (Hq + 2 * heads) * D, H) / 16).to(torch.bfloat16))
    wo, so = R.fp8_quantize_rows((_randn(g, H, Hq * D) / 22).to(torch.bfloat16))
    cache = make_cache(g, 12, heads, 16, D, True)
    pages = torch.arange(12, dtype=torch.int32).cuda().view(3, 4)
    starts, lens, pos = _i32(0, 4, 5, 12), _i32(17, 40, 0), _i32(17, 18, 19, 20, 40, 0, 1, 2, 3, 4, 5, 6)
    f, _ = R.rotary_frequencies(D)

    def half():
        a, s = R.fp8_rmsnorm(x, w)[:2]
        qkv = R.fp8_linear(a, s, wqkv, sqkv).view(N, Hq + 2 * heads, D)
        q, k, v = qkv.split((Hq, heads, heads), dim=1)
        q = R.rotary_append(q, k, v, pos, f, cache, pages, starts, lens)
        o = R.tree_attention(q, cache, pages, starts, lens, max_tokens=7)
        oq, os_ = R.fp8_quantize_rows(o.view(N, Hq * D))
        return q, o, R.fp8_linear(oq, os_, wo, so, residual=x)
    q, o, y = half()
    compare(q, cache, pages, starts, lens, max_tokens=7)
    oq, os_ = R.fp8_quantize_rows(o.view(N, Hq * D))
    want = (e4m3(oq) * os_.double()[:, None]) @ (e4m3(wo) * so.double()[:, None]).t().contiguous() + x.double()
    # (the product's sums in 32 bits of 512 terms, and its rounding)
    lim = want.abs() * 2.0 ** -8 + ((e4m3(oq).abs() * os_.double()[:, None])
                                   @ (e4m3(wo).abs() * so.double()[:, None]).t().contiguous()) * 512 * 2.0 ** -23
    assert ((y.double() - want).abs() <= lim * (1 + 2.0 ** -7)).all()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        held = half()
    for i in range(3):
        x.copy_(_randn(g, N, H))
        gr.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, half()):
            assert torch.equal(a, b), f"replay {i}"


def _case():
    g = _gen(5)
    import rans_vectoradd as R
    f, _ = R.rotary_frequencies(64)
    return {"q": _randn(g, 4, 4, 64).to(torch.bfloat16), "k": _randn(g, 4, 2, 64).to(torch.bfloat16),
            "v": _randn(g, 4, 2, 64).to(torch.bfloat16), "pos": _i32(0, 1, 2, 3), "f": f,
            "cache": make_cache(g, 2, 2, 16, 64, False), "pages": _i32(1).view(1, 1), "starts": _i32(0, 4),
            "lens": _i32(0), "mask": torch.ones(4, 4, dtype=torch.bool, device="cuda")}


def _calls():
    import rans_vectoradd as R
    return {"rotary": lambda c, **kw: R.rotary(c["q"], c["pos"], c["f"], **kw),
            "append": lambda c, **kw: R.rotary_append(c["q"], c["k"], c["v"], c["pos"], c["f"], c["cache"], c["pages"],
                                                      c["starts"], c["lens"], **kw),
            "attend": lambda c, **kw: R.tree_attention(c["q"], c["cache"], c["pages"], c["starts"], c["lens"], c["mask"],
                                                       **kw)}


def test_refusals():
    import rans_vectoradd as R
    calls = _calls()

    def refuses(match, names="rotary append attend", kw={}, **change):
        for n in names.split():
            with pytest.raises(RuntimeError, match=match):
                calls[n]({**_case(), **change}, **kw)
    c = _case()
    for n in calls:
        calls[n](_case())
    refuses("q must be|x must be", q=c["q"].float())
    refuses("contiguous", q=c["q"].transpose(1, 2))
    refuses(r"\[N, H, D\]", q=c["q"][0])
    refuses("requires a gradient", q=c["q"].clone().requires_grad_())
    refuses("k must be", "append", k=c["k"].half())
    refuses("as the cache's rows", "append", k=c["k"][:3])
    refuses("as the cache's rows", "append", v=c["v"][:, :1])
    refuses("as the cache's rows", "attend", q=c["q"][..., :32].contiguous())
    refuses("positions must be", "rotary append", pos=c["pos"].long())
    refuses("positions must be", "rotary append", pos=c["pos"][:3])
    refuses("frequencies must be", "rotary append", f=c["f"].float())
    refuses("frequencies", "rotary append", f=None)
    refuses("rotated part", "rotary append", f=c["f"][:7])
    refuses("rotated part", "rotary append", f=torch.ones(40, dtype=torch.float64, device="cuda"))
    refuses("magnitude must be a number", "rotary append", kw={"magnitude": "x"})
    refuses("KvCache", "append attend", cache=None)
    refuses("the cache's k", "append attend", cache=R.KvCache(c["cache"].k.cpu(), c["cache"].v))
    refuses("the cache's", "append attend", cache=R.KvCache(c["cache"].k, c["cache"].v[:1]))
    refuses("the cache's", "append attend", cache=R.KvCache(c["cache"].k, c["cache"].v, torch.ones(2, 2, 16, device="cuda")))
    e = make_cache(_gen(1), 2, 2, 16, 64, True)
    refuses("scales must be|the cache's", "append attend", cache=R.KvCache(e.k, e.v, e.k_scale, e.v_scale[:1]))
    refuses("the cache's", "append attend", cache=R.KvCache(e.k, e.v))
    refuses("pages must be", "append attend", pages=c["pages"].long())
    refuses("pages must be", "append attend", pages=c["pages"][0])
    refuses("starts must be", "append attend", starts=c["starts"][:1])
    refuses("lens must be", "append attend", lens=c["starts"])
    refuses("mask must be", "attend", mask=c["mask"].to(torch.uint8))
    refuses("mask must be", "attend", mask=c["mask"][:3])
    refuses("scale", "attend", kw={"scale": -1.0})
    refuses("scale must be a number", "attend", kw={"scale": "x"})
    refuses("max_tokens", "attend", kw={"max_tokens": -1})
    refuses("max_tokens", "attend", kw={"max_tokens": 1.5})
    refuses("out must be", kw={"out": torch.empty(4, 4, 32, dtype=torch.bfloat16, device="cuda")})
    refuses("out must be", kw={"out": torch.empty(4, 4, 64, device="cuda")})


def test_inputs_with_a_tangent_are_refused():
    calls = _calls()
    for n, name in (("rotary", "x"), ("append", "q"), ("attend", "q")):
        with fwd.dual_level():
            c = _case()
            c["q"] = fwd.make_dual(c["q"], torch.ones_like(c["q"]))
            with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
                calls[n](c)
    with torch.no_grad():   # what requires a gradient is taken where none is recorded
        for n in calls:
            c = _case()
            c["q"].requires_grad_()
            calls[n](c)


def test_buffers_and_masks_of_other_widths():
    """out in a larger buffer; masks with fewer and more columns than new tokens."""
    import rans_vectoradd as R
    c = _case()
    a = (c["q"], c["cache"], c["pages"], c["starts"], c["lens"])
    whole = R.tree_attention(*a, c["mask"])
    buf = torch.full((6, 4, 64), 2.0, dtype=torch.bfloat16, device="cuda")
    assert R.tree_attention(*a, c["mask"], out=buf[1:5]).data_ptr() == buf[1:5].data_ptr()
    assert torch.equal(buf[1:5], whole) and (buf[0] == 2).all() and (buf[5] == 2).all()
    wide = torch.ones(4, 9, dtype=torch.bool, device="cuda")
    assert torch.equal(R.tree_attention(*a, wide, max_tokens=4), whole)
    two = c["mask"].clone()
    two[:, 2:] = False
    assert torch.equal(R.tree_attention(*a, c["mask"][:, :2].contiguous(), max_tokens=4),
                       R.tree_attention(*a, two))
    assert (R.tree_attention(*a, torch.ones(4, 0, dtype=torch.bool, device="cuda")) == 0).all()
    assert math.isfinite(whole.float().abs().max().item())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_outputs_over_the_queries(D, fp8):
    """In every kernel, whole items and shared ones."""
    import rans_vectoradd as R
    g = _gen(D)
    for tokens, context in ((1, 90), (1, 3000), (9, 2000), (13, 500), (30, 1500), (70, 20), (70, 2500)):
        cache = make_cache(g, -(-(context + tokens) // 16), 4, 16, D, fp8)
        pages = torch.arange(cache.k.shape[0], dtype=torch.int32).cuda().view(1, -1)
        q = _randn(g, tokens, 16, D).to(torch.bfloat16)
        want = R.tree_attention(q, cache, pages, _i32(0, tokens), _i32(context))
        same = q.clone()
        assert R.tree_attention(same, cache, pages, _i32(0, tokens), _i32(context), out=same) is same
        assert torch.equal(same, want), (tokens, context)
    k, v = (_randn(g, 70, 4, D).to(torch.bfloat16) for _ in range(2))
    f, _ = R.rotary_frequencies(D)
    pos = torch.arange(70, dtype=torch.int32).cuda()
    for interleaved in (False, True):
        want = R.rotary(q, pos, f, interleaved=interleaved)
        same = q.clone()
        R.rotary_append(same, k, v, pos, f, cache, pages, _i32(0, 70), _i32(context), interleaved=interleaved, out=same)
        assert torch.equal(same, want)


def test_many_sequences_of_nothing():
    """Sequences without new tokens between others, none at all, and B above the tokens."""
    import rans_vectoradd as R
    g = _gen(6)
    cache = make_cache(g, 40, 2, 16, 64, False)
    B = 1000
    pages = torch.randint(0, 40, (B, 12), generator=g, device="cuda").to(torch.int32)
    counts = [1 if b % 97 == 5 else 0 for b in range(B)]
    starts = _i32(*[sum(counts[:b]) for b in range(B + 1)])
    lens = torch.randint(0, 150, (B,), generator=g, device="cuda").to(torch.int32)
    q = _randn(g, sum(counts), 6, 64).to(torch.bfloat16)
    compare(q, cache, pages, starts, lens, max_tokens=1)
    out = torch.full_like(q, 4.0)
    R.tree_attention(q, cache, pages, torch.zeros_like(starts), lens, out=out)
    assert (out == 4).all()
    wide = torch.cat((pages, pages), dim=1)   # (items shared by workgroups, none of them any)
    R.tree_attention(q, cache, wide, torch.zeros_like(starts), lens, out=out)
    assert (out == 4).all()
    compare(q, cache, wide, starts, lens, max_tokens=1)
