"""rotary and rotary_append (no counterpart in the reference) against rotations in 64
bits (attention_reference.py)."""
import math
import random

import pytest
import torch

from attention_reference import e4m3, rotated
from test_gpu_tree_attention import _gen, _randn, make_batch, make_cache

pytestmark = pytest.mark.gpu


def _say(msg):
    print(msg, flush=True)


def limits(x, positions, frequencies, interleaved, magnitude, want):
    """How far 32 bits may be off, from the kernel's arithmetic.  The frequency in turns
    has two roundings in 64 bits (2^-53 of it each), so the angle is off by 2^-52 of itself
    and three last bits of a 32-bit fraction of a turn (2^-27.8 radians); sine and cosine
    and their products and sum are a dozen roundings of 2^-24 of |u| + |v|, below 2^-20.
    What is copied is exact."""
    n = frequencies.numel()
    u, v = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    far = positions.double().abs()[:, None, None] * frequencies.double()
    one = (x[..., u].double().abs() + x[..., v].double().abs()) * abs(magnitude) * (2.0 ** -20 + far * 2.0 ** -51)
    lim = torch.zeros_like(want)
    lim[..., u], lim[..., v] = one, one
    return lim


def close(got, want, lim):
    """lim, and the rounding to bf16 (2^-8 of the value; half the smallest step)."""
    bad = (got.double() - want).abs() > (want.abs() + lim) * 2.0 ** -8 + lim + 2.0 ** -134
    assert not bad.any(), (f"{bad.sum().item()} off, the first at {torch.nonzero(bad)[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N,H,D,rot,far", [
    (1, 1, 16, 16, 1), (1, 48, 128, 128, 5000), (7, 1, 64, 32, 100), (3, 5, 80, 32, 1 << 20), (65, 9, 80, 80, 1 << 24),
    (257, 2, 256, 64, (1 << 31) - 1), (33, 65, 16, 16, 10), (100, 3, 1024, 1024, 4096), (5, 7, 1008, 496, 1 << 30),
    (2000, 12, 128, 128, 131072), (4099, 1, 48, 16, 99)])
def test_matches_64_bits(N, H, D, rot, far, interleaved):
    import rans_vectoradd as R
    _say(f"case: rotary {N} x {H} x {D}, {rot} turned, positions to {far}, interleaved={interleaved}")
    g = _gen(N + D)
    x = _randn(g, N, H, D).to(torch.bfloat16)
    p = torch.randint(-far, far + 1, (N,), generator=g, device="cuda").to(torch.int32)
    p[0] = far
    for scaling, factor in (("none", 1.0), ("yarn", 8.0), ("ntk", 3.0), ("linear", 5.0)):
        f, magnitude = R.rotary_frequencies(rot, scaling=scaling, factor=factor)
        for inverse in (False, True):
            got = R.rotary(x, p, f, interleaved=interleaved, magnitude=magnitude, inverse=inverse)
            want = rotated(x, p, f, interleaved, magnitude, inverse)
            close(got, want, limits(x, p, f, interleaved, magnitude, want))
            assert torch.equal(got[..., rot:], x[..., rot:])
            assert torch.equal(got, R.rotary(x, p, f, interleaved=interleaved, magnitude=magnitude, inverse=inverse))


def test_rows_in_longer_rows_in_place_and_into_a_buffer():
    import rans_vectoradd as R
    g = _gen(2)
    f, _ = R.rotary_frequencies(64)
    wide = _randn(g, 37, 11, 64).to(torch.bfloat16)
    p = torch.arange(37, dtype=torch.int32).cuda()
    x = wide[:, 2:7]
    want = R.rotary(x.contiguous(), p, f)
    assert torch.equal(R.rotary(x, p, f), want)
    out = torch.full((39, 5, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    assert R.rotary(x, p, f, out=out[1:38]).data_ptr() == out[1:38].data_ptr()
    assert torch.equal(out[1:38], want) and (out[0] == 7).all() and (out[38] == 7).all()
    same = x.contiguous()
    assert torch.equal(R.rotary(same, p, f, out=same), want)
    # (every second head of a row is no run of heads)
    with pytest.raises(RuntimeError, match="contiguous"):
        R.rotary(wide[:, ::2], p, f)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        R.rotary(_randn(g, 4, 67).to(torch.bfloat16)[:, :64].unsqueeze(1), p[:4], f)


def test_infinities_and_nan_stay_in_their_pairs():
    import rans_vectoradd as R
    f, _ = R.rotary_frequencies(32)
    x = torch.ones(4, 3, 48, dtype=torch.bfloat16, device="cuda")
    x[1, 1, 5], x[2, 2, 40] = math.inf, math.nan
    p = torch.arange(4, dtype=torch.int32).cuda()
    got = R.rotary(x, p, f)
    clean = x.clone()
    clean[1, 1, 5], clean[2, 2, 40] = 1, 1
    want = R.rotary(clean, p, f)
    bad = ~torch.isfinite(got)
    assert set(map(tuple, torch.nonzero(bad).tolist())) == {(1, 1, 5), (1, 1, 21), (2, 2, 40)}
    assert torch.equal(got[~bad], want[~bad])


def test_none_and_one():
    import rans_vectoradd as R
    f, _ = R.rotary_frequencies(32)
    none = torch.empty(0, 3, 64, dtype=torch.bfloat16, device="cuda")
    assert R.rotary(none, torch.empty(0, dtype=torch.int32, device="cuda"), f).shape == (0, 3, 64)
    x = _randn(_gen(3), 1, 3, 64).to(torch.bfloat16)
    assert torch.equal(R.rotary(x, torch.zeros(1, dtype=torch.int32, device="cuda"), f), x)


def test_the_inverse_is_the_gradient():
    """The rotation's gradient by the formula (the transposed matrix) and by differences,
    against inverse=True."""
    import rans_vectoradd as R
    g = _gen(4)
    for interleaved in (False, True):
        f, m = R.rotary_frequencies(48, scaling="yarn", factor=2.0)
        x, w = (_randn(g, 9, 2, 64).to(torch.bfloat16) for _ in range(2))
        p = torch.randint(0, 9000, (9,), generator=g, device="cuda").to(torch.int32)
        got = R.rotary(w, p, f, interleaved=interleaved, magnitude=m, inverse=True)
        y = x.double().requires_grad_()
        (rotated(y, p, f, interleaved, m) * w.double()).sum().backward()
        # (reference.rotated clones x: the gradient is that of the whole operator)
        want = y.grad
        close(got, want, limits(w, p, f, interleaved, m, want))
        step = torch.zeros_like(y.detach())
        for at in ((0, 0, 0), (4, 1, 30), (8, 0, 47), (3, 1, 63)):
            step[at] = 1.0   # (linear: any step)
            d = ((rotated(x.double() + step, p, f, interleaved, m) - rotated(x.double(), p, f, interleaved, m))
                 * w.double()).sum()
            assert abs(d - want[at]) < 1e-9
            step[at] = 0.0


# -- with the writing into the cache ---------------------------------------------


def _append_case(g, rng, lens, counts, Hq, heads, D, page, fp8):
    pages, starts, ctx, total = make_batch(rng, lens, counts, page)
    cache = make_cache(g, total, heads, page, D, fp8)
    N = sum(counts)
    qkv = _randn(g, N + 2, Hq + 2 * heads, D).to(torch.bfloat16)
    q, k, v = qkv[:N].split((Hq, heads, heads), dim=1)
    p = torch.randint(0, 1 << 20, (N,), generator=g, device="cuda").to(torch.int32)
    return q, k, v, p, cache, pages, starts, ctx


def _written(lens, counts, pages, page, total):
    """(row of q, page, row of the page) of every token whose slot the table has."""
    table, n, rows = pages.tolist(), 0, []
    for b, (c, t) in enumerate(zip(lens, counts)):
        for i in range(t):
            s = max(c, 0) + i
            if s < len(table[b]) * page and 0 <= table[b][s // page] < total:
                rows.append((n, table[b][s // page], s % page))
            n += 1
    return rows


def check_append(q, k, v, p, cache, pages, starts, ctx, lens, counts, interleaved, rot=None):
    import rans_vectoradd as R
    D, page, total = q.shape[2], cache.k.shape[2], cache.k.shape[0]
    f, m = R.rotary_frequencies(rot or D, scaling="yarn", factor=4.0)
    before = [None if x is None else x.clone() for x in cache]
    got = R.rotary_append(q, k, v, p, f, cache, pages, starts, ctx, interleaved=interleaved, magnitude=m)
    assert torch.equal(got, R.rotary(q, p, f, interleaved=interleaved, magnitude=m))
    want = rotated(q, p, f, interleaved, m)
    close(got, want, limits(q, p, f, interleaved, m, want))
    rows = _written(lens, counts, pages, page, total)
    n = torch.tensor([r[0] for r in rows], dtype=torch.long).cuda()
    at = (torch.tensor([r[1] for r in rows], dtype=torch.long).cuda(), slice(None),
          torch.tensor([r[2] for r in rows], dtype=torch.long).cuda())
    if cache.k_scale is None:
        assert torch.equal(cache.k[at], R.rotary(k, p, f, interleaved=interleaved, magnitude=m)[n])
        assert torch.equal(cache.v[at], v[n])
    else:
        # v is what fp8_quantize_rows makes of it; k from 32 bits
        b, s = R.fp8_quantize_rows(v[n].reshape(-1, D))
        assert torch.equal(cache.v[at].reshape(-1, D), b) and torch.equal(cache.v_scale[at].flatten(), s)
        want = rotated(k, p, f, interleaved, m)[n]
        lim = limits(k, p, f, interleaved, m, rotated(k, p, f, interleaved, m))[n]
        amax, off = want.abs().amax(dim=2), lim.amax(dim=2)
        scale = cache.k_scale[at].double()
        assert ((scale * 448.0 - amax).abs() <= off + amax * 2.0 ** -22).all()
        # half a step of E4M3: 2^-4 of the value, or 2^-10 where it is subnormal; the quotient's
        # own roundings are 2^-22 of it
        x = e4m3(cache.k[at]) * scale[..., None]
        bad = (x - want).abs() > (want.abs() + lim) * 2.0 ** -4 * (1 + 2.0 ** -18) + lim + scale[..., None] * 2.0 ** -10
        assert not bad.any(), torch.nonzero(bad)[0].tolist()
    # nothing else was written
    left = torch.ones(cache.k.shape[0], page, dtype=torch.bool, device="cuda")
    left[at[0], at[2]] = False
    for x, y in zip(cache, before):
        if x is not None:
            assert torch.equal(x.transpose(1, 2)[left].view(torch.uint8), y.transpose(1, 2)[left].view(torch.uint8))
    return got


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lens,counts,Hq,heads,D,page", [
    ([0], [1], 1, 1, 64, 1), ([700], [1], 40, 8, 128, 16), ([15, 16, 17, 0], [1, 1, 1, 1], 8, 2, 256, 16),
    ([5, 0, 31], [9, 0, 40], 6, 3, 64, 48), ([100] * 70, [1 + i % 4 for i in range(70)], 4, 4, 128, 20),
    ([1, 2000], [700, 3], 10, 2, 64, 64), ([3, 0], [600, 1000], 5, 5, 128, 100), ([9], [257], 65, 65, 256, 7)])
def test_append_matches_64_bits(lens, counts, Hq, heads, D, page, interleaved, fp8):
    _say(f"case: append {lens[:4]} {counts[:4]} {Hq}/{heads} x {D} page={page} interleaved={interleaved} fp8={fp8}")
    g, rng = _gen(sum(lens) + D), random.Random(page)
    q, k, v, p, cache, pages, starts, ctx = _append_case(g, rng, lens, counts, Hq, heads, D, page, fp8)
    check_append(q, k, v, p, cache, pages, starts, ctx, lens, counts, interleaved)
    if D > 64:
        check_append(q, k, v, p, cache, pages, starts, ctx, lens, counts, interleaved, rot=48)


@pytest.mark.parametrize("fp8", [False, True])
def test_append_bounds_every_number(fp8):
    """Negative lengths, slots past the table, entries that are no page, and rows of q of
    no sequence: in range, and the others as without them."""
    import rans_vectoradd as R
    g, rng = _gen(7), random.Random(7)
    lens, counts = [-3, 40, 10, 5], [4, 9, 6, 2]
    q, k, v, p, cache, pages, starts, ctx = _append_case(g, rng, [0, 40, 10, 5], counts, 4, 2, 128, 16, fp8)
    pages, ctx = pages[:, :3].contiguous(), torch.tensor(lens, dtype=torch.int32).cuda()   # 48 slots: 40 + 9 is one more
    pages[2, 0] = cache.k.shape[0]
    pages[3, 0] = -1
    check_append(q, k, v, p, cache, pages, starts, ctx, lens, counts, False)
    # rows before the first sequence and behind the last are left
    f, _ = R.rotary_frequencies(128)
    out = torch.full((21, 4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([2, 6, 15, 15, 19], dtype=torch.int32).cuda()
    R.rotary_append(q, k, v, p, f, cache, pages, some, ctx, out=out)
    want = R.rotary(q, p, f)
    assert torch.equal(out[2:19], want[2:19]) and (out[:2] == 3).all() and (out[19:] == 3).all()
    # starts out of range and going back: whatever they give, nothing outside is touched
    guard = torch.full((5, 21, 4, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    R.rotary_append(q, k, v, p, f, cache, pages, torch.tensor([-7, 99, 3, 50, 1 << 30], dtype=torch.int32).cuda(),
                    torch.tensor([1 << 30, -(1 << 31), 47, 48], dtype=torch.int32).cuda(), out=guard[2])
    torch.cuda.synchronize()
    assert (guard[:2] == 9).all() and (guard[3:] == 9).all()


def test_append_rows_of_zeros_infinities_and_nan():
    """Rows of zeros get the smallest scale and zero bytes; others' rows are not reached."""
    import rans_vectoradd as R
    f, _ = R.rotary_frequencies(64)
    cache = make_cache(_gen(1), 2, 2, 16, 64, True)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    v = torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    v[1, 0, 3] = math.nan
    i = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()   # noqa: E731
    R.rotary_append(v, k, v, i(0, 1, 2), f, cache, i(1).view(1, 1), i(0, 3), i(0))
    assert (cache.k[1, :, :3] == 0).all()
    assert torch.equal(cache.k_scale[1, :, :3], torch.full((2, 3), 2.0 ** -100 / 448.0, device="cuda"))
    b, s = R.fp8_quantize_rows(v.reshape(-1, 64))
    assert torch.equal(cache.v[1, :, :3].transpose(0, 1).reshape(-1, 64), b)
    assert torch.equal(cache.v_scale[1, :, :3].t().flatten().view(torch.int32), s.view(torch.int32))


def test_append_on_another_stream_and_in_graphs():
    import rans_vectoradd as R
    g, rng = _gen(9), random.Random(9)
    lens, counts = [30, 3], [2, 5]
    q, k, v, p, cache, pages, starts, ctx = _append_case(g, rng, lens, counts, 4, 2, 64, 16, True)
    f, _ = R.rotary_frequencies(64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = R.rotary_append(q, k, v, p, f, cache, pages, starts, ctx)
    side.synchronize()
    assert torch.equal(got, R.rotary(q, p, f))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = R.rotary_append(q, k, v, p, f, cache, pages, starts, ctx)
    for i in range(4):
        q.copy_(_randn(g, *q.shape))
        k.copy_(_randn(g, *k.shape))
        ctx.copy_(torch.tensor([[30, 3], [0, 1], [14, 27], [5, 0]][i], dtype=torch.int32))
        p.add_(1)
        gr.replay()
        torch.cuda.synchronize()
        after = [x.clone() for x in cache]
        assert torch.equal(o, R.rotary(q, p, f))
        for x in cache:
            x.zero_()
        gr.replay()
        eager = R.KvCache(*(torch.zeros_like(x) for x in cache))
        R.rotary_append(q, k, v, p, f, eager, pages, starts, ctx)
        torch.cuda.synchronize()
        for x, y in zip(cache, eager):
            assert torch.equal(x, y), f"replay {i}"
        for x, y in zip(cache, after):
            x.copy_(y)
