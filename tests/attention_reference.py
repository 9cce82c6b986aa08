"""Rotary positions, the paged cache and attention over it in 64 bits, written from
their definitions with loops over sequences and heads, for the tests."""
import math

import torch


def e4m3(b):
    return b.view(torch.float8_e4m3fn).to(torch.float32).double()


def rotated(x, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False):
    y = x.double().clone()
    n = frequencies.numel()
    a = positions.double()[:, None, None] * frequencies.double()[None, None, :]
    if inverse:
        a = -a
    u, v = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    xu, xv = x.double()[..., u], x.double()[..., v]
    y[..., u] = magnitude * (xu * torch.cos(a) - xv * torch.sin(a))
    y[..., v] = magnitude * (xu * torch.sin(a) + xv * torch.cos(a))
    return y


def rows_of(cache, b_pages, slots):
    """(K, V, exists) [slots, heads, D] in 64 bits of a sequence's slots."""
    k, v, ks, vs = cache
    pages, heads, page, D = k.shape
    s = torch.arange(slots, device=k.device)
    p = b_pages[torch.div(s, page, rounding_mode="floor")].long()
    ok = (p >= 0) & (p < pages)
    p = torch.where(ok, p, 0)
    at = (p[:, None], torch.arange(heads, device=k.device)[None, :], (s % page)[:, None])
    if ks is None:
        return k[at].double(), v[at].double(), ok
    return e4m3(k[at]) * ks[at].double()[..., None], e4m3(v[at]) * vs[at].double()[..., None], ok


def attention(q, cache, pages, starts, lens, mask, scale):
    """(o, spread, off): the result [N, Hq, D]; sum p |v| / sum p, what roundings of
    the probabilities are relative to; and of each row the largest sum |q k| scale, what
    the scores' are.  Rows of no sequence are NaN."""
    N, Hq, D = q.shape
    heads, page = cache[0].shape[1], cache[0].shape[2]
    G = Hq // heads
    o = torch.full((N, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    spread, off = torch.zeros_like(o), torch.zeros(N, Hq, dtype=torch.float64, device=q.device)
    capacity = pages.shape[1] * page
    st = [min(max(int(x), 0), N) for x in starts.tolist()]
    for b, c in enumerate(lens.tolist()):
        n0, n1 = st[b], st[b + 1]
        T = n1 - n0
        if T <= 0:
            continue
        c = min(max(c, 0), capacity)
        slots = min(c + T, capacity)
        K, V, ok = rows_of(cache, pages[b], slots)
        j = torch.arange(slots, device=q.device) - c
        t = torch.arange(T, device=q.device)
        if mask is None:
            sees = j[None, :] <= t[:, None]
        else:
            W = mask.shape[1]
            sees = (j < 0)[None, :].expand(T, slots).clone()
            new = (j >= 0) & (j < W)
            sees[:, new] = mask[n0:n1][:, j[new]]
        sees = sees & ok[None, :]
        for h in range(Hq):
            qh, kh, vh = q[n0:n1, h].double(), K[:, h // G], V[:, h // G]
            # what a row does not see is left out row by row: it may be infinite or NaN
            s = torch.where(sees, (qh @ torch.nan_to_num(kh, 0.0, 0.0, 0.0).t().contiguous()) * scale, -math.inf)
            bad_k = ~torch.isfinite(kh).all(dim=1)
            s = torch.where(sees & bad_k[None, :], math.nan, s)
            m = s.amax(dim=1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
            p = torch.where(sees, p, 0.0)
            l = p.sum(dim=1, keepdim=True)
            clean = torch.nan_to_num(vh, 0.0, 0.0, 0.0)
            r = (p @ clean) / torch.where(l == 0, 1.0, l)
            if not torch.isfinite(vh).all():
                for i in torch.nonzero(~torch.isfinite(vh).all(dim=1)).flatten().tolist():
                    hit = ~torch.isfinite(vh[i])[None, :] & sees[:, i:i + 1]
                    r = torch.where(hit, r + vh[i][None, :], r)
            o[n0:n1, h] = r
            spread[n0:n1, h] = (p @ clean.abs()) / torch.where(l == 0, 1.0, l)
            a = qh.abs() @ torch.nan_to_num(kh, 0.0, 0.0, 0.0).abs().t().contiguous() * scale
            off[n0:n1, h] = torch.where(sees, a, 0.0).amax(dim=1) if slots else 0.0
    return o, spread, off


def check(got, want, spread, off, D):
    """The kernel's roundings, from its arithmetic.  Probabilities are rounded to bf16
    (2^-8 of each at most) for the product with v, the result once more (2^-8 of it).
    A score is a sum of D products in 32 bits (each step 2^-24 of the sum of their
    absolute values, and bf16 matrix instructions cut off at 2^-24 as well) and goes
    with a handful of roundings of itself into the exponent: a relative error of the
    probability of (2 D + 8) 2^-24 off, in numerator and sum.  Joining parts and
    scales: 2^-16 of the spread covers some hundreds of 32-bit roundings."""
    assert torch.isfinite(got.double()).equal(torch.isfinite(want))
    fine = torch.isfinite(want)
    lim = (2.0 ** -8 * want.abs() * (1 + 2.0 ** -7)
           + spread * (2.0 ** -8 + 2.0 ** -16 + 2 * (2 * D + 8) * 2.0 ** -24 * off[..., None]) * (1 + 2.0 ** -7)
           + 2.0 ** -126)
    bad = ((got.double() - want).abs() > lim) & fine
    assert not bad.any(), (f"{bad.sum().item()} outputs are off, the first at {torch.nonzero(bad)[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}")
