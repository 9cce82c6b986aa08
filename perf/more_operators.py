"""The operators of a layer's attention, as a program that serves a model with
drafted tokens calls them: rotary positions, rotary positions with the writing of
keys and values into a paged cache, and attention of each sequence's new tokens (a
tree, or a chain) over that cache.

listed() holds named cases, draw() more of the same ranges; prepare() makes what
such a program holds before the call, run() is one call (the plain form in torch's
elementary operations, or with `own` the framework's), work() what the call cannot
do without, exact() the result in 64 bits.

A batch is packed: the tokens of sequence b are rows starts[b] .. starts[b + 1] - 1.
They belong in the slots lens[b], lens[b] + 1, ... of the sequence, and slot s is
row s % page of the cache's page pages[b][s / page].  8-bit rows of a cache are
E4M3FN bytes with one float32 scale each, and are returned as float8_e4m3fn.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FP8_MAX = 448.0
AMAX_MIN = 2.0 ** -100   # rows of zeros get the scale of this maximum


def listed():
    return [
        # -- rotary positions: the q and k heads in the rows of a qkv product -------
        # one token of a decoding step: latency
        {"name": "rotary_1", "op": "rotary", "N": 1, "H": 48, "D": 128, "rot": 128,
         "interleaved": False, "scaling": "none", "far": 32768},
        # part of the head, pairs beside each other, positions far past the trained length
        {"name": "rotary_odd", "op": "rotary", "N": 1777, "H": 9, "D": 80, "rot": 32,
         "interleaved": True, "scaling": "yarn", "far": 1 << 20},
        # a batch of prompts
        {"name": "rotary_8192", "op": "rotary", "N": 8192, "H": 48, "D": 128, "rot": 128,
         "interleaved": False, "scaling": "linear", "far": 131072},
        # -- rotary positions, keys and values into the cache ----------------------
        # a decoding step of a few sequences
        {"name": "append_7", "op": "append", "B": 7, "tokens": 1, "Hq": 40, "Hkv": 8, "D": 128,
         "page": 16, "low": 100, "high": 4000, "fp8": False, "interleaved": False},
        # a tree of drafted tokens for each of many sequences, pages of no power of two
        {"name": "append_trees", "op": "append", "B": 61, "tokens": 25, "Hq": 16, "Hkv": 16, "D": 64,
         "page": 48, "low": 100, "high": 2000, "fp8": True, "interleaved": True},
        # prompts
        {"name": "append_prompts", "op": "append", "B": 4, "tokens": 2048, "Hq": 40, "Hkv": 8,
         "D": 128, "page": 64, "low": 1, "high": 100, "fp8": True, "interleaved": False},
        # -- attention of the new tokens over the cache ----------------------------
        # one token of one short conversation: latency
        {"name": "one_700", "op": "attention", "B": 1, "tokens": 1, "tree": False, "Hq": 40,
         "Hkv": 8, "D": 128, "page": 16, "low": 700, "high": 700, "fp8": False},
        # one long document's tree of drafted tokens
        {"name": "tree_32771", "op": "attention", "B": 1, "tokens": 61, "tree": True, "Hq": 40,
         "Hkv": 8, "D": 128, "page": 64, "low": 32771, "high": 32771, "fp8": False},
        # a serving batch: one token each, contexts of all lengths, 8-bit cache
        {"name": "batch_96", "op": "attention", "B": 96, "tokens": 1, "tree": False, "Hq": 40,
         "Hkv": 8, "D": 128, "page": 16, "low": 100, "high": 16000, "fp8": True},
        # trees of all sizes, a head of keys for each of the queries, odd pages
        {"name": "trees_17", "op": "attention", "B": 17, "tokens": 31, "tree": True, "Hq": 16,
         "Hkv": 16, "D": 64, "page": 48, "low": 300, "high": 9000, "fp8": True},
        # one token over the longest context
        {"name": "one_262144", "op": "attention", "B": 1, "tokens": 1, "tree": False, "Hq": 40,
         "Hkv": 8, "D": 128, "page": 256, "low": 262144, "high": 262144, "fp8": False},
        # the last piece of a long prompt
        {"name": "prompt_2048", "op": "attention", "B": 1, "tokens": 2048, "tree": False, "Hq": 40,
         "Hkv": 8, "D": 128, "page": 64, "low": 14000, "high": 14000, "fp8": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "append", "attention", "attention", "attention"))
    if op == "rotary":
        d = 16 * rng.randint(1, 16)
        h = _log_int(rng, 1, 64)
        return {"op": op, "N": min(_log_int(rng, 1, 16384), 8192 * 48 * 128 // (h * d)), "H": h, "D": d,
                "rot": rng.choice((d, 16 * rng.randint(1, d // 16))),
                "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(("none", "linear", "ntk", "yarn")),
                "far": _log_int(rng, 1000, 1 << 20)}
    d = rng.choice((64, 128, 128, 256))
    hkv = rng.choice((1, 2, 4, 8, 8, 16))
    hq = hkv * rng.randint(1, 64 // hkv if hkv > 4 else 16)
    page = rng.choice((16, 16, 32, 64, 256, rng.randint(1, 100)))
    case = {"op": op, "Hq": hq, "Hkv": hkv, "D": d, "page": page, "fp8": rng.random() < 0.5}
    b = _log_int(rng, 1, 128)
    if op == "append":
        t = min(_log_int(rng, 1, 2048), 5 * 1024 * 56 * 128 // (b * (hq + 2 * hkv) * d))
        high = min(_log_int(rng, 16, 4000), max(16, (1 << 27) // (b * hkv * d)))
        return {**case, "B": b, "tokens": max(1, t), "low": rng.randint(0, high), "high": high,
                "interleaved": rng.random() < 0.5}
    tree = rng.random() < 0.5
    t = _log_int(rng, 1, 128 if tree else 2048) if rng.random() < 0.7 else 1
    t = max(1, min(t, (1 << 26) // (b * hq * d)))
    high = min(_log_int(rng, 16, 262144), max(16, (3 << 26) // (b * hkv * d) - t))
    t = max(1, min(t, 2048 * 40 * 15000 * 128 // (b * hq * d * (high + t))))
    return {**case, "B": b, "tokens": t, "tree": tree,
            "low": _log_int(rng, 1, high) if rng.random() < 0.7 else high, "high": high}


# ---------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n lengths from lo to hi, spread over their logarithm, in no order."""
    if n == 1 or lo == hi:
        return [hi] * n
    at = [(i * 0.6180339887498949) % 1.0 for i in range(n)]
    at[0] = 1.0
    return [min(hi, max(lo, int(round(max(lo, 1) * (hi / max(lo, 1)) ** a)))) for a in at]


def _lens(case):
    """(tokens, context) of each sequence."""
    b, t = case["B"], case["tokens"]
    counts = _spread((t + 3) // 4, t, b) if case["op"] == "append" or case["tree"] else [t] * b
    return counts, _spread(case["low"], case["high"], b)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _frequencies(rot, scaling, original=4096, factor=8.0):
    """Radians a position of each pair, and the factor of the rotated vectors."""
    base, magnitude = 10000.0, 1.0
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        # pairs that turn often within the trained length keep their frequency, slow ones are
        # stretched, those between are blended
        def pair(turns):
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.cuda(), magnitude


def _rows_to_fp8(x):
    """E4M3FN bytes of the rows of x (overwritten) and their scales."""
    scale = x.abs().amax(dim=-1).clamp_(min=AMAX_MIN).div_(FP8_MAX)
    return x.div_(scale.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _tree(counts, width, g):
    """mask[n][j]: token n of its sequence sees the sequence's j-th: itself, its
    parent, and so on to the root.  Parents are among the four tokens before."""
    up = torch.randint(1, 5, (sum(counts),), generator=g, device="cuda").tolist()
    rows = []
    for c in counts:
        above = []
        for t in range(c):
            parent = t - up[len(rows) + t]
            row = list(above[parent]) if parent >= 0 else [False] * width
            row[t] = True
            above.append(row)
        rows += above
    return torch.tensor(rows, dtype=torch.bool).cuda()


def prepare(case, seed):
    g = _gen(seed)
    d = case["D"]
    s = {"op": case["op"], "interleaved": case.get("interleaved", False)}
    if case["op"] == "rotary":
        n, h = case["N"], case["H"]
        # the first heads of a wider row, as the product's output holds them
        s["x"] = _randn(g, n, h + 8, d).to(torch.bfloat16)[:, :h]
        s["frequencies"], s["magnitude"] = _frequencies(case["rot"], case["scaling"])
        s["positions"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda",
                                       dtype=torch.int32)
        return s
    counts, context = _lens(case)
    b, hq, hkv, page = case["B"], case["Hq"], case["Hkv"], case["page"]
    n = sum(counts)
    per = -(-max(c + t for c, t in zip(context, counts)) // page)
    need = [-(-(c + t) // page) for c, t in zip(context, counts)]
    total = sum(need)
    # pages in no order; entries past a sequence's last are not used
    order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32).tolist()
    table, at = [], 0
    for k in need:
        table.append(order[at:at + k] + [0] * (per - k))
        at += k
    s["pages"] = torch.tensor(table, dtype=torch.int32).cuda()
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    s["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
    s["lens"] = torch.tensor(context, dtype=torch.int32).cuda()
    s["most"] = max(counts)
    cache = []
    for _ in range(2):
        rows = _randn(g, total, hkv, page, d)
        cache.append(_rows_to_fp8(rows) if case["fp8"] else (rows.to(torch.bfloat16), None))
        del rows
    s["cache"] = (cache[0][0], cache[1][0], cache[0][1], cache[1][1])
    if case["op"] == "append":
        qkv = _randn(g, n, hq + 2 * hkv, d).to(torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv.split((hq, hkv, hkv), dim=1)
        s["frequencies"], s["magnitude"] = _frequencies(d, "none")
        depth = [c + min(t, 9) for c, k in zip(context, counts) for t in range(k)]
        s["positions"] = torch.tensor(depth, dtype=torch.int32).cuda()
        return s
    # queries that look at some places more than at others
    s["q"] = _randn(g, n, hq, d).mul_(2.0).to(torch.bfloat16)
    s["mask"] = _tree(counts, s["most"], g) if case["tree"] else None
    s["scale"] = d ** -0.5
    return s


# -- plain forms: elementary operations in 32 bits, rounded once at the end ------


def _plain_rotated(x, s):
    """x [N, H, D] in 32 bits with its first dimensions turned."""
    f = s["frequencies"]
    half = f.numel()
    angle = s["positions"].double()[:, None] * f
    cos = (torch.cos(angle) * s["magnitude"]).to(torch.float32)[:, None, :]
    sin = (torch.sin(angle) * s["magnitude"]).to(torch.float32)[:, None, :]
    x = x.to(torch.float32)
    if s["interleaved"]:
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((u * cos - v * sin, u * sin + v * cos), dim=-1).flatten(-2)
    else:
        u, v = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((u * cos - v * sin, u * sin + v * cos), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _sequences(s, n):
    """(sequence, number within it) of each of n tokens."""
    token = torch.arange(n, device="cuda")
    b = (token[:, None] >= s["starts"][None, 1:]).sum(dim=1)
    return b, token - s["starts"][b]


def _plain_write(rows, cache, scales, at, row):
    if scales is None:
        cache[at, :, row] = rows.to(torch.bfloat16)
    else:
        scale = rows.abs().amax(dim=-1).clamp(min=AMAX_MIN) / FP8_MAX
        cache[at, :, row] = (rows / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        scales[at, :, row] = scale


def _plain_append(s):
    k, v, k_scale, v_scale = s["cache"]
    page = k.shape[2]
    b, t = _sequences(s, s["q"].shape[0])
    slot = s["lens"][b] + t
    at, row = s["pages"][b, slot // page].long(), slot % page
    _plain_write(_plain_rotated(s["k"], s), k, k_scale, at, row)
    _plain_write(s["v"].to(torch.float32), v, v_scale, at, row)
    return _plain_rotated(s["q"], s).to(torch.bfloat16)


def _plain_rows(cache, scales, pages):
    """The sequences' rows [B, Hkv, slots, D] in 32 bits."""
    x = cache[pages]                                   # [B, P, Hkv, page, D]
    if scales is None:
        x = x.to(torch.float32)
    else:
        x = x.view(torch.float8_e4m3fn).to(torch.float32) * scales[pages][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    k, v, k_scale, v_scale = s["cache"]
    n, hq, d = s["q"].shape
    hkv, pages = k.shape[1], s["pages"].long()
    count, most = s["starts"].numel() - 1, s["most"]
    # padded to one length: [B, Hkv, most * G, D]
    t = torch.arange(most, device="cuda")
    at = torch.clamp(s["starts"][:-1, None] + t, max=n - 1)
    q = s["q"].to(torch.float32)[at].view(count, most, hkv, hq // hkv, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(count, hkv, -1, d)
    score = torch.matmul(q, _plain_rows(k, k_scale, pages).transpose(2, 3))
    score = score.mul_(s["scale"]).view(count, hkv, most, hq // hkv, -1)
    slots = score.shape[-1]
    new = torch.arange(slots, device="cuda")[None, :] - s["lens"][:, None]   # [B, slots]
    if s["mask"] is None:
        seen = new[:, None, :] <= t[None, :, None]
    else:
        tree = s["mask"][at]                                                 # [B, most, most]
        inside = torch.clamp(new, 0, most - 1)[:, None, :].expand(count, most, slots)
        seen = (new < 0)[:, None, :] | ((new < most)[:, None, :] & torch.gather(tree, 2, inside))
    seen = seen[:, None, :, None, :]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(count, hkv, -1, slots), _plain_rows(v, v_scale, pages))
    o = o.view(count, hkv, most, -1, d) / torch.where(total == 0.0, 1.0, total)
    b, t = _sequences(s, n)
    return o.permute(0, 2, 1, 3, 4).reshape(count, most, hq, d)[b, t].to(torch.bfloat16)


def _framework():
    path = os.path.join(_ROOT, "tans-vectoradd_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rans_vectoradd
    return rans_vectoradd


def run(state):
    s = state
    if s["op"] == "rotary":
        if own:
            return _framework().rotary(s["x"], s["positions"], s["frequencies"],
                                       interleaved=s["interleaved"], magnitude=s["magnitude"])
        return _plain_rotated(s["x"], s).to(torch.bfloat16)
    if s["op"] == "append":
        if own:
            R = _framework()
            q = R.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["frequencies"],
                                R.KvCache(*s["cache"]), s["pages"], s["starts"], s["lens"],
                                interleaved=s["interleaved"], magnitude=s["magnitude"])
        else:
            q = _plain_append(s)
        k, v, k_scale, v_scale = s["cache"]
        if k_scale is None:
            return [q, k, v]
        return [q, k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), k_scale, v_scale]
    if own:
        R = _framework()
        return R.tree_attention(s["q"], R.KvCache(*s["cache"]), s["pages"], s["starts"], s["lens"],
                                s["mask"], scale=s["scale"], max_tokens=s["most"])
    return _plain_attention(s)


# ---------------------------------------------------------------------------


def work(case):
    """Bytes: inputs once, outputs once (of the cache the rows that are read or
    written, of the mask its bytes).  Operations: the two products over the slots
    that a token may see; for the rotation six a pair."""
    d = case["D"]
    if case["op"] == "rotary":
        n, h, rot = case["N"], case["H"], case["rot"]
        return {"bytes": 4 * n * h * d + 4 * n + 4 * rot, "flops": 3 * n * h * rot}
    counts, context = _lens(case)
    n, b = sum(counts), case["B"]
    hq, hkv = case["Hq"], case["Hkv"]
    row = d + 4 if case["fp8"] else 2 * d
    used = sum(-(-(c + t) // case["page"]) for c, t in zip(context, counts))
    if case["op"] == "append":
        return {"bytes": 4 * n * hq * d + 2 * n * hkv * (2 * d + row) + 8 * n + 4 * d + 8 * b,
                "flops": 3 * n * (hq + hkv) * d}
    rows = sum(c + t for c, t in zip(context, counts))
    tree = case["tree"]
    pairs = sum(t * c + (t * t if tree else t * (t + 1) // 2) for c, t in zip(context, counts))
    return {"bytes": 4 * n * hq * d + 2 * rows * hkv * row + 4 * used + 8 * b
                     + (n * max(counts) if tree else 0),
            "flops": 4 * pairs * hq * d}


def _f64(b):
    """The values of E4M3FN bytes from the format's definition: sign, 4 exponent
    bits (bias 7), 3 mantissa bits; exponent 0 is subnormal."""
    i = torch.arange(256, dtype=torch.float64, device="cuda")
    sign = torch.where(i >= 128, -1.0, 1.0).double()
    e = torch.floor(i / 8) % 16
    f = i % 8
    mag = torch.where(e > 0, (1 + f / 8) * torch.pow(2.0, e - 7), f / 8 * 2.0 ** -6)
    return (sign * mag)[b.to(torch.int32)]


def _exact_turned(x, s):
    """Pairs as complex numbers, each times the unit number of its angle."""
    f = s["frequencies"]
    m = f.numel()
    y = x.double().clone()
    turn = torch.polar(torch.full_like(f, s["magnitude"]).expand(len(y), m),
                       torch.outer(s["positions"].double(), f)).unsqueeze(1)
    if s["interleaved"]:
        at = (slice(0, 2 * m, 2), slice(1, 2 * m, 2))
    else:
        at = (slice(0, m), slice(m, 2 * m))
    z = torch.complex(y[:, :, at[0]].contiguous(), y[:, :, at[1]].contiguous()) * turn
    y[:, :, at[0]], y[:, :, at[1]] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rotary":
        return _exact_turned(s["x"], s)
    k, v, k_scale, v_scale = s["cache"]
    hkv, page, d = k.shape[1:]
    counts, context = _lens(case)
    if s["op"] == "append":
        slots = torch.tensor([c + i for c, n in zip(context, counts) for i in range(n)]).cuda()
        of = torch.repeat_interleave(torch.arange(case["B"]), torch.tensor(counts)).cuda()
        row = (s["pages"][of, torch.div(slots, page, rounding_mode="floor")].long() * hkv * page
               + slots % page)
        row = row[:, None] + page * torch.arange(hkv, device="cuda")     # [N, Hkv]
        out = [_exact_turned(s["q"], s)]
        scales = []
        for new, cache, scale in ((_exact_turned(s["k"], s), k, k_scale), (s["v"].double(), v, v_scale)):
            if scale is not None:
                by = torch.clamp(new.abs().max(dim=2).values, min=AMAX_MIN) / FP8_MAX
                new = new / by.unsqueeze(2)
                whole = scale.double().flatten()
                whole[row.flatten()] = by.flatten()
                scales.append(whole.view_as(scale))
            rows = (cache.double() if scale is None else _f64(cache)).view(-1, d)
            rows[row.flatten()] = new.flatten(0, 1)
            out.append(rows.view(cache.shape))
        return out + scales
    group = s["q"].shape[1] // hkv
    result = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, c) in enumerate(zip(counts, context)):
        slot = torch.arange(c + n, device="cuda")
        where = s["pages"][b, torch.div(slot, page, rounding_mode="floor")].long()
        sees = torch.ones(n, c + n, dtype=torch.bool, device="cuda")
        sees[:, c:] = (torch.ones(n, n, device="cuda").tril() > 0 if s["mask"] is None
                       else s["mask"][first:first + n, :n])
        for h in range(hkv):
            keys, values = k[where, h, slot % page], v[where, h, slot % page]
            if k_scale is None:
                keys, values = keys.double(), values.double()
            else:
                keys = _f64(keys) * k_scale[where, h, slot % page].double().unsqueeze(1)
                values = _f64(values) * v_scale[where, h, slot % page].double().unsqueeze(1)
            q = s["q"][first:first + n, h * group:(h + 1) * group].double().transpose(0, 1)
            e = (q.reshape(-1, d) @ keys.t().contiguous()).view(group, n, -1) * s["scale"]
            e = e.masked_fill(~sees, -math.inf)
            e = torch.exp(e - torch.logsumexp(e, dim=2, keepdim=True))
            o = (e.view(group * n, -1) @ values).view(group, n, d)
            result[first:first + n, h * group:(h + 1) * group] = o.transpose(0, 1)
        first += n
    return result
