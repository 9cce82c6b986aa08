"""What the attention operators refuse, without a GPU: sizes, strides, alignment and
null pointers at the C entries, and what is no CUDA tensor at the wrappers."""
import ctypes

import pytest
import torch

D16 = ctypes.c_void_p(4096)   # never looked at: every call below ends before a launch
P, F = ctypes.c_void_p, ctypes.c_float


def _lib():
    from rans_vectoradd._lib import lib
    return lib


def _says(text):
    lib = _lib()
    return text in lib.tans_last_error()


def rotary(x=D16, stride=256, pos=D16, f=D16, N=4, H=2, D=128, rot=128, out=D16, out_stride=256):
    return _lib().tans_rotary(x, stride, pos, f, N, H, D, rot, 0, 0, F(1.0), out, out_stride, None)


def append(q=D16, sq=1024, k=D16, sk=256, v=D16, sv=256, pos=D16, f=D16, rot=128, kc=D16, vc=D16, ks=None, vs=None,
           pages=4, heads=2, page=16, dim=128, table=D16, per=4, starts=D16, lens=D16, B=2, N=5, Hq=8, out=D16):
    return _lib().tans_rotary_append(q, sq, k, sk, v, sv, pos, f, rot, 0, F(1.0), kc, vc, ks, vs, pages, heads, page,
                                     dim, table, per, starts, lens, B, N, Hq, out, None)


def attend(q=D16, sq=1024, kc=D16, vc=D16, ks=None, vs=None, pages=4, heads=2, page=16, dim=128, table=D16, per=4,
           starts=D16, lens=D16, B=2, mask=None, cols=0, N=5, Hq=8, scale=1.0, most=5, ws=D16, ws_bytes=1 << 40,
           out=D16):
    return _lib().tans_tree_attention(q, sq, kc, vc, ks, vs, pages, heads, page, dim, table, per, starts, lens, B, mask,
                                      cols, N, Hq, F(scale), most, ws, ws_bytes, out, None)


def test_rotary_refuses():
    for kw in ({"x": None}, {"out": None}, {"pos": None}, {"f": None}):
        assert rotary(**kw) == -1 and _says(b"null"), kw
    for kw in ({"N": -1}, {"N": 1 << 30}):
        assert rotary(**kw) == -1 and _says(b"N must"), kw
    for kw in ({"H": 0}, {"H": 65536}):
        assert rotary(**kw) == -1 and _says(b"H must"), kw
    for D in (0, 8, 24, 1040, -16):
        assert rotary(D=D) == -1 and _says(b"D must"), D
    for rot in (0, 8, 144, -16, 24):
        assert rotary(rot=rot) == -1 and _says(b"rotated part"), rot
    for kw in ({"stride": 248}, {"stride": 260}, {"out_stride": 128}, {"stride": -256}):
        assert rotary(**kw) == -1 and _says(b"stride"), kw
    for kw in ({"x": P(4104)}, {"out": P(4104)}, {"pos": P(4098)}, {"f": P(4100)}):
        assert rotary(**kw) == -1 and _says(b"misaligned"), kw
    assert rotary(N=0, x=None, out=None) == 0


@pytest.mark.parametrize("call", [append, attend])
def test_batches_refused(call):
    for kw in ({"kc": None}, {"vc": None}, {"starts": None}, {"lens": None}, {"table": None}, {"q": None}, {"out": None}):
        assert call(**kw) == -1 and _says(b"null"), kw
    for dim in (0, 32, 96, 512):
        assert call(dim=dim) == -1 and _says(b"64, 128 or 256"), dim
    for kw in ({"heads": 0}, {"heads": 3}, {"Hq": 1}, {"Hq": 65536, "heads": 1}, {"Hq": 7}):
        assert call(**kw) == -1 and _says(b"query heads"), kw
    for kw in ({"pages": 0}, {"page": 0}, {"page": (1 << 20) + 1}, {"pages": 1 << 27}, {"pages": 1 << 31}):
        assert call(**kw) == -1 and _says(b"pages"), kw
    for kw in ({"B": -1}, {"per": -1}, {"per": 1 << 27}, {"B": (1 << 31) - 1}):
        assert call(**kw) == -1 and _says(b"need B"), kw
    for N in (-1, 1 << 30):
        assert call(N=N) == -1 and _says(b"N must"), N
    for kw in ({"ks": D16}, {"vs": D16}):
        assert call(**kw) == -1 and _says(b"scales"), kw
    for kw in ({"kc": P(4104)}, {"vc": P(4104)}, {"table": P(4098)}, {"starts": P(4098)}, {"lens": P(4097)},
               {"ks": P(4098), "vs": D16}, {"q": P(4104)}, {"out": P(4104)}):
        assert call(**kw) == -1 and _says(b"misaligned"), kw
    for kw in ({"sq": 1020}, {"sq": 1016}, {"sq": 0}):
        assert call(**kw) == -1 and _says(b"stride of q"), kw
    assert call(N=0, q=None, out=None, kc=None) == 0
    assert call(B=0, q=None, out=None, kc=None) == 0


def test_append_refuses():
    for kw in ({"k": None}, {"v": None}, {"pos": None}, {"f": None}):
        assert append(**kw) == -1 and _says(b"null"), kw
    for kw in ({"sk": 248}, {"sk": 257}):
        assert append(**kw) == -1 and _says(b"stride of k"), kw
    assert append(sv=8) == -1 and _says(b"stride of v")
    for rot in (0, 120, 144):
        assert append(rot=rot) == -1 and _says(b"rotated part"), rot


def test_attention_refuses():
    for scale in (0.0, -1.0, float("inf"), float("nan"), 2e38):
        assert attend(scale=scale) == -1 and _says(b"scale"), scale
    assert attend(most=-1) == -1 and _says(b"max_tokens")
    for cols in (-1, 0, 1 << 31):
        assert attend(mask=D16, cols=cols) == -1 and _says(b"columns"), cols
    assert attend(N=1 << 28) == -1 and _says(b"2^31")
    n = ctypes.c_int64(-1)

    def need(N=5, B=2, Hq=8, heads=2, dim=128, slots=4096, most=5, to=ctypes.byref(n)):
        return _lib().tans_tree_attention_workspace(N, B, Hq, heads, dim, slots, most, to)
    assert need(to=None) == -1 and _says(b"null")
    for kw in ({"N": -1}, {"B": -1}, {"Hq": 7}, {"heads": 0}, {"dim": 96}, {"slots": -1}, {"most": -1},
               {"N": 1 << 28}, {"slots": 1 << 31}):
        assert need(**kw) == -1 and _says(b"out of range"), kw
    assert need(N=0) == 0 and n.value == 0
    assert need(B=0) == 0 and n.value == 0
    assert need() == 0 and n.value > 0


def test_wrappers_refuse_what_they_cannot_take():
    import rans_vectoradd as R
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    f, _ = R.rotary_frequencies(64, device="cpu")
    cache = R.KvCache.empty(2, 2, 16, 64, device="cpu")
    t = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda q: R.rotary(q, i, f),
                 lambda q: R.rotary_append(q, x, x, i, f, cache, t, i, i[:1]),
                 lambda q: R.tree_attention(q, cache, t, i, i[:1])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(x)
        for bad in (None, 3, [1.0]):
            with pytest.raises(RuntimeError, match="must be a tensor"):
                call(bad)


def test_frequencies():
    """The scalings at their ends: the fastest pairs keep their frequency, the slowest are
    stretched by the factor."""
    import rans_vectoradd as R
    f, m = R.rotary_frequencies(128, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64)
    assert f.dtype is torch.float64 and m == 1.0 and torch.allclose(f, want, rtol=1e-14, atol=0)
    g, m = R.rotary_frequencies(128, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(g * 4.0, want, rtol=1e-14, atol=0) and m == 1.0
    g, m = R.rotary_frequencies(128, scaling="ntk", factor=4.0, device="cpu")
    assert g[0] == 1.0 and abs(g[-1] * 4.0 / want[-1] - 1) < 1e-12 and m == 1.0
    g, m = R.rotary_frequencies(128, scaling="yarn", factor=4.0, device="cpu")
    turns = want * 4096 / (2 * torch.pi)
    # (the blend begins and ends at whole pairs: one beyond the turns on either side)
    assert torch.equal(g[:-1][turns[1:] >= 32.0], f[:-1][turns[1:] >= 32.0])
    slow = torch.nonzero(turns <= 1.0).flatten()[1:]
    assert torch.allclose(g[slow] * 4.0, want[slow], rtol=1e-14, atol=0)
    assert (g <= f).all() and (g * 4.0 >= f * (1 - 1e-14)).all() and abs(m - 1.138629436) < 1e-8
    for kw in ({"dim": 24}, {"dim": 0}, {"dim": 64, "scaling": "other"}, {"dim": 64, "base": 1.0},
               {"dim": 64, "factor": 0.5}, {"dim": 64, "scaling": "yarn", "fast": 1.0},
               {"dim": 64, "scaling": "yarn", "original_length": 0}):
        with pytest.raises(RuntimeError):
            R.rotary_frequencies(device="cpu", **kw)
