"""The layer operators (fp8_rmsnorm, fp8_quantize_rows, fp8_linear; no
counterpart in the reference) against plain 64-bit forms written from their
definitions.

Tolerances, from the arithmetic:

* q: nearest E4M3FN of t = y / scale: half a step, 2^-4 |t| (3 mantissa bits;
  2^-10 below the smallest normal), and t's own 32-bit rounding, 2^-18 of it.
* scale: a few 32-bit roundings and the sum of squares' (pairwise over at most
  2^8 terms in a row): 2^-16 relative.
* products: bf16 (8 significant bits) rounds to 2^-8 of |y|.  The FP8 matrix
  instructions add products in groups of 8 columns, each cut off at 2^-13 of
  the largest of its group (shown by a pair of +-2^16 that cancels beside a
  small product: 2^3 is kept and 2^2 is not, while one of another group is
  kept to 32 bits): with S = sum |a w| a_scale w_scale, at most 8 2^-13 S in
  all, and one 32-bit rounding per 32 columns at most and a few in the
  epilogue, (C / 32 + 16) 2^-23 S.  The cut-off parts have random signs, about
  2^-13 S / sqrt(C / 8) together, which bounds the 2-norm of the whole output
  (with a factor 2).  The activations' slopes are below 1.13.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

AMAX_MIN = 2.0 ** -100


def _say(msg):
    print(msg, flush=True)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bf16(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _e4m3(b):
    return b.view(torch.float8_e4m3fn).to(torch.float32).double()


def _fp8(g, *shape):
    """E4M3FN bytes over the format's range, both signs, zeros and subnormals,
    no NaN."""
    x = torch.randn(*shape, generator=g, device="cuda") * 40.0
    x = torch.where(torch.rand(*shape, generator=g, device="cuda") < 0.05, x * 2.0 ** -10, x)
    return x.clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _check_q(q, scale, y):
    """q, scale against y (float64 rows)."""
    want = y.abs().amax(dim=-1).clamp(min=AMAX_MIN) / 448.0
    assert ((scale.double() - want).abs() <= want * 2.0 ** -16).all()
    t = y / scale.double().unsqueeze(-1)
    off = (_e4m3(q) - t).abs()
    lim = torch.clamp(t.abs() * 2.0 ** -4, min=2.0 ** -10) * (1 + 2.0 ** -14) + 2.0 ** -18 * t.abs()
    assert (off <= lim).all(), f"{(off > lim).sum().item()} bytes are not the nearest"


def _norm64(x, weight, residual, eps):
    h = x.double() + (residual.double() if residual is not None else 0.0)
    return h * weight.double() / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + eps)


# row widths: one 16-byte load, less and more than a wave's, a workgroup's and
# several of either, and no power of two; row counts around the same borders
NORM_SHAPES = [(1, 16), (3, 48), (5, 512), (64, 528), (2, 1024), (7, 1040), (257, 2048), (1, 5120),
               (33, 5120), (3, 8192), (2, 8208), (9, 17408), (2, 32784), (1, 65552), (1, 131088),
               (4099, 64), (1030, 1296)]


@pytest.mark.parametrize("M,D", NORM_SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_rmsnorm_matches_64_bits(M, D, with_residual):
    import rans_vectoradd as R
    _say(f"case: rmsnorm {M}x{D} residual={with_residual}")
    g = _gen(M * 131 + D)
    x = _bf16(g, M, D, std=3.0)
    res = _bf16(g, M, D) if with_residual else None
    w = _bf16(g, D)
    q, scale, h = R.fp8_rmsnorm(x, w, res, eps=1e-5)
    assert q.shape == (M, D) and q.dtype == torch.uint8 and scale.shape == (M,)
    if with_residual:
        assert torch.equal(h, (x.float() + res.float()).to(torch.bfloat16))
    else:
        assert h is x
    _check_q(q, scale, _norm64(x, w, res, 1e-5))


@pytest.mark.parametrize("M,D", NORM_SHAPES)
def test_quantize_rows_matches_64_bits(M, D):
    import rans_vectoradd as R
    _say(f"case: quantize_rows {M}x{D}")
    g = _gen(M * 137 + D)
    x = _bf16(g, M, D, std=0.3)
    q, scale = R.fp8_quantize_rows(x)
    _check_q(q, scale, x.double())
    # the scale is one division away: correctly rounded (through 64 bits, which
    # rounds a quotient of 32-bit values to the same 32 bits)
    assert torch.equal(scale, (x.double().abs().amax(dim=1) / 448.0).float())


# rows of 4, 6 and 7 loads a thread, and the longest that a workgroup holds
@pytest.mark.parametrize("D", [12304, 16384, 40976, 49152, 49168, 57344, 57360])
@pytest.mark.parametrize("op", ["norm", "norm_residual", "quantize"])
def test_long_rows_match_64_bits(D, op):
    import rans_vectoradd as R
    _say(f"case: {op} 3x{D}")
    g = _gen(D)
    x = _bf16(g, 3, D, std=2.0)
    if op == "quantize":
        q, scale = R.fp8_quantize_rows(x)
        _check_q(q, scale, x.double())
        return
    res = _bf16(g, 3, D) if op == "norm_residual" else None
    w = _bf16(g, D)
    q, scale, h = R.fp8_rmsnorm(x, w, res, eps=1e-5)
    if res is not None:
        assert torch.equal(h, (x.float() + res.float()).to(torch.bfloat16))
    _check_q(q, scale, _norm64(x, w, res, 1e-5))


def test_more_rows_than_one_launch_has_threads_for():
    import rans_vectoradd as R
    n, times = 1024, (1 << 16) + 1          # 2^26 + 1024 rows of one wave each
    _say(f"case: quantize_rows and rmsnorm of {n * times} rows")
    g = _gen(5)
    x, res, w = _bf16(g, n, 16), _bf16(g, n, 16), _bf16(g, 16)
    many = x.repeat(times, 1)
    q0, s0 = R.fp8_quantize_rows(x)
    q, s = R.fp8_quantize_rows(many)
    assert torch.equal(q.view(times, n, 16), q0.expand(times, n, 16))
    assert torch.equal(s.view(times, n), s0.expand(times, n))
    q0, s0, h0 = R.fp8_rmsnorm(x, w, res)
    q, s, h = R.fp8_rmsnorm(many, w, res.repeat(times, 1))
    assert torch.equal(q.view(times, n, 16), q0.expand(times, n, 16))
    assert torch.equal(s.view(times, n), s0.expand(times, n))
    assert torch.equal(h.view(torch.int16).view(times, n, 16), h0.view(torch.int16).expand(times, n, 16))


def test_rows_of_zeros_and_tiny_and_huge_values():
    import rans_vectoradd as R
    D = 272
    x = torch.zeros(6, D, device="cuda")
    x[1, 5] = 2.0 ** -110            # below the smallest maximum
    x[2] = 2.0 ** -90
    x[3, 7] = 3.0e38
    x[4] = -1.0e30
    x[5, ::2] = -0.0
    x = x.to(torch.bfloat16)
    q, scale = R.fp8_quantize_rows(x)
    assert torch.isfinite(scale).all() and (scale > 0).all()
    _check_q(q, scale, x.double())
    assert (_e4m3(q[0]) == 0).all() and (_e4m3(q[5]) == 0).all()
    w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    rows = x[[0, 1, 2, 5]].contiguous()
    q, scale, _ = R.fp8_rmsnorm(rows, w, eps=1e-6)
    _check_q(q, scale, _norm64(rows, w, None, 1e-6))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [64, 5120])
def test_rows_with_nan_or_infinity_spoil_only_themselves(bad, D):
    import rans_vectoradd as R
    g = _gen(7)
    M = 9
    x = _bf16(g, M, D)
    w = _bf16(g, D)
    clean = R.fp8_rmsnorm(x, w, x)
    cleanq = R.fp8_quantize_rows(x)
    y = x.clone()
    y[4, D - 3] = bad
    got = R.fp8_rmsnorm(y, w, x)
    gotq = R.fp8_quantize_rows(y)
    keep = [i for i in range(M) if i != 4]
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
    for a, b in zip(gotq, cleanq):
        assert torch.equal(a[keep], b[keep])
    assert not torch.isfinite(got[1][4]) and not torch.isfinite(gotq[1][4])
    assert torch.isnan(_e4m3(got[0][4, D - 3])) and torch.isnan(_e4m3(gotq[0][4, D - 3]))


# ---------------------------------------------------------------------------


def _act64(v, act):
    if act == "relu":
        return v.clamp(min=0.0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v * math.sqrt(0.5))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def _linear64(a, sa, w, sw, bias, act, residual, gated):
    """(y, most that the kernel's y may be off before the last rounding, S as
    it reaches y)."""
    A, W = _e4m3(a), _e4m3(w)
    if sa is not None:
        A = A * sa.double().unsqueeze(1)
    W = W * (sw.double().unsqueeze(1) if isinstance(sw, torch.Tensor) else sw)
    Wt = W.t().contiguous()
    v = A @ Wt
    S = A.abs() @ Wt.abs()
    dv = S * (2.0 ** -10 + (a.shape[1] / 32 + 16) * 2.0 ** -23)
    if bias is not None:
        v = v + bias.double()
        dv = dv + v.abs() * 2.0 ** -23
    if gated:
        F = v.shape[1] // 2
        g, u, dg, du = v[:, :F], v[:, F:], dv[:, :F], dv[:, F:]
        ag = _act64(g, act)
        y = ag * u
        dy = 1.13 * dg * u.abs() + ag.abs() * du + 1.13 * dg * du + (y.abs() + (g * u).abs()) * 2.0 ** -20
        S = 1.13 * S[:, :F] * u.abs() + ag.abs() * S[:, F:]
    else:
        y = _act64(v, act)
        dy = 1.13 * dv + (y.abs() + v.abs()) * 2.0 ** -20
        S = 1.13 * S
    if residual is not None:
        y = y + residual.double()
        dy = dy + y.abs() * 2.0 ** -23
    return y, dy, S


def _run_linear(M, R_, C, act="none", gated=False, bias=False, residual=False, sa=True, sw=True,
                seed=0):
    import rans_vectoradd as R
    g = _gen(seed + 1000003 * M + 1009 * R_ + C)
    a, w = _fp8(g, M, C), _fp8(g, R_, C)
    N = R_ // 2 if gated else R_
    a_scale = torch.rand(M, generator=g, device="cuda") * 0.01 + 1e-4 if sa else None
    w_scale = torch.rand(R_, generator=g, device="cuda") * 0.02 + 1e-4 if sw else 0.0125
    b = _bf16(g, R_) if bias else None
    res = _bf16(g, M, N) if residual else None
    y = R.fp8_linear(a, a_scale, w, w_scale, bias=b, activation=act, residual=res, gated=gated)
    assert y.shape == (M, N) and y.dtype == torch.bfloat16
    want, off, S = _linear64(a, a_scale, w, w_scale, b, act, res, gated)
    err = (y.double() - want).abs()
    lim = off + (want.abs() + off) * 2.0 ** -8 + 2.0 ** -130
    bad = ~(err <= lim)
    assert not bad.any(), (f"{bad.sum().item()} of {bad.numel()} outputs, first at "
                           f"{bad.nonzero()[0].tolist()}")
    most = 2.0 ** -8 * want.norm() + 2.0 ** -12 / math.sqrt(C / 8) * S.norm()
    assert err.norm() <= most, f"2-norm of the error {err.norm():.3g}, at most {most:.3g}"
    again = R.fp8_linear(a, a_scale, w, w_scale, bias=b, activation=act, residual=res, gated=gated)
    assert torch.equal(y, again)


# rows of a around 1, the matrix instruction's 16 and the tiles' borders;
# outputs and columns that fill no tile
@pytest.mark.parametrize("M", [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 128, 129,
                               192, 255, 256, 257, 300, 513])
@pytest.mark.parametrize("R_,C", [(272, 144), (257, 400), (64, 16), (1030, 1296)])
def test_linear_sizes(M, R_, C):
    _say(f"case: linear {M}x{R_}x{C}")
    _run_linear(M, R_, C, bias=M % 2 == 0, residual=M % 3 == 0)


@pytest.mark.parametrize("C", [16, 32, 48, 112, 128, 144, 240, 256, 272, 384, 400, 1008, 2064])
@pytest.mark.parametrize("M", [1, 20, 70, 260])
def test_linear_columns(M, C):
    _say(f"case: linear columns {M}x{C}")
    _run_linear(M, 530, C)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [1, 5, 40, 150, 600])
def test_linear_epilogues(M, act, gated):
    _say(f"case: linear epilogue {M} {act} gated={gated}")
    for bias in (False, True):
        for residual in (False, True):
            _run_linear(M, 534, 656, act, gated, bias, residual)
    _run_linear(M, 512, 640, act, gated, True, True, sa=False)
    _run_linear(M, 512, 640, act, gated, True, True, sw=False)


# gates and values whose number fills no tile, so that both halves' tiles end
# inside
@pytest.mark.parametrize("R_", [2, 6, 30, 126, 130, 254, 258, 514, 1030, 2186])
@pytest.mark.parametrize("M", [1, 24, 130, 270])
def test_linear_gated_widths(M, R_):
    _say(f"case: linear gated {M}x{R_}")
    _run_linear(M, R_, 272, "silu", True, True, True)


@pytest.mark.parametrize("M,R_,C", [(1, 17408, 5120), (8, 5120, 17408), (16, 5120, 5120),
                                    (97, 17408, 5120), (250, 5120, 17408), (1000, 5120, 5120),
                                    (2048, 5120, 2560), (4100, 2560, 1280)])
def test_linear_layer_sizes(M, R_, C):
    _say(f"case: linear {M}x{R_}x{C}")
    _run_linear(M, R_, C, "silu", gated=M % 2 == 1, residual=True)


def test_linear_one_row_equals_the_same_row_of_a_vector():
    import rans_vectoradd as R
    g = _gen(5)
    a, w = _fp8(g, 1, 512), _fp8(g, 96, 512)
    s = torch.full((1,), 0.01, device="cuda")
    y2 = R.fp8_linear(a, s, w, 0.5)
    y1 = R.fp8_linear(a[0], s[0], w, 0.5)
    assert y1.shape == (96,) and torch.equal(y1, y2[0])
    x = _bf16(g, 512)
    q, sc = R.fp8_quantize_rows(x)
    assert q.shape == (512,) and sc.shape == ()
    y = R.fp8_linear(q, sc, w, 0.5)
    assert y.shape == (96,)


@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_nan_and_infinite_inputs_stay_in_their_rows_and_columns(M):
    import rans_vectoradd as R
    g = _gen(11)
    a, w = _fp8(g, M, 272), _fp8(g, 300, 272)
    s = torch.full((M,), 0.01, device="cuda")
    clean = R.fp8_linear(a, s, w, 0.1)
    a2, w2, s2 = a.clone(), w.clone(), s.clone()
    w2[37, 271] = 0x7F                      # NaN weight: column 37
    if M > 1:
        a2[M - 2, 0] = 0xFF                 # NaN activation: row M - 2
        s2[M - 1] = float("inf")
    y = R.fp8_linear(a2, s2, w2, 0.1)
    assert torch.isnan(y[:, 37]).all()
    cols = [i for i in range(300) if i != 37]
    rows = list(range(M)) if M == 1 else list(range(M - 2))
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    if M > 1:
        assert torch.isnan(y[M - 2]).all()
        assert not torch.isfinite(y[M - 1]).any()
    # activations of infinite values
    bias = torch.zeros(300, dtype=torch.bfloat16, device="cuda")
    bias[0], bias[1], bias[2] = float("inf"), float("-inf"), float("nan")
    for act, minus in (("relu", 0.0), ("silu", None), ("gelu", None)):
        z = R.fp8_linear(a, s, w, 0.1, bias=bias, activation=act)
        assert torch.isinf(z[:, 0]).all() and torch.isnan(z[:, 2]).all()
        if minus is not None:
            assert (z[:, 1] == minus).all()


@pytest.mark.parametrize("M", [0, 1])
def test_no_rows_and_one_row(M):
    import rans_vectoradd as R
    x = torch.ones(M, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, s, h = R.fp8_rmsnorm(x, w, x)
    assert q.shape == (M, 64) and s.shape == (M,) and h.shape == (M, 64)
    q, s = R.fp8_quantize_rows(x)
    assert q.shape == (M, 64) and s.shape == (M,)
    wq = torch.full((32, 64), 0x38, dtype=torch.uint8, device="cuda")
    y = R.fp8_linear(q, s, wq)
    assert y.shape == (M, 32)
    assert M == 0 or (y == 64.0).all()


def test_runs_on_the_current_stream():
    """Work queued behind a slow kernel on another stream sees its result."""
    import rans_vectoradd as R
    g = _gen(3)
    w = _bf16(g, 5120)
    wq = _fp8(g, 512, 5120)
    x0 = _bf16(g, 40, 5120)
    want = R.fp8_linear(*R.fp8_rmsnorm(x0, w)[:2], wq, 0.01)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-3
        x = x0.clone()
        got = R.fp8_linear(*R.fp8_rmsnorm(x, w)[:2], wq, 0.01)
    s.synchronize()
    assert torch.equal(got, want)


def test_graph_replays():
    """The three operators captured once, replayed with new inputs in place."""
    import rans_vectoradd as R
    g = _gen(4)
    w, res = _bf16(g, 2560), _bf16(g, 20, 2560)
    up, down = _fp8(g, 2080, 2560), _fp8(g, 2560, 1040)

    def block(x):
        q, s, h = R.fp8_rmsnorm(x, w, res)
        t = R.fp8_linear(q, s, up, 1e-4, activation="silu", gated=True)
        q, s = R.fp8_quantize_rows(t)
        return R.fp8_linear(q, s, down, 1e-4, residual=h)

    x = _bf16(g, 20, 2560)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        block(x)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x)
    for k in range(4):
        x.copy_(_bf16(g, 20, 2560))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, block(x)), f"replay {k}"


def test_output_may_be_written_over_its_residual():
    """The C entry points allow h = residual and y = residual."""
    import rans_vectoradd as R
    from rans_vectoradd._lib import lib
    g = _gen(9)
    x, res, w = _bf16(g, 12, 1296), _bf16(g, 12, 1296), _bf16(g, 1296)
    q, s, h = R.fp8_rmsnorm(x, w, res)
    buf, q2, s2 = res.clone(), torch.empty_like(q), torch.empty_like(s)
    st = torch.cuda.current_stream().cuda_stream
    assert lib.tans_fp8_rmsnorm(x.data_ptr(), buf.data_ptr(), w.data_ptr(), 12, 1296, 1e-6,
                                q2.data_ptr(), s2.data_ptr(), buf.data_ptr(), st) == 0
    torch.cuda.synchronize()
    assert torch.equal(buf, h) and torch.equal(q2, q) and torch.equal(s2, s)


def test_refusals_on_the_gpu():
    import rans_vectoradd as R
    g = _gen(1)
    x, w = _bf16(g, 4, 64), _bf16(g, 64)
    a, wq = _fp8(g, 4, 64), _fp8(g, 32, 64)
    s = torch.ones(4, device="cuda")

    def refuses(match, f, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)

    refuses("bfloat16", R.fp8_rmsnorm, x.float(), w)
    refuses("contiguous", R.fp8_rmsnorm, x.t().contiguous().t(), w)
    refuses("multiple of 16", R.fp8_rmsnorm, x[:, :40].contiguous(), w[:40])
    refuses("weight must be", R.fp8_rmsnorm, x, w[:48].contiguous())
    refuses("shape of x", R.fp8_rmsnorm, x, w, x[:2].contiguous())
    refuses("eps", R.fp8_rmsnorm, x, w, eps=-1.0)
    refuses("gradient", R.fp8_rmsnorm, x.clone().requires_grad_(), w)
    refuses("misaligned", R.fp8_quantize_rows, x.view(-1)[1:65].view(1, 64))
    refuses(r"\[D\] or \[M, D\]", R.fp8_quantize_rows, x.view(2, 2, 64))
    refuses("uint8", R.fp8_linear, x, s, wq)
    refuses("w must be", R.fp8_linear, a, s, wq[:, :48].contiguous())
    refuses("one scale per row", R.fp8_linear, a, s[:3].contiguous(), wq)
    refuses("w_scale", R.fp8_linear, a, s, wq, s)
    refuses("bias", R.fp8_linear, a, s, wq, bias=w)
    refuses("residual", R.fp8_linear, a, s, wq, residual=x)
    refuses("activation", R.fp8_linear, a, s, wq, activation="tanh")
    refuses("even number", R.fp8_linear, a, s, wq[:31].contiguous(), gated=True)
