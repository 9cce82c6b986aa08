"""How the FP8 product chooses its kernel (csrc/linear_plan.h, plain C++, run
here from a small library built with g++): the tiles cover the outputs, the
workspace is what the splits' sums take, no split is empty, every variant is
the choice of some product, and a device of any CU count gets a plan."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
STREAM, MID, TILES = 0, 1, 2


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src = d / "plan.cpp"
    src.write_text('''#include "linear_plan.h"
extern "C" void plan(int64_t M, int64_t N, int64_t C, int gated, int cus, int64_t* o) {
    const tans_linear::Plan p = tans_linear::plan(M, N, C, gated, cus);
    const int64_t v[] = {p.kind, p.few, p.mi, p.nw, p.splits, p.tiles_m, p.tiles_n, p.Np, p.bytes};
    for (int i = 0; i < 9; i++) o[i] = v[i];
}
extern "C" int mids(int64_t* o) {
    int n = 0;
    for (const auto& t : tans_linear::kMids) { o[n++] = t.mi; o[n++] = t.nw; }
    return n / 2;
}
''')
    out = d / "libplan.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    I = ctypes.c_int64
    lib.plan.argtypes = [I, I, I, ctypes.c_int, ctypes.c_int, ctypes.POINTER(I)]

    def f(M, N, C, gated, cus=256):
        o = (I * 9)()
        lib.plan(M, N, C, int(gated), cus, o)
        return dict(zip(("kind", "few", "mi", "nw", "splits", "tiles_m", "tiles_n", "Np", "bytes"),
                        o))
    f.mids = lambda: [(a[0], a[1]) for a in [(o[2 * i], o[2 * i + 1]) for o in [(I * 64)()]
                                             for i in range(lib.mids(o))]]
    return f


def _products(n, seed):
    rng = random.Random(seed)

    def size(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))
    return [(size(1, 20000), size(1, 40000), 16 * size(1, 2000), rng.random() < 0.5)
            for _ in range(n)]


@pytest.mark.parametrize("cus", [1, 64, 256, 304])
def test_tiles_cover_and_no_split_is_empty(plan, cus):
    for M, N, C, gated in _products(800, cus):
        p = plan(M, N, C, gated, cus)
        steps, halves = -(-C // 128), 2 if gated else 1
        if p["kind"] == STREAM:
            assert M <= 32 and p["bytes"] == 0
            continue
        rows_m, rows_w = 32 * p["mi"], 32 * p["nw"]
        assert p["kind"] == MID or (rows_m, rows_w) in ((256, 256), (256, 192))
        assert not (gated and rows_w == 192 and p["kind"] == TILES)
        assert (p["tiles_m"] - 1) * rows_m < M <= p["tiles_m"] * rows_m
        assert (p["tiles_n"] - 1) * rows_w < N * halves and p["tiles_n"] * rows_w >= N * halves
        assert 1 <= p["splits"] <= max(1, steps // 3)
        if p["splits"] == 1:
            assert p["bytes"] == 0
        else:
            assert p["kind"] == MID and p["Np"] % 16 == 0 and N <= p["Np"] < N + 16
            assert p["bytes"] == p["splits"] * M * halves * p["Np"] * 4


def test_every_variant_is_some_products_choice(plan):
    seen = set()
    for M, N, C, gated in _products(6000, 5):
        p = plan(M, N, C, gated)
        seen.add(("stream", p["few"]) if p["kind"] == STREAM else
                 ("tiles", p["nw"]) if p["kind"] == TILES else ("mid", p["mi"], p["nw"]))
    mids = {("mid", *t) for t in plan.mids()}
    assert seen == mids | {("stream", 0), ("stream", 1), ("tiles", 8), ("tiles", 6)}


def test_few_rows_stream_the_weights(plan):
    for M in (1, 8, 16):
        assert plan(M, 34816, 5120, False)["kind"] == STREAM
    assert plan(24, 3403, 5232, True)["kind"] == STREAM     # w of 36 MB
    assert plan(24, 17408, 5120, True)["kind"] == MID       # of 178 MB
    assert plan(1, 4096, 4096, False)["few"] and not plan(1, 7000, 4096, False)["few"]


def test_launches_stay_below_2_31_threads(plan):
    for M, N, C, gated in ((2 ** 31 - 1, 16, 16, False), (2 ** 31 - 1, 16, 16, True),
                           (2 ** 28, 300, 2048, False), (17, 2 ** 27, 16, False), (100, 2 ** 26, 16, True)):
        p = plan(M, N, C, gated)
        if p["kind"] == MID:
            assert p["tiles_m"] * p["tiles_n"] * p["splits"] * 64 * p["nw"] < 2 ** 31
        elif p["kind"] == TILES:
            assert p["tiles_m"] * p["tiles_n"] < 2 ** 31
