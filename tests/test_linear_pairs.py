"""Which FP8 products take the tiles that run two to a CU (csrc/linear_plan.h,
plain C++, run here from a small library built with g++): those of few steps
with many mostly filled tiles, and the tiles cover the outputs."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
MID = 1


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("pairs")
    src = d / "pairs.cpp"
    src.write_text('''#include "linear_plan.h"
extern "C" void plan(int64_t M, int64_t N, int64_t C, int gated, int cus, int64_t* o) {
    const tans_linear::Plan p = tans_linear::plan(M, N, C, gated, cus);
    const int64_t v[] = {p.kind, p.pairs, p.mi, p.nw, p.splits, p.tiles_m, p.tiles_n, p.bytes};
    for (int i = 0; i < 8; i++) o[i] = v[i];
}
''')
    out = d / "libpairs.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    I = ctypes.c_int64
    lib.plan.argtypes = [I, I, I, ctypes.c_int, ctypes.c_int, ctypes.POINTER(I)]

    def f(M, N, C, gated, cus=256):
        o = (I * 8)()
        lib.plan(M, N, C, int(gated), cus, o)
        return dict(zip(("kind", "pairs", "mi", "nw", "splits", "tiles_m", "tiles_n", "bytes"), o))
    return f


def test_few_steps_and_many_tiles(plan):
    p = plan(1101, 15045, 528, False)
    assert p["kind"] == MID and p["pairs"] and (p["mi"], p["nw"], p["splits"]) == (4, 4, 1)
    assert (p["tiles_m"], p["tiles_n"], p["bytes"]) == (9, 118, 0)
    assert plan(2047, 2177, 144, True)["pairs"]
    assert not plan(1101, 15045, 896, False)["pairs"]      # seven steps
    assert not plan(129, 40000, 528, False)["pairs"]       # half of the tiles' rows empty
    assert not plan(1000, 5000, 528, False)["pairs"]       # 320 tiles


@pytest.mark.parametrize("cus", [1, 256, 304])
def test_tiles_cover_and_launches_fit(plan, cus):
    rng = random.Random(cus)
    pairs = 0
    for _ in range(2000):
        M, N = (int(2 ** rng.uniform(0, 20)) for _ in range(2))
        C, gated = 16 * rng.randint(1, 60), rng.random() < 0.5
        p = plan(M, N, C, gated, cus)
        if not p["pairs"]:
            continue
        pairs += 1
        rows_n = 64 if gated else 128
        assert C <= 768 and p["splits"] == 1 and p["tiles_m"] * p["tiles_n"] >= 2 * cus
        assert (p["tiles_m"] - 1) * 128 < M <= p["tiles_m"] * 128
        assert (p["tiles_n"] - 1) * rows_n < N <= p["tiles_n"] * rows_n
        assert p["tiles_m"] * p["tiles_n"] * 256 < 2 ** 31
    assert pairs > 100
    assert not plan(2 ** 31 - 1, 2 ** 27, 16, False, cus)["pairs"]
