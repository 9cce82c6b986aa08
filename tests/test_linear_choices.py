"""The kernels that the products of the GPU tests take on 256 CUs
(csrc/linear_plan.h, plain C++, run here from a small library built with g++), so
that a change of the choice's constants cannot leave a kernel without its tests:
each named case takes the kernel that it names, those of several tiles a
workgroup are more tiles than CUs, and every kernel and tile is some product's."""
import ctypes
import os
import random
import subprocess

import pytest

import test_gpu_layer_in_place as in_place
import test_gpu_linear_exact as exact

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
CUS = 256


@pytest.fixture(scope="module")
def choice(tmp_path_factory):
    d = tmp_path_factory.mktemp("choices")
    src = d / "choices.cpp"
    src.write_text('''#include "linear_plan.h"
extern "C" void plan(int64_t M, int64_t N, int64_t C, int gated, int cus, int64_t* o) {
    const tans_linear::Plan p = tans_linear::plan(M, N, C, gated, cus);
    const int64_t v[] = {p.kind, p.few, p.pairs, p.mi, p.nw, p.splits, p.tiles_m * p.tiles_n};
    for (int i = 0; i < 7; i++) o[i] = v[i];
}
extern "C" int mids(int64_t* o) {
    int n = 0;
    for (const auto& t : tans_linear::kMids) { o[n++] = t.mi; o[n++] = t.nw; }
    return n / 2;
}
''')
    out = d / "libchoices.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    I = ctypes.c_int64
    lib.plan.argtypes = [I, I, I, ctypes.c_int, ctypes.c_int, ctypes.POINTER(I)]

    def f(M, R_, C, gated):
        """(kernel's name, (mi, nw), tiles)"""
        o = (I * 7)()
        lib.plan(M, R_ // 2 if gated else R_, C, int(gated), CUS, o)
        kind, few, pairs, mi, nw, splits, tiles = o
        name = (("few" if few else "stream") if kind == 0 else f"tiles {32 * nw}" if kind == 2 else
                "pairs" if pairs else "mid split" if splits > 1 else "mid")
        return name, (mi, nw), tiles
    o = (I * 64)()
    f.mids = [(o[2 * i], o[2 * i + 1]) for i in range(lib.mids(o))]
    return f


@pytest.mark.parametrize("M,R_,C,gated,kernel",
                         exact.CASES + exact.MANY + [exact.PAST_4_GIB] + in_place.CASES)
def test_case_takes_the_kernel_it_names(choice, M, R_, C, gated, kernel):
    assert choice(M, R_, C, gated)[0] == kernel


@pytest.mark.parametrize("M,R_,C,gated,kernel", exact.MANY + [exact.PAST_4_GIB])
def test_case_has_several_tiles_a_workgroup(choice, M, R_, C, gated, kernel):
    assert choice(M, R_, C, gated)[2] > CUS


def test_every_kernel_is_named(choice):
    want = {"few", "stream", "mid", "mid split", "pairs", "tiles 192", "tiles 256"}
    assert {c[4] for c in exact.CASES} == want == {c[4] for c in in_place.CASES}
    assert {(c[3], c[4]) for c in exact.MANY} == {(True, "tiles 256"), (False, "tiles 256"),
                                                  (False, "tiles 192")}


def test_every_tile_is_some_products_choice_without_pairs(choice):
    """Tiles of 128 x 128 one to a CU are a choice beside the pairs."""
    rng = random.Random(5)

    def size(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))
    seen = set()
    for _ in range(6000):
        name, tile, _ = choice(size(17, 20000), 2 * size(1, 40000), 16 * size(1, 2000), rng.random() < 0.5)
        if name.startswith("mid"):
            seen.add(tile)
    assert seen == set(choice.mids)
