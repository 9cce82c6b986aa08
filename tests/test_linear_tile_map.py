"""Which workgroup of the FP8 product takes which tile (csrc/linear_plan.h, plain
C++, run here from a small library built with g++): over all workgroups of a
launch every tile is taken exactly once, whatever the number of CUs, and lies
where no other does."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("tile_map")
    src = d / "map.cpp"
    src.write_text('''#include "linear_plan.h"
#include <vector>
using namespace tans_linear;
// 0, or what is wrong with the persistent workgroups' shares
extern "C" int shares(int tiles_m, int tiles_n, int cus) {
    const TileMap map = {tiles_m, tiles_n};
    const int T = map.count();
    const int64_t blocks = tile_blocks(T, cus);
    if (blocks < 1 || blocks > T || (cus >= kXcds && blocks > cus)) return 1;
    std::vector<int> taken(T, 0), at(T, 0);
    for (int b = 0; b < blocks; b++) {
        if (map.at(0, b, (int)blocks) < 0) return 2;    // a workgroup without a tile
        for (int i = 0, t; (t = map.at(i, b, (int)blocks)) >= 0; i++) {
            if (t >= T || taken[t]++) return 3;
            int tm = -1, tn = -1;
            map.place(t, tm, tn);
            if (tm < 0 || tm >= tiles_m || tn < 0 || tn >= tiles_n || at[tm * tiles_n + tn]++) return 4;
        }
    }
    for (int t = 0; t < T; t++)
        if (taken[t] != 1) return 5;
    return 0;
}
extern "C" int permutes(int blocks) {
    std::vector<int> seen(blocks, 0);
    for (int b = 0; b < blocks; b++) {
        const int k = xcd_order(b, blocks);
        if (k < 0 || k >= blocks || seen[k]++) return 1;
    }
    return 0;
}
''')
    out = d / "libmap.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    return ctypes.CDLL(str(out))


@pytest.mark.parametrize("cus", [1, 2, 7, 8, 9, 32, 64, 255, 256, 304])
def test_every_tile_is_taken_once(lib, cus):
    for tm in (1, 2, 3, 7, 8, 9, 16, 17, 33, 274):
        for tn in (1, 2, 5, 8, 13, 64, 137, 182):
            assert lib.shares(tm, tn, cus) == 0, (tm, tn, cus)


def test_the_order_by_xcd_is_a_permutation(lib):
    for blocks in (*range(1, 70), 255, 256, 257, 1003, 8050):
        assert lib.permutes(blocks) == 0, blocks
