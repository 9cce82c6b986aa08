"""How much work a batch is counted as, and who computes it where its starts go back
(csrc/attention_plan.h and cache_rows.h, plain C++, run here from a small library built
with g++)."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
I, I32 = ctypes.c_int64, ctypes.c_int32
TOP = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("work")
    src = d / "work.cpp"
    src.write_text('''#include "attention_plan.h"
using namespace tans_attention;
static Plan plan_of(int64_t N, int64_t B, int64_t Hq, int64_t heads, int64_t dim, int64_t slots, int64_t most) {
    return plan(N, B, Hq, heads, dim, false, slots, most, 256);
}
// o: whole, workgroups, the most pieces, the batch's (a lane's sums, then theirs), the tiles
extern "C" void work(const int32_t* starts, const int32_t* lens, int64_t N, int64_t B, int64_t Hq, int64_t heads,
                     int64_t dim, int64_t per, int64_t page, int64_t most, int64_t* o) {
    const Plan p = plan_of(N, B, Hq, heads, dim, per * page, most);
    tans_cache::Batch x = {nullptr, starts, lens, (int)B, (int)per, (int)N, 1, (uint32_t)heads, 0, 0, 0};
    x.set_page((uint32_t)page);
    int64_t lane[64] = {}, all = 0, tiles = 0;
    for (int b = 0; b < B; b++) {
        const int t = row_tiles(x.tokens(b), Hq / heads, p.work.rows);
        const int64_t s = (int64_t)x.context(b) + x.tokens(b);
        const int u = slot_units((int)(s < x.capacity() ? s : x.capacity()));
        lane[b % 64] = add_pieces(p.work, lane[b % 64], pieces_of(p.work, heads, t, u));
        tiles += t;
    }
    for (int i = 0; i < 64; i++) all = add_pieces(p.work, all, lane[i]);
    o[0] = p.work.whole, o[1] = p.blocks, o[2] = p.work.most, o[3] = all, o[4] = tiles;
    o[5] = p.work.rows, o[6] = p.work.item;
}
extern "C" int64_t start_(int64_t all, int groups, int i) { return range_start(all, groups, i); }
extern "C" int of_(int64_t all, int groups, int64_t at) { return range_of(all, groups, at); }
''')
    out = d / "libwork.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.work.argtypes = [ctypes.POINTER(I32)] * 2 + [I] * 8 + [ctypes.POINTER(I)]
    lib.start_.argtypes, lib.start_.restype = [I, ctypes.c_int, ctypes.c_int], I
    lib.of_.argtypes = [I, ctypes.c_int, I]
    return lib


def _work(lib, starts, lens, N, Hq, heads, dim, per, page, most):
    o = (I * 7)()
    lib.work((I32 * len(starts))(*starts), (I32 * len(lens))(*lens), N, len(lens), Hq, heads, dim, per, page, most, o)
    return dict(zip(("whole", "blocks", "most", "all", "tiles", "rows", "item"), o))


def test_batches_are_counted_whole(lib):
    """Sorted starts: every piece, whatever the lengths are."""
    rng = random.Random(1)
    for _ in range(2000):
        B, heads, page = int(300 ** rng.random()), rng.choice((1, 2, 8)), rng.choice((1, 7, 16, 64))
        G, per = rng.randint(1, 9), int(3000 ** rng.random())
        counts = [rng.choice((0, 1, int(700 ** rng.random()))) for _ in range(B)]
        starts = [sum(counts[:b]) for b in range(B + 1)]
        lens = [rng.choice((0, rng.randint(0, per * page), TOP)) for _ in range(B)]
        N = starts[-1] + rng.randint(0, 3)
        if N == 0:
            continue
        w = _work(lib, starts, lens, N, heads * G, heads, rng.choice((64, 128, 256)), per, page, rng.randint(0, N))
        want = 0
        for c, t in zip(lens, counts):
            tiles = -(-t * G // w["rows"])
            units = max(1, -(-min(min(c, per * page) + t, per * page) // 32))
            want += heads * tiles * (1 if w["whole"] else units + w["item"])
        assert w["all"] == want <= w["most"]
        assert not w["whole"] or want <= w["blocks"]


@pytest.mark.parametrize("B,N,per", [(1000, 1000, 100), (4001, 50000, 1 << 11), (70001, (1 << 30) - 1, 1 << 11)])
def test_starts_that_go_back_are_counted_up_to_a_proper_batch(lib, B, N, per):
    page = TOP // per
    starts, lens = [(b % 2) * TOP for b in range(B + 1)], [TOP] * B
    w = _work(lib, starts, lens, N, 1, 1, 128, per, page, 1)
    assert w["all"] == w["most"] <= 1 << 50 and w["tiles"] > 2 * N // w["rows"]
    assert not w["whole"]
    groups = w["blocks"]
    # the runs are in order, and whose a piece is stays a workgroup, also behind the last
    starts = [lib.start_(w["all"], groups, i) for i in range(groups + 1)]
    assert starts[0] == 0 and starts[-1] == w["all"] and all(a < b for a, b in zip(starts, starts[1:]))
    for i in (0, 1, groups // 2, groups - 1):
        assert lib.of_(w["all"], groups, starts[i]) == i == lib.of_(w["all"], groups, starts[i + 1] - 1)
    for behind in (0, 1, 1 << 30, 1 << 50):
        assert lib.of_(w["all"], groups, w["all"] + behind) == groups - 1


def test_the_longest_line_of_work_stays_in_range(lib):
    """The most sequences, tokens, heads and slots that the entry takes: no product of
    pieces and workgroups leaves 64 bits."""
    for N, B, Hq, heads in ((TOP // 2, TOP - 1, 1, 1), (TOP // 65535, TOP - 1, 65535, 65535), (TOP // 64, 1 << 22, 64, 64)):
        w = _work(lib, [0, 0], [0], N, Hq, heads, 64, 1, TOP, 1)
        assert 0 < w["most"] <= 1 << 50
        assert lib.start_(w["most"], 4095, 4095) == w["most"] and lib.of_(w["most"], 4095, w["most"] - 1) == 4094
