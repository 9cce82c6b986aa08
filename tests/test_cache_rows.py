"""Which row of the cache and which piece of the work is whose (csrc/cache_rows.h and
csrc/attention_plan.h, plain C++, run here from a small library built with g++)."""
import bisect
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
FEW, SOME, MANY, MOST = range(4)
I, P = ctypes.c_int64, ctypes.POINTER


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("rows")
    src = d / "rows.cpp"
    src.write_text('''#include "attention_plan.h"
using namespace tans_attention;
extern "C" int64_t wrong_pages(uint32_t page, const uint32_t* slots, int64_t n) {
    tans_cache::Batch b = {};
    b.set_page(page);
    int64_t bad = 0;
    for (int64_t i = 0; i < n; i++) bad += b.page_of(slots[i]) != slots[i] / page;
    return bad;
}
extern "C" int find(const int32_t* starts, int B, int n) {
    return tans_cache::find_sequence(B, [&](int lo, int step, int hi) {
        int k = 0;
        for (int lane = 0; lane < 64; lane++) {
            const int64_t i = lo + (int64_t)(lane + 1) * step - 1;
            k += i < hi && starts[i] <= n;
        }
        return k;
    });
}
extern "C" int row(const int32_t* table, const int32_t* starts, const int32_t* lens, int B, int per, int N,
                   uint32_t pages, uint32_t heads, uint32_t page, int b, uint32_t s, uint32_t h, int64_t* o) {
    tans_cache::Batch x = {table, starts, lens, B, per, N, pages, heads, 0, 0, 0};
    x.set_page(page);
    uint32_t r = 0;
    const bool ok = x.row(b, s, h, r);
    o[0] = r, o[1] = x.tokens(b), o[2] = x.context(b), o[3] = x.start(b);
    return ok;
}
extern "C" int64_t range_start_(int64_t all, int groups, int i) { return range_start(all, groups, i); }
extern "C" int range_of_(int64_t all, int groups, int64_t at) { return range_of(all, groups, at); }
extern "C" void plan_(int64_t N, int64_t B, int64_t Hq, int64_t heads, int64_t dim, int eight, int64_t slots,
                      int64_t most, int cus, int64_t* o) {
    const Plan p = plan(N, B, Hq, heads, dim, eight, slots, most, cus);
    const int64_t v[] = {p.kind, p.work.rows, p.work.groups, p.work.least, p.work.item, p.work.whole, p.pairs,
                         p.blocks, p.parts_bytes, p.bytes};
    for (int i = 0; i < 10; i++) o[i] = v[i];
}
extern "C" int run_of_(int i, int groups) { return run_of(i, groups); }
extern "C" int groups_(int least, int groups, int64_t all) {
    Work w = {};
    w.least = least, w.groups = groups;
    return work_groups(w, all);
}
''')
    out = d / "librows.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.wrong_pages.argtypes, lib.wrong_pages.restype = [ctypes.c_uint32, P(ctypes.c_uint32), I], I
    lib.range_start_.argtypes, lib.range_start_.restype = [I, ctypes.c_int, ctypes.c_int], I
    lib.range_of_.argtypes = [I, ctypes.c_int, I]
    lib.plan_.argtypes = [I, I, I, I, I, ctypes.c_int, I, I, ctypes.c_int, P(I)]
    lib.groups_.argtypes = [ctypes.c_int, ctypes.c_int, I]
    return lib


def _plan(lib, *a):
    o = (I * 10)()
    lib.plan_(*a, o)
    return dict(zip(("kind", "rows", "groups", "least", "item", "whole", "pairs", "blocks", "parts", "bytes"), o))


def test_pages_of_slots_without_a_division(lib):
    """At every multiple of the page's rows and beside it, the largest slots among them."""
    rng = random.Random(1)
    pages = list(range(1, 300)) + [1000, 4095, 4096, 4097, 65535, 65536, 65537, (1 << 20) - 1, 1 << 20]
    pages += [rng.randint(1, 1 << 20) for _ in range(200)]
    for page in pages:
        top = (1 << 31) - 1
        at = [0, 1, top, top - 1]
        for k in [1, 2, 3, top // page] + [rng.randint(1, top // page) for _ in range(60)]:
            at += [k * page - 1, k * page, k * page + 1]
        at = [x for x in at if 0 <= x <= top]
        assert lib.wrong_pages(page, (ctypes.c_uint32 * len(at))(*at), len(at)) == 0, page


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 129, 4096, 4097, 5000])
def test_the_last_sequence_that_starts_before_a_row(lib, B):
    rng = random.Random(B)
    starts = sorted(rng.randint(0, 3 * B) for _ in range(B))
    starts[0] = rng.choice((0, 2))
    starts.sort()
    c = (ctypes.c_int32 * (B + 1))(*starts, 3 * B)
    for n in [0, 1, 2, 3 * B - 1] + [rng.randint(0, 3 * B) for _ in range(200)]:
        assert lib.find(c, B, n) == bisect.bisect_right(starts, n) - 1, n


def test_rows_and_numbers_out_of_range(lib):
    o = (I * 4)()
    i32 = lambda *x: (ctypes.c_int32 * len(x))(*x)   # noqa: E731
    table, starts, lens = i32(4, -1, 7, 2, 0, 1), i32(0, 3, 2, 99), i32(-5, 1 << 30, 13)

    def row(b, s, h):
        ok = lib.row(table, starts, lens, 3, 2, 10, 7, 3, 5, b, s, h, o)
        return ok, o[0]
    assert row(0, 3, 2) == (1, (4 * 3 + 2) * 5 + 3)
    assert row(0, 5, 0)[0] == 0                       # page -1
    assert row(1, 0, 0)[0] == 0                       # page 7 of 7
    assert row(1, 9, 1) == (1, (2 * 3 + 1) * 5 + 4)
    assert list(o)[1:] == [0, 10, 3]                  # starts that go back; more slots than the table has
    row(0, 0, 0)
    assert list(o)[1:] == [3, 0, 0]
    row(2, 0, 0)
    assert list(o)[1:] == [8, 10, 2]                  # starts past the rows


def test_runs_of_the_work_share_it_and_say_whose_a_piece_is(lib):
    rng = random.Random(3)
    for _ in range(300):
        groups = rng.choice((1, 2, 3, 64, 255, 256, 512, 2048))
        all_ = rng.choice((groups, groups + 1, rng.randint(groups, 100 * groups), rng.randint(1 << 30, 1 << 40),
                           1 << 47))
        start = [lib.range_start_(all_, groups, i) for i in range(groups + 1)]
        assert start[0] == 0 and start[-1] == all_ and all(a < b for a, b in zip(start, start[1:]))
        assert max(b - a for a, b in zip(start, start[1:])) - min(b - a for a, b in zip(start, start[1:])) <= 1
        for at in [0, all_ - 1] + [start[rng.randrange(groups)] for _ in range(9)] + \
                [rng.randrange(all_) for _ in range(9)] + [start[rng.randrange(1, groups + 1)] - 1 for _ in range(9)]:
            i = lib.range_of_(all_, groups, at)
            assert start[i] <= at < start[i + 1]
    for all_ in (1, 7, 8, 9, 100, 10 ** 9):
        g = lib.groups_(8, 256, all_)
        assert 1 <= g <= 256 and (g == 256 or g * 8 >= all_)


def _batches(n, seed):
    rng = random.Random(seed)
    for _ in range(n):
        B = int(300 ** rng.random())
        counts = [int(2000 ** rng.random()) for _ in range(B)] if rng.random() < 0.7 else [1] * B
        heads = rng.choice((1, 2, 4, 8, 16))
        yield counts, B, heads * rng.randint(1, 16), heads, rng.choice((64, 128, 256)), rng.random() < 0.5, \
            16 * int(20000 ** rng.random())


@pytest.mark.parametrize("groups", [1, 7, 8, 60, 256, 304, 512, 513])
def test_every_run_has_its_workgroup(lib, groups):
    runs = [lib.run_of_(i, groups) for i in range(groups)]
    assert sorted(runs) == list(range(groups))
    if groups % 8 == 0:   # an XCD's workgroups have runs that follow each other
        for x in range(8):
            assert runs[x::8] == list(range(x * groups // 8, (x + 1) * groups // 8))


@pytest.mark.parametrize("cus", [1, 64, 256, 304])
def test_plans(lib, cus):
    seen = set()
    for counts, B, Hq, heads, D, eight, slots in _batches(4000, cus):
        N, G = sum(counts), Hq // heads
        p = _plan(lib, N, B, Hq, heads, D, eight, slots, max(counts), cus)
        # a tile's rows are its kernel's, and D = 256 has none for 64 rows or 256
        assert p["rows"] == 32 << p["kind"] and (D < 256 or p["kind"] in (FEW, MANY))
        if p["whole"]:
            # a workgroup for each item at least, whatever the sequences' tokens
            assert p["blocks"] >= heads * sum(-(-t * G // p["rows"]) for t in counts) and p["bytes"] == 0
        else:
            # two workgroups a CU where the plan says so, and of 128 rows with D below 256
            two = p["pairs"] or (p["kind"] == MANY and D < 256)
            assert p["blocks"] == p["groups"] == cus * (2 if two else 1)
            # two parts of a tile and its rows' statistics for each workgroup, and its record
            assert p["parts"] == p["groups"] * 2 * p["rows"] * (D + 2) * 4
            assert p["bytes"] == p["parts"] + p["groups"] * 20
            assert p["rows"] % 32 == 0 and p["item"] >= 1
        # what the workspace is asked for holds either cache
        assert _plan(lib, N, B, Hq, heads, D, True, slots, max(counts), cus)["bytes"] >= p["bytes"]
        seen.add((p["kind"], p["whole"], p["pairs"]))
    if cus == 256:   # each kernel is some batch's choice
        assert seen >= {(k, w, 0) for k in range(4) for w in (0, 1)} | {(FEW, 0, 1)}
