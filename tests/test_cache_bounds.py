"""Which slot of the cache a row of the batch is written to (csrc/cache_rows.h, plain
C++, run here from a small library built with g++), whatever starts, lengths and page
table hold."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
I32, I64 = ctypes.c_int32, ctypes.c_int64
LOW, HIGH = -(1 << 31), (1 << 31) - 1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("bounds")
    src = d / "bounds.cpp"
    src.write_text('''#include "cache_rows.h"
// o[0]: 0 row n is no sequence's, 1 it is one's but has no slot, 2 nor a page, 3 it has a row;
// then its sequence, slot, entry of the table and row
extern "C" void place(const int32_t* table, const int32_t* starts, const int32_t* lens, int B, int per, int N,
                      uint32_t pages, uint32_t heads, uint32_t page, int n, uint32_t h, int64_t* o) {
    tans_cache::Batch x = {table, starts, lens, B, per, N, pages, heads, 0, 0, 0};
    x.set_page(page);
    const int b = tans_cache::find_sequence(B, [&](int lo, int step, int hi) {
        int k = 0;
        for (int lane = 0; lane < 64; lane++) {
            const int64_t i = lo + (int64_t)(lane + 1) * step - 1;
            k += i < hi && starts[i] <= n;
        }
        return k;
    });
    for (int i = 0; i < 5; i++) o[i] = 0;
    if (!x.owns(b, n)) return;
    o[0] = 1, o[1] = b;
    uint32_t s, r;
    if (!x.slot_of(b, n, s)) return;
    o[0] = 2, o[2] = s, o[3] = (int64_t)b * per + x.page_of(s);
    if (o[3] < 0 || o[3] >= (int64_t)B * per) return;   // (outside the table: the test fails)
    if (x.row(b, s, h, r)) o[0] = 3, o[4] = r;
}
''')
    out = d / "libbounds.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    return ctypes.CDLL(str(out))


def _place(lib, table, starts, lens, per, N, pages, heads, page, n, h):
    o = (I64 * 5)()
    c = lambda x: (I32 * max(len(x), 1))(*x)   # noqa: E731
    lib.place(c(table), c(starts), c(lens), len(lens), per, N, pages, heads, page, n, h, o)
    return list(o)


def test_starts_that_go_back_give_no_slot_before_the_first(lib):
    for n in range(8):
        kind, b, slot, entry, row = _place(lib, [0, 1, 2, 3] * 3, [5, 6, 0, 8], [0, 0, 0], 4, 8, 4, 2, 16, n, 1)
        # rows 0 .. 4 would be tokens -5 .. -1 of sequence 0
        assert (kind, b, slot) == ((0, 0, 0) if n < 6 else (3, 2, n)), n


@pytest.mark.parametrize("seed", range(40))
def test_no_number_leaves_the_table_or_the_cache(lib, seed):
    rng = random.Random(seed)
    for _ in range(60):
        B, N, per = int(200 ** rng.random()), int(300 ** rng.random()), rng.choice((0, 1, 2, 5, 40))
        pages, heads, page = rng.randint(1, 9), rng.randint(1, 4), rng.choice((1, 2, 7, 16, 48, 1 << 20))
        page = min(page, HIGH // max(per, 1), ((1 << 32) - 1) // (pages * heads))
        some = lambda: rng.choice((rng.randint(-3, N + 3), rng.randint(0, N), LOW, HIGH))   # noqa: E731
        starts = [some() for _ in range(B + 1)]
        if rng.random() < 0.2:
            starts.sort()
        lens = [rng.choice((0, rng.randint(-5, per * page + 5), per * page - 1, LOW, HIGH)) for _ in range(B)]
        table = [rng.choice((rng.randint(0, pages - 1), -1, pages, LOW, HIGH)) for _ in range(B * per)]
        for n in range(N):
            kind, b, slot, entry, row = _place(lib, table, starts, lens, per, N, pages, heads, page, n, heads - 1)
            clamped = lambda x: min(max(x, 0), N)   # noqa: E731
            if kind:
                assert 0 <= b < B and clamped(starts[b]) <= n < clamped(starts[b + 1])
            if kind >= 2:
                assert slot == min(max(lens[b], 0), per * page) + n - clamped(starts[b])
                assert 0 <= slot < per * page and entry == b * per + slot // page
                assert (kind == 3) == (0 <= table[entry] < pages)
            if kind == 3:
                assert row == (table[entry] * heads + heads - 1) * page + slot % page < pages * heads * page


@pytest.mark.parametrize("B", [1, 3, 64, 65, 700])
def test_rows_of_sorted_starts_have_the_slots_behind_the_context(lib, B):
    rng = random.Random(B)
    counts = [rng.randint(0, 4) for _ in range(B)]
    starts = [2 + sum(counts[:b]) for b in range(B + 1)]
    lens = [rng.randint(0, 60) for _ in range(B)]
    N = starts[-1] + 3
    table = [rng.randint(0, 8) for _ in range(B * 4)]
    owner = [None] * 2 + [(b, t) for b in range(B) for t in range(counts[b])] + [None] * 3
    for n in range(N):
        kind, b, slot, entry, row = _place(lib, table, starts, lens, 4, N, 9, 2, 16, n, 0)
        if owner[n] is None:
            assert kind == 0
        else:
            assert (b, slot) == (owner[n][0], lens[owner[n][0]] + owner[n][1]) if kind > 1 else \
                (kind == 1 and lens[owner[n][0]] + owner[n][1] >= 64)
