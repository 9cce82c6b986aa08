"""Which units of a row tile are computed, and which of them without a mask
(csrc/attention_plan.h, plain C++, run here from a small library built with g++),
against the rule of what a token sees."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
UNIT = 32


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("tiles")
    src = d / "tiles.cpp"
    src.write_text('''#include "attention_plan.h"
using namespace tans_attention;
extern "C" void tile(int masked, int context, int tokens, int slots, int tile, int rows, int G, int end, int* o) {
    o[0] = tile_stop(masked, context, tokens, slots, tile, rows, G, end);
    o[1] = tile_plain(masked, context, slots, tile, rows, G, o[0]);
    o[2] = slot_units(slots);
    o[3] = row_tiles(tokens, G, rows);
}
''')
    out = d / "libtiles.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    return ctypes.CDLL(str(out))


def _tile(lib, *a):
    o = (ctypes.c_int * 4)()
    lib.tile(*(int(x) for x in a), o)
    return list(o)


def _sequence(lib, masked, context, tokens, capacity, rows, G):
    """Every tile of a sequence, whole and cut at some unit."""
    context = min(context, capacity)
    slots = min(context + tokens, capacity)
    units, tiles = _tile(lib, masked, context, tokens, slots, 0, rows, G, 0)[2:]
    for tile in range(tiles):
        first = tile * rows // G
        last = min(tokens - 1, (tile * rows + rows - 1) // G)
        for end in {units, units // 2 + 1}:
            stop, plain = _tile(lib, masked, context, tokens, slots, tile, rows, G, end)[:2]
            assert 0 <= plain <= stop <= end
            # plain units hold slots of the sequence only, and the first token sees them all
            assert plain * UNIT <= slots
            assert plain * UNIT <= context + (0 if masked else first + 1)
            # no slot that the last token sees lies behind stop
            seen = slots if masked else min(slots, context + last + 1)
            assert stop == end or stop * UNIT >= seen
    return tiles


@pytest.mark.parametrize("rows", [32, 64, 128, 256])
def test_tables_without_columns_have_no_plain_unit(lib, rows):
    for masked in (0, 1):
        for G in (1, 3, 8):
            for tokens in (1, 31, 32, 129, 200, 700):
                assert _sequence(lib, masked, 0, tokens, 0, rows, G) > 0
                for tile in range(-(-tokens * G // rows)):
                    assert _tile(lib, masked, 0, tokens, 0, tile, rows, G, 1)[:2] == [1, 0]


@pytest.mark.parametrize("rows", [32, 64, 128, 256])
def test_tiles(lib, rows):
    rng = random.Random(rows)
    for _ in range(3000):
        context = rng.choice((0, rng.randint(0, 40), int(5000 ** rng.random())))
        tokens = int(1500 ** rng.random())
        capacity = rng.choice((1 << 20, context + tokens, context, rng.randint(0, context + tokens)))
        _sequence(lib, rng.random() < 0.5, context, tokens, capacity, rows, rng.randint(1, 16))


def test_the_longest_sequences(lib):
    top = (1 << 31) - 1
    for masked in (0, 1):
        for context, tokens in ((top, 3), (top - 70, 70), (1 << 30, 5000)):
            _sequence(lib, masked, context, tokens, top, 256, 5)
