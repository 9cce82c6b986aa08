"""The choice of attention's kernel at the largest numbers that its entries take
(csrc/attention_plan.h, plain C++, run here from a small library built with g++)."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "tans-vectoradd_amd", "csrc")
I = ctypes.c_int64
MOST = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("limits")
    src = d / "limits.cpp"
    src.write_text('''#include "attention_plan.h"
using namespace tans_attention;
extern "C" void plan_(int64_t N, int64_t B, int64_t Hq, int64_t heads, int64_t dim, int eight, int64_t slots,
                      int64_t most, int cus, int64_t* o) {
    const Plan p = plan(N, B, Hq, heads, dim, eight, slots, most, cus);
    const int64_t v[] = {p.kind, p.work.rows, p.work.groups, p.work.whole, p.pairs, p.blocks, p.bytes};
    for (int i = 0; i < 7; i++) o[i] = v[i];
}
''')
    out = d / "liblimits.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(src), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.plan_.argtypes = [I, I, I, I, I, ctypes.c_int, I, I, ctypes.c_int, ctypes.POINTER(I)]
    return lib


def _plan(lib, *a):
    o = (I * 7)()
    lib.plan_(*a, 256, o)
    return list(o)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_any_number_of_tokens_that_a_sequence_may_have(lib, dim):
    for heads, G in ((1, 1), (1, 2), (3, 5), (8, 8), (1, 65535)):
        for slots in (100, 100000):
            want = _plan(lib, 5000, 7, heads * G, heads, dim, 0, slots, MOST)
            assert want[1] == (128 if dim == 256 else 256)
            for most in (MOST + 1, 1 << 40, 1 << 61, 1 << 62, (1 << 63) - 1, ((1 << 63) - 1) // G):
                assert _plan(lib, 5000, 7, heads * G, heads, dim, 0, slots, most) == want, (heads, G, most)
