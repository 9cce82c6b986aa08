"""The alignment that tans_fp8_linear asks for, of each buffer (CPU only: an
error code before any GPU work)."""
import ctypes

P = ctypes.c_void_p


def test_each_buffers_alignment():
    from rans_vectoradd._lib import lib
    ok = 1 << 12

    def call(**kw):
        p = {n: P(kw.get(n, ok)) for n in ("a", "sa", "w", "sw", "bias", "res", "ws", "y")}
        return lib.tans_fp8_linear(p["a"], p["sa"], p["w"], p["sw"], ctypes.c_float(1.0), p["bias"],
                                   p["res"], 0, 0, 4, 64, 64, p["ws"], 1 << 40, p["y"], None)

    for name, least in (("a", 16), ("w", 16), ("y", 16), ("sa", 4), ("sw", 4), ("bias", 2), ("res", 2)):
        assert call(**{name: ok + least // 2}) == -1, name
        assert b"misaligned" in lib.tans_last_error(), name
