"""Host side of the microscaled operators: sizes, the refusals of every entry point, and the place of each scale byte
(csrc/mx_index.h, compiled here as plain C). No GPU."""
import ctypes as C
import os
import subprocess
import threading

import pytest

import tcg

CSRC = os.path.join(os.path.dirname(os.path.dirname(tcg.LIB_PATH)), "csrc")
P = 1 << 20                          # a pointer that nothing reads: every call here is refused before


def _mx(rows=3, cols=64, bits=8, codes=P, scales=P):
    return tcg.Mx(codes, scales, rows, cols, bits)


def _refused(fn, *args, about=None):
    assert fn(*args) is False, args
    assert fn.__name__ in tcg.err() and (about is None or about in tcg.err()), tcg.err()


def test_sizes():
    L = tcg.lib()
    for rows, cols, wide in [(1, 1, 128), (1, 128, 128), (3, 129, 256), (128, 4096, 4096), (129, 14336, 14336)]:
        assert L.tcg_mx_code_bytes(rows, cols, 8) == rows * wide
        assert L.tcg_mx_code_bytes(rows, cols, 4) == rows * wide // 2
        assert L.tcg_mx_scale_bytes(rows, cols) == (rows + 127) // 128 * 128 * wide // 32
    assert L.tcg_mx_code_bytes(1 << 30, 1 << 24, 8) == 1 << 54 and L.tcg_mx_scale_bytes(1 << 30, 1 << 24) == 1 << 49
    for rows, cols, bits in [(-1, 4, 4), (1, 0, 4), (1, -3, 4), (1, 4, 6), ((1 << 30) + 1, 4, 4), (1, (1 << 24) + 1, 4)]:
        assert L.tcg_mx_code_bytes(rows, cols, bits) == 0
        assert bits == 6 or L.tcg_mx_scale_bytes(rows, cols) == 0
    assert L.tcg_mx_code_bytes(0, 4, 4) == 0 and L.tcg_mx_scale_bytes(0, 4) == 0


BAD_MX = [dict(bits=6), dict(bits=0), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(cols=0), dict(cols=-5), dict(cols=(1 << 24) + 1),
          dict(codes=None), dict(scales=None), dict(codes=P + 16), dict(scales=P + 8)]


@pytest.mark.parametrize("bad", BAD_MX, ids=str)
def test_matrices_that_cannot_be(bad):
    L, m, fine = tcg.lib(), _mx(**bad), _mx()
    w = _mx(rows=5, bits=4)
    rows, cols = bad.get("rows", 3), bad.get("cols", 64)
    _refused(L.tcg_mx_quantize, C.byref(m), P, 64, 0)
    _refused(L.tcg_mx_dequantize, P, C.byref(m), 64, 0)
    _refused(L.tcg_mx_linear, P, C.byref(m), C.byref(w), None, 64, 0)
    _refused(L.tcg_mx_linear, P, C.byref(fine), C.byref(m), None, 64, 0)
    _refused(L.tcg_add_rms_norm, None, None, C.byref(m), P, None, P, 1e-6, rows, cols, 64, 64, 64, 64, 0)


def test_refusals():
    L, m, r = tcg.lib(), _mx(), C.byref
    w = _mx(rows=5, bits=4)
    for t in (2, 12, -1, 99):
        _refused(L.tcg_mx_quantize, r(m), P, 64, t, about="type")
        _refused(L.tcg_mx_dequantize, P, r(m), 64, t, about="type")
        _refused(L.tcg_mx_linear, P, r(m), r(w), None, 64, t, about="type")
        _refused(L.tcg_add_rms_norm, P, None, None, P, None, P, 1e-6, 3, 64, 64, 64, 64, 64, t, about="type")
    for fn, args in ((L.tcg_mx_quantize, lambda p, ld, t: (r(m), p, ld, t)), (L.tcg_mx_dequantize, lambda p, ld, t: (p, r(m), ld, t))):
        _refused(fn, *args(None, 64, 0))
        _refused(fn, *args(P, 63, 0), about="stride")
        _refused(fn, *args(P, -64, 0), about="stride")
        _refused(fn, *args(P + 2, 64, 0), about="misaligned")
        _refused(fn, *args(P + 1, 64, 1), about="misaligned")
    _refused(L.tcg_mx_quantize, None, P, 64, 0)
    _refused(L.tcg_mx_dequantize, P, None, 64, 0)
    _refused(L.tcg_mx_linear, P, None, r(w), None, 64, 0)
    _refused(L.tcg_mx_linear, P, r(m), None, None, 64, 0)
    _refused(L.tcg_mx_linear, None, r(m), r(w), None, 64, 0)
    _refused(L.tcg_mx_linear, P, r(m), r(w), None, 4, 0, about="stride")
    _refused(L.tcg_mx_linear, P + 2, r(m), r(w), None, 64, 0, about="misaligned")
    _refused(L.tcg_mx_linear, P, r(m), r(w), P + 2, 64, 0, about="bias")
    _refused(L.tcg_mx_linear, P, r(m), r(_mx(rows=5, bits=8)), None, 64, 0, about="8 bits")
    _refused(L.tcg_mx_linear, P, r(m), r(_mx(rows=5, bits=4, cols=65)), None, 64, 0, about="columns")


def test_norm_refusals():
    L, m, r = tcg.lib(), _mx(), C.byref
    def norm(h=P, y=None, mx=None, x=P, res=None, w=P, eps=1e-6, n=3, cols=64, ldh=64, ldy=64, ldx=64, ldr=64, t=0):
        return (L.tcg_add_rms_norm, h, y, mx, x, res, w, eps, n, cols, ldh, ldy, ldx, ldr, t)
    for bad in (dict(h=None), dict(n=-1), dict(cols=0), dict(cols=32769), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
                dict(x=None), dict(x=P + 2), dict(ldx=63), dict(res=P, ldr=63), dict(res=P + 1), dict(ldh=60), dict(h=P + 2),
                dict(y=P, ldy=63), dict(y=P + 2), dict(y=P, w=None), dict(y=P, w=P + 2), dict(mx=r(m), w=None),
                dict(mx=r(m), n=4), dict(mx=r(m), cols=63), dict(mx=r(_mx(bits=5)))):
        _refused(*norm(**bad))


@pytest.mark.parametrize("bad, about", [
    (dict(h=P, y=P), "same rows"), (dict(h=P, y=P, n=1), "same rows"), (dict(h=P, x=P, ldh=128), "stride"),
    (dict(h=3 * P, y=P, x=P, ldx=128), "stride"), (dict(h=P, x=2 * P, res=P, ldr=65), "stride"),
    (dict(h=2 * P, y=P, x=3 * P, res=P, ldy=100), "stride"), (dict(h=P, y=2 * P, x=P, res=P, ldr=65), "stride")], ids=str)
def test_norm_in_place_refusals(bad, about):
    """Outputs over inputs only row on row, and never one over the other."""
    a = dict(h=None, y=None, x=5 * P, res=None, n=3, ldh=64, ldy=64, ldx=64, ldr=64) | bad
    _refused(tcg.lib().tcg_add_rms_norm, a["h"], a["y"], None, a["x"], a["res"], P, 1e-6, a["n"], 64, a["ldh"], a["ldy"], a["ldx"],
             a["ldr"], 0, about=about)


def test_without_a_device():
    L, got, r = tcg.lib(), {}, C.byref

    def body():                                                          # a fresh thread has no device context
        m, w = _mx(), _mx(rows=5, bits=4)
        got["quantize"] = (L.tcg_mx_quantize(r(m), P, 64, 0), tcg.err())
        got["dequantize"] = (L.tcg_mx_dequantize(P, r(m), 64, 0), tcg.err())
        got["linear"] = (L.tcg_mx_linear(P, r(m), r(w), None, 64, 0), tcg.err())
        got["norm"] = (L.tcg_add_rms_norm(P, 2 * P, r(m), P, P, P, 1e-6, 3, 64, 64, 64, 64, 64, 0), tcg.err())
        # nothing to do is still nothing without a device
        got["none"] = (L.tcg_mx_quantize(r(_mx(rows=0, codes=None, scales=None)), None, 64, 0), tcg.err())

    t = threading.Thread(target=body)
    t.start()
    t.join()
    assert len(got) == 5
    for ok, msg in got.values():
        assert ok is False and "tcg_init" in msg


def test_every_scale_has_a_place(tmp_path):
    src, so = tmp_path / "index.c", tmp_path / "index.so"
    src.write_text('''#include "mx_index.h"
size_t at(int64_t r, int64_t b, int64_t atoms) { return mx_scale_at(r, b, atoms); }
int64_t wide(int64_t cols) { return mx_wide(cols); }
int64_t pitch(int64_t cols, int bits) { return mx_pitch(cols, bits); }
''')
    subprocess.run(["gcc", "-std=c11", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-o", str(so), str(src)], check=True)
    L = C.CDLL(str(so))
    L.at.restype, L.at.argtypes = C.c_size_t, [C.c_int64] * 3
    L.wide.restype, L.wide.argtypes = C.c_int64, [C.c_int64]
    L.pitch.restype, L.pitch.argtypes = C.c_int64, [C.c_int64, C.c_int]
    for rows, cols in [(1, 1), (128, 128), (129, 33), (300, 700)]:
        atoms, up = L.wide(cols) // 128, -(-rows // 128) * 128
        assert L.pitch(cols, 8) == atoms * 128 and L.pitch(cols, 4) == atoms * 64
        seen = sorted(L.at(r, b, atoms) for r in range(up) for b in range(4 * atoms))
        assert seen == list(range(up * 4 * atoms)) and len(seen) == tcg.lib().tcg_mx_scale_bytes(rows, cols)
    # four rows 32 apart, and a row's four blocks, are neighbours
    assert [L.at(5 + 32 * i, 4, 9) for i in range(4)] == [512 + 80 + 4 * i for i in range(4)]
    assert [L.at(5, 4 + i, 9) for i in range(4)] == [512 + 80 + i for i in range(4)]
    assert L.at((1 << 30) - 1, (1 << 19) - 1, 1 << 17) == (1 << 49) - 1
