"""Host side of the language-model operators: the rotary plan (tcg_rope_*), also
from GGUF metadata, the refusals of every entry point, and the index arithmetic
of the 8-bit key/value cache (csrc/kv8_index.h, compiled here as plain C):
whatever lengths and pages a step holds, nothing outside the buffers is named.
No GPU."""
import ctypes as C
import itertools
import math
import os
import random
import subprocess
import threading

import numpy as np
import pytest

import tcg
import tcg_gguf as G

PKG = os.path.dirname(tcg.LIB_PATH)
CSRC = os.path.join(os.path.dirname(PKG), "csrc")


def _plan(d=128, n_rot=128, layout=tcg.ROPE_HALF, base=10000.0):
    r = tcg.Rope()
    tcg.check(tcg.lib().tcg_rope_init(C.byref(r), d, n_rot, layout, base))
    return r


def _turns(r):
    return np.array(r.turns[:r.n_rot // 2])


def _freq(n_rot, base):
    return base ** (-2.0 * np.arange(n_rot // 2) / n_rot) / (2 * math.pi)


# ------------------------------------------------------------------ rotary plan

@pytest.mark.parametrize("d,n_rot,base", [(128, 128, 10000.0), (80, 20, 500000.0), (256, 256, 1e6), (2, 2, 0.5)])
def test_plan(d, n_rot, base):
    r = _plan(d, n_rot, tcg.ROPE_INTERLEAVED, base)
    # pow and one division in 64 bits
    np.testing.assert_allclose(_turns(r), _freq(n_rot, base), rtol=1e-14)
    assert r.mscale == 1.0 and r.head_dim == d and not any(r.turns[n_rot // 2:])


def test_context_rules():
    L = tcg.lib()
    f = _freq(128, 10000.0)
    r = _plan()
    assert L.tcg_rope_scale_linear(C.byref(r), 4.0)
    np.testing.assert_allclose(_turns(r), f / 4, rtol=1e-14)

    # by bands: turns over the context decide
    r = _plan()
    assert L.tcg_rope_scale_bands(C.byref(r), 8.0, 8192, 1.0, 4.0)
    n = 8192 * f
    want = np.where(n >= 4, f, np.where(n <= 1, f / 8, f * (n - 1) / 3 + f / 8 * (4 - n) / 3))
    np.testing.assert_allclose(_turns(r), want, rtol=1e-13)
    assert (n > 4).any() and (n < 1).any() and ((n > 1) & (n < 4)).any()

    # by pair index between the pairs of 32 turns and of one turn
    r = _plan()
    assert L.tcg_rope_scale_yarn(C.byref(r), 32.0, 4096, 32.0, 1.0, 0.0)
    def pair(turns): return 128 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
    lo, hi = math.floor(pair(32)), math.ceil(pair(1))
    ramp = np.clip((np.arange(64) - lo) / (hi - lo), 0, 1)
    np.testing.assert_allclose(_turns(r), f * (1 - ramp) + f / 32 * ramp, rtol=1e-13)
    assert r.mscale == pytest.approx(0.1 * math.log(32) + 1, rel=2.0 ** -23)
    assert L.tcg_rope_scale_yarn(C.byref(_plan()), 0.5, 4096, 32.0, 1.0, 0.0)
    r = _plan()
    assert L.tcg_rope_scale_yarn(C.byref(r), 32.0, 4096, 32.0, 1.0, 1.25) and r.mscale == 1.25

    r = _plan()
    g = np.linspace(1, 9, 64).astype(np.float32)
    assert L.tcg_rope_scale_factors(C.byref(r), g.ctypes.data, 64)
    np.testing.assert_allclose(_turns(r), f / g.astype(np.float64), rtol=1e-14)


def test_plan_refusals():
    L, r = tcg.lib(), tcg.Rope()
    for d, n, lay, base in [(0, 2, 0, 1e4), (127, 2, 0, 1e4), (258, 2, 0, 1e4), (64, 0, 0, 1e4), (64, 63, 0, 1e4),
                            (64, 66, 0, 1e4), (64, 64, 2, 1e4), (64, 64, 0, 0.0), (64, 64, 0, -1.0),
                            (64, 64, 0, float("nan")), (64, 64, 0, float("inf"))]:
        assert not L.tcg_rope_init(C.byref(r), d, n, lay, base) and "tcg_rope_init" in tcg.err()
    assert not L.tcg_rope_init(None, 64, 64, 0, 1e4)
    empty = tcg.Rope()
    assert not L.tcg_rope_scale_linear(C.byref(empty), 2.0) and "not initialised" in tcg.err()
    p = _plan()
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert not L.tcg_rope_scale_linear(C.byref(p), bad)
        assert not L.tcg_rope_scale_yarn(C.byref(p), bad, 4096, 32.0, 1.0, 0.0)
        assert not L.tcg_rope_scale_bands(C.byref(p), bad, 4096, 1.0, 4.0)
    assert not L.tcg_rope_scale_yarn(C.byref(p), 2.0, 0, 32.0, 1.0, 0.0)
    assert not L.tcg_rope_scale_yarn(C.byref(p), 2.0, 4096, 1.0, 32.0, 0.0)
    assert not L.tcg_rope_scale_yarn(C.byref(p), 2.0, 4096, 32.0, 1.0, -1.0)
    assert not L.tcg_rope_scale_yarn(C.byref(_plan(base=1.0)), 2.0, 4096, 32.0, 1.0, 0.0)
    assert not L.tcg_rope_scale_bands(C.byref(p), 2.0, 4096, 4.0, 4.0)
    g = np.ones(64, np.float32)
    assert not L.tcg_rope_scale_factors(C.byref(p), g.ctypes.data, 63)
    assert not L.tcg_rope_scale_factors(C.byref(p), None, 64)
    g[5] = 0
    assert not L.tcg_rope_scale_factors(C.byref(p), g.ctypes.data, 64)
    np.testing.assert_array_equal(_turns(p), _turns(_plan()))          # a refused call changes nothing


def _from_gguf(tmp_path, kvs, tensors=()):
    path = str(tmp_path / "m.gguf")
    G.write_gguf(path, kvs, list(tensors))
    L = tcg.lib()
    a, g, r = L.arena_create(1 << 20, b"t"), tcg.Gguf(), tcg.Rope()
    assert L.gguf_open(C.byref(g), path.encode(), C.byref(a)), g.err
    try:
        return L.tcg_rope_from_gguf(C.byref(r), C.byref(g), tcg.ROPE_HALF), r
    finally:
        L.gguf_close(C.byref(g))
        L.arena_destroy(C.byref(a))


def test_plan_from_gguf(tmp_path):
    base = {"general.architecture": "lm", "lm.embedding_length": 512, "lm.attention.head_count": 8}
    ok, r = _from_gguf(tmp_path, base)
    assert ok and (r.head_dim, r.n_rot, r.layout, r.mscale) == (64, 64, tcg.ROPE_HALF, 1.0)
    np.testing.assert_allclose(_turns(r), _freq(64, 10000.0), rtol=1e-14)

    f = np.linspace(1, 4, 16).astype(np.float32)
    ok, r = _from_gguf(tmp_path, {**base, "lm.attention.key_length": 96, "lm.rope.dimension_count": 32,
                                  "lm.rope.freq_base": 500000.0, "lm.rope.scaling.type": "linear",
                                  "lm.rope.scaling.factor": 2.0}, [("rope_freqs.weight", f, G.F32, (16,))])
    assert ok and (r.head_dim, r.n_rot) == (96, 32)
    np.testing.assert_allclose(_turns(r), _freq(32, 500000.0) / f / 2, rtol=1e-14)

    ok, r = _from_gguf(tmp_path, {**base, "lm.rope.scaling.type": "yarn", "lm.rope.scaling.factor": 4.0,
                                  "lm.rope.scaling.original_context_length": 2048, "lm.rope.scaling.attn_factor": 0.5})
    want = _plan(64, 64)
    tcg.check(tcg.lib().tcg_rope_scale_yarn(C.byref(want), 4.0, 2048, 32.0, 1.0, 0.0))
    assert ok and r.mscale == np.float32(want.mscale) * np.float32(0.5)
    np.testing.assert_array_equal(_turns(r), _turns(want))

    for bad in ({"lm.embedding_length": 512}, {"general.architecture": "lm"},
                {**base, "lm.rope.scaling.type": "other"},
                {**base, "lm.rope.scaling.type": "linear"}, {**base, "lm.rope.dimension_count": 66},
                {**base, "lm.attention.key_length": 512}):
        ok, r = _from_gguf(tmp_path, bad)
        assert not ok and "tcg_rope" in tcg.err()
        assert r.n_rot == 0                                             # untouched
    assert not _from_gguf(tmp_path, base, [("rope_freqs.weight", f, G.F32, (16,))])[0]      # 16 factors for 32 pairs


def test_plan_from_gguf_passes_nothing_over(tmp_path):
    """What changes the angles or the magnitude is followed or refused; what changes nothing is taken."""
    base = {"general.architecture": "lm", "lm.embedding_length": 512, "lm.attention.head_count": 8}
    yarn = {**base, "lm.rope.scaling.type": "yarn", "lm.rope.scaling.factor": 4.0,
            "lm.rope.scaling.original_context_length": 2048}
    f = np.full(32, 2.0, np.float32)
    for kvs in ({"lm.rope.scale_linear": 4.0}, {"lm.rope.freq_base_swa": 1e5}, {"lm.rope.dimension_sections": [16.0, 24.0]},
                {"lm.rope.scaling.factor": 4.0}, {"lm.rope.scaling.attn_factor": 1.2}, {"lm.rope.scaling.alpha": 2.0},
                {"lm.rope.scaling.type": "linear", "lm.rope.scaling.factor": 2.0, "lm.rope.scaling.attn_factor": 0.5},
                {"lm.rope.scaling.type": 1}, {"lm.rope.freq_base": "10000"}, {"lm.rope.scaling.yarn_log_multiplier": 0.1}):
        ok, r = _from_gguf(tmp_path, {**base, **kvs})
        assert not ok and "tcg_rope_from_gguf" in tcg.err() and r.n_rot == 0, kvs
    for kvs in ({"lm.rope.scaling.yarn_log_multiplier": 0.1}, {"lm.rope.scaling.yarn_beta_fast": 16.0},
                {"lm.rope.scaling.yarn_beta_slow": 2.0}, {"lm.rope.scaling.yarn_ext_factor": 0.0},
                {"lm.rope.scaling.yarn_attn_factor": 2.0}):
        assert not _from_gguf(tmp_path, {**yarn, **kvs})[0], kvs
    for name in ("rope_factors_long.weight", "rope_factors_short.weight", "blk.0.rope_freqs.weight"):
        ok, r = _from_gguf(tmp_path, base, [(name, f, G.F32, (32,))])
        assert not ok and name in tcg.err() and r.n_rot == 0

    plain, scaled = (_from_gguf(tmp_path, x)[1] for x in (base, yarn))
    for kvs in ({"lm.rope.scale_linear": 1.0}, {"lm.rope.scaling.finetuned": True}, {"lm.rope.scaling.factor": 1.0},
                {"lm.rope.scaling.attn_factor": 1.0}, {"lm.rope.scaling.type": "none", "lm.rope.scaling.factor": 4.0},
                {"lm.rope.freq_base": 10000}, {"other.rope.scale_linear": 4.0}, {"lm.ropes": 1}):
        ok, r = _from_gguf(tmp_path, {**base, **kvs})
        assert ok and bytes(r) == bytes(plain), kvs
    for kvs in ({"lm.rope.scaling.yarn_beta_fast": 32.0, "lm.rope.scaling.yarn_beta_slow": 1.0},
                {"lm.rope.scaling.yarn_ext_factor": 1.0, "lm.rope.scaling.yarn_log_multiplier": 0.0}):
        ok, r = _from_gguf(tmp_path, {**yarn, **kvs})
        assert ok and bytes(r) == bytes(scaled), kvs
    ok, r = _from_gguf(tmp_path, {**base, "lm.rope.freq_base": 500000})  # a whole number is a number
    assert ok and r.base == 500000.0


# ------------------------------------------------------------------ refusals

P = 1 << 20          # an aligned address that is never dereferenced: every call here is refused before any launch


def _cache(**kw):
    return tcg.Kv8(*(kw.get(n, d) for n, d in (("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("n_pages", 4),
                                               ("n_kv_head", 2), ("head_dim", 64))))


def _step(**kw):
    return tcg.Kv8Step(*(kw.get(n, d) for n, d in (("tok_start", P), ("kv_len", P), ("table", P), ("table_ld", 2),
                                                   ("n_seq", 1), ("n_tok", 3), ("max_new", 3), ("max_kv", 100))))


def _refused(fn, *args):
    assert fn(*args) is False
    msg = tcg.err()
    assert msg and "tcg_init" not in msg, msg
    return msg


CACHES = [dict(head_dim=0), dict(head_dim=24), dict(head_dim=144), dict(n_kv_head=0), dict(n_kv_head=65536), dict(n_pages=0),
          dict(n_pages=1 << 30), dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(k=P + 8), dict(v=P + 4),
          dict(k_scale=P + 2)]
STEPS = [dict(n_seq=-1), dict(n_seq=65536), dict(n_tok=-1), dict(max_new=-1), dict(max_kv=-1), dict(table_ld=-1),
         dict(tok_start=0), dict(kv_len=0), dict(table=0), dict(kv_len=P + 1)]


@pytest.mark.parametrize("kw", CACHES + STEPS, ids=str)
def test_cache_and_step_refusals(kw):
    L = tcg.lib()
    cache = kw.keys() <= {"k", "v", "k_scale", "v_scale", "n_pages", "n_kv_head", "head_dim"}
    c, s = C.byref(_cache(**kw) if cache else _cache()), C.byref(_step() if cache else _step(**kw))
    for fn in (L.tcg_kv8_append, ):
        assert "tcg_kv8_append" in _refused(fn, c, s, P, P, 128, 128, 0)
    _refused(L.tcg_kv8_read, P, P, c, s, 128, 128, 0)
    _refused(L.tcg_kv8_attention, P, P, c, s, 4, 256, 256, 0.125, True, 0, 0)


def test_argument_refusals():
    L = tcg.lib()
    c, s, r = C.byref(_cache()), C.byref(_step()), C.byref(_plan(64, 64))
    for args in [(None, s, P, P, 128, 128, 0), (c, None, P, P, 128, 128, 0), (c, s, None, P, 128, 128, 0),
                 (c, s, P, None, 128, 128, 0), (c, s, P + 2, P, 128, 128, 0), (c, s, P, P, 127, 128, 0),
                 (c, s, P, P, 128, 0, 0), (c, s, P, P, 128, 128, 12), (c, s, P, P, -128, 128, 0)]:
        _refused(L.tcg_kv8_append, *args)
    for n_head, ldo, ldq, scale, causal, win, t in [
            (3, 256, 256, 1.0, True, 0, 0), (0, 256, 256, 1.0, True, 0, 0), (4, 255, 256, 1.0, True, 0, 0),
            (4, 256, 255, 1.0, True, 0, 0), (4, 256, 256, 0.0, True, 0, 0), (4, 256, 256, -1.0, True, 0, 0),
            (4, 256, 256, float("nan"), True, 0, 0), (4, 256, 256, float("inf"), True, 0, 0),
            (4, 256, 256, 1.0, True, -1, 0), (4, 256, 256, 1.0, False, 5, 0), (4, 256, 256, 1.0, True, 0, 2),
            (2 * 4097, 1 << 20, 1 << 20, 1.0, True, 0, 0)]:
        _refused(L.tcg_kv8_attention, P, P, c, s, n_head, ldo, ldq, scale, causal, win, t)
    _refused(L.tcg_kv8_attention, None, P, c, s, 4, 256, 256, 1.0, True, 0, 0)
    _refused(L.tcg_kv8_attention, P + 1, P, c, s, 4, 256, 256, 1.0, True, 0, 1)
    many = C.byref(_step(n_tok=1 << 30, max_new=1 << 30))
    _refused(L.tcg_kv8_attention, P, P, c, many, 4, 256, 256, 1.0, True, 0, 0)

    for args in [(P, P, P, r, -1, 2, 128, 128, 0), (P, P, None, r, 3, 2, 128, 128, 0), (None, P, P, r, 3, 2, 128, 128, 0),
                 (P, None, P, r, 3, 2, 128, 128, 0), (P, P, P, r, 3, -2, 128, 128, 0), (P, P, P, r, 3, 2, 127, 128, 0),
                 (P, P, P, r, 3, 2, 128, 127, 0), (P, P, P, r, 3, 2, 128, 128, 12), (P + 1, P, P, r, 3, 2, 128, 128, 1),
                 (P, P, P, None, 3, 2, 128, 128, 0), (P, P, P, C.byref(tcg.Rope()), 3, 2, 128, 128, 0)]:
        _refused(L.tcg_rope, *args)
    for eps, qw, nh, nk in [(-1.0, P, 2, 1), (float("nan"), P, 2, 1), (1e-6, None, 2, 1), (1e-6, P + 2, 2, 1),
                            (1e-6, P, -1, 1), (1e-6, P, 2, -1)]:
        _refused(L.tcg_qk_norm_rope, P, P, P, P, qw, P, eps, P, r, 3, nh, nk, 128, 64, 128, 64, 0)


def test_without_a_device():
    L, got = tcg.lib(), {}
    c, s, r = C.byref(_cache()), C.byref(_step()), C.byref(_plan(64, 64))

    def body():                                                          # a fresh thread has no device context
        got["append"] = (L.tcg_kv8_append(c, s, P, P, 128, 128, 0), tcg.err())
        got["read"] = (L.tcg_kv8_read(P, P, c, s, 128, 128, 0), tcg.err())
        got["attention"] = (L.tcg_kv8_attention(P, P, c, s, 4, 256, 256, 0.125, True, 0, 0), tcg.err())
        got["rope"] = (L.tcg_rope(P, P, P, r, 3, 2, 128, 128, 0), tcg.err())
        got["norm"] = (L.tcg_qk_norm_rope(P, P, P, P, P, P, 1e-6, P, r, 3, 2, 1, 128, 64, 128, 64, 0), tcg.err())

    t = threading.Thread(target=body)
    t.start()
    t.join()
    assert len(got) == 5
    for ok, msg in got.values():
        assert ok is False and "tcg_init" in msg


# ------------------------------------------------------------------ index arithmetic

@pytest.fixture(scope="module")
def index(tmp_path_factory):
    """csrc/kv8_index.h as a shared library: the functions the kernels use, compiled for the host."""
    d = tmp_path_factory.mktemp("kv8")
    src = d / "index.c"
    src.write_text('''#include "kv8_index.h"
bool seq_ok(int a, int b, int kv, int n_tok, int max_new, int ld, int *o) {
    kv8_seq_t q; const bool ok = kv8_seq_ok(a, b, kv, n_tok, max_new, ld, &q); o[0] = q.row0; o[1] = q.n; o[2] = q.kv; return ok; }
bool page_ok(int p, int n) { return kv8_page_ok(p, n); }
int reach(int n) { return kv8_reach(n); }
bool place(int row0, int n, int kv, int j, int *o) {
    kv8_seq_t q = { row0, n, kv }; kv8_place_t a; const bool ok = kv8_place(&q, j, &a);
    if (ok) { o[0] = a.index; o[1] = a.lo; o[2] = a.hi; o[3] = a.row; } return ok; }
int hi(int n, int kv, int tok, int causal) { kv8_seq_t q = { 0, n, kv }; return kv8_hi(&q, tok, causal); }
int lo(int n, int kv, int tok, int window) { kv8_seq_t q = { 0, n, kv }; return kv8_lo(&q, tok, window); }
int tiles(int n, int kv, int a, int z, int causal, int window, int rank, int ranks, int part, int parts, int *t0) {
    kv8_seq_t q = { 0, n, kv }; return kv8_tiles(&q, a, z, causal, window, rank, ranks, part, parts, t0); }
''')
    so = d / "index.so"
    subprocess.run(["gcc", "-std=c11", "-O2", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-o", str(so), str(src)],
                   check=True)
    return C.CDLL(str(so))


def test_bad_lengths_and_pages(index):
    o = (C.c_int * 3)()
    index.seq_ok.restype = index.page_ok.restype = index.place.restype = C.c_bool
    big = 2 ** 31 - 1
    for a, b, kv, n_tok, max_new, ld in itertools.product((-1, 0, 5, big), (-7, 0, 5, 9, big), (-1, 0, 3, 64, 65, big),
                                                          (0, 9), (0, 4, 9), (0, 1, 2, big)):
        ok = index.seq_ok(a, b, kv, n_tok, max_new, ld, o)
        good = 0 <= a <= b <= n_tok and b - a <= max_new and b - a <= kv <= ld * 64
        assert ok == good
        assert not ok or list(o) == [a, b - a, kv]
        assert ok or o[1] == 0                                           # a refused sequence has no rows
    for p, n in itertools.product((-2 ** 31, -1, 0, 3, 4, big), (1, 4)):
        assert index.page_ok(p, n) == (0 <= p < n)


def test_places_cover_the_new_rows_once(index):
    index.place.restype = C.c_bool
    rnd = random.Random(3)
    for _ in range(4000):
        n = rnd.choice([1, 2, 63, 64, 65, 66, 127, 128, 129, rnd.randint(1, 700)])
        kv = n + rnd.choice([0, 1, 62, 63, 64, rnd.randint(0, 5000), 2 ** 30])
        row0, o, seen = rnd.randint(0, 50), (C.c_int * 4)(), []
        for j in range(index.reach(n)):
            if not index.place(row0, n, kv, j, o):
                continue
            page, lo, hi, row = o
            assert 0 <= lo < hi <= 64 and 0 <= page <= (kv - 1) // 64
            seen += [(page * 64 + s, row + s - lo) for s in range(lo, hi)]
        assert seen == [(kv - n + i, row0 + i) for i in range(n)]
        assert not index.place(row0, n, kv, index.reach(n), o)           # nothing lies behind the reach
    assert not index.place(0, 0, 100, 0, (C.c_int * 4)())


def test_tiles_cover_the_visible_keys_once(index):
    rnd = random.Random(5)
    for _ in range(1500):
        n = rnd.choice([1, 2, 5, 64, rnd.randint(1, 300)])
        kv = n + rnd.choice([0, 1, 63, 64, rnd.randint(0, 3000)])
        causal = rnd.random() < 0.7
        window = rnd.choice([0, 1, 64, rnd.randint(1, 3500)]) if causal else 0
        a = rnd.randrange(n)
        z = min(n - 1, a + rnd.randint(0, 40))
        ranks, parts, t0, seen = rnd.choice([1, 2, 4, 8]), rnd.choice([1, 8]), C.c_int(), []
        for rank, part in itertools.product(range(ranks), range(parts)):
            cnt = index.tiles(n, kv, a, z, causal, window, rank, ranks, part, parts, C.byref(t0))
            seen += [t0.value + i * parts for i in range(cnt)]
        need = set()
        for tok in (a, z):                                               # the rows between see no key outside these two's
            pos = kv - n + tok
            lo = max(0, pos - window + 1) if window else 0
            hi = pos if causal else kv - 1
            assert (index.lo(n, kv, tok, window), index.hi(n, kv, tok, causal)) == (lo, hi)
            need |= {lo // 64, hi // 64}
        assert sorted(seen) == list(range(min(need), max(need) + 1))
        assert max(seen) <= (kv - 1) // 64
