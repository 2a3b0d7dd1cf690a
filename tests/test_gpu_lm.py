"""Language-model operators on the GPU against their formulas in 64 bits:
rotary positions, head norms with the rotation, the 8-bit key/value cache
(bytes compared exactly) and the attention over it, and a run of them together.

Tolerances are sums of the roundings each kernel makes, written beside them;
u = 2^-24 is half a step of fp32, eps(t) / 2 that of the output type.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import tcg

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, tcg.F32), "f16": (torch.float16, tcg.F16), "bf16": (torch.bfloat16, tcg.BF16)}
U = 2.0 ** -24
PAGE = tcg.KV8_PAGE


def half_step(dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture()
def lib(gpu):
    """The library on torch's legacy default stream's device, with a stream of its own: tests synchronise around calls."""
    L = tcg.lib()
    tcg.check(L.tcg_clear_device_error())
    yield L
    torch.cuda.synchronize()
    assert L.tcg_device_error() == 0


def call(fn, *args):
    torch.cuda.synchronize()
    tcg.check(fn(*args))
    torch.cuda.synchronize()


def randn(gen, *shape, dtype=torch.float32, spread=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * spread).to(dtype).cuda()


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ rotary positions and head norms

def plan(d, n_rot, half, base=10000.0):
    r = tcg.Rope()
    tcg.check(tcg.lib().tcg_rope_init(C.byref(r), d, n_rot, int(half), base))
    return r


def rotated(x, pos, r):
    """x [n, heads, d] in 64 bits, rotated; and the sum of the magnitudes that each value is made of."""
    n_rot, out = r.n_rot, x.clone()
    mag = x.abs()
    t = pos.double()[:, None] * torch.tensor(list(r.turns[:n_rot // 2]), dtype=torch.float64, device=x.device)
    a = (t - t.round()) * (2 * math.pi)
    c, s = (torch.cos(a) * r.mscale)[:, None], (torch.sin(a) * r.mscale)[:, None]
    i = torch.arange(n_rot // 2, device=x.device)
    lo, hi = (i, i + n_rot // 2) if r.layout == tcg.ROPE_HALF else (2 * i, 2 * i + 1)
    p, q = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = p * c - q * s, p * s + q * c
    mag[..., lo] = mag[..., hi] = (p.abs() + q.abs()) * abs(r.mscale)
    return out, mag


# fp32 fraction of a turn: 2^-25 of [-1, 1], pi times that in the angle (1.6 u); sincospi 2 ulp (2 u); times mscale 1 u;
# the two products' rounding and the sum's 2 u: under 7 u of |a| + |b|. The norm adds a sum of at most 16 squares a lane
# and 5 adds over lanes, halved by the root (10.5 u), the division and eps 2 u / 2, rsqrtf 2 ulp (4 u), two products 2 u: 18 u.
ROPE_U, NORM_U = 7, 18

ROPES = [  # d, n_rot, half, heads, tokens, type
    (128, 128, True, 5, 1, "f32"), (128, 128, False, 40, 1, "f32"), (128, 64, True, 3, 129, "bf16"),
    (64, 64, False, 8, 33, "f16"), (80, 80, True, 7, 17, "bf16"), (80, 40, True, 7, 17, "f16"), (96, 96, False, 2, 600, "f32"),
    (256, 256, True, 2, 9, "f16"), (256, 128, False, 3, 70, "f32"), (2, 2, True, 3, 5, "f32"), (6, 4, False, 1, 2, "bf16"),
    (34, 22, True, 5, 11, "f32"), (258 - 4, 250, True, 2, 3, "bf16"), (32, 16, True, 1, 4000, "bf16"), (128, 2, False, 4, 3, "f16"),
]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("d,n_rot,half,heads,n,t", ROPES)
def test_rope_and_norm(lib, d, n_rot, half, heads, n, t, norm):
    dt, code = TYPES[t]
    g, r = gen(d + n), plan(d, n_rot, half)
    tcg.check(lib.tcg_rope_scale_yarn(C.byref(r), 4.0, 4096, 32.0, 1.0, 1.25))
    x = randn(g, n, heads, d, dtype=dt, spread=3.0)
    pos = torch.randint(-5, 1 << 20, (n,), generator=g, dtype=torch.int32).cuda()
    kv = heads // 2 if norm else 0
    wq, wk = randn(g, d) + 1, randn(g, d) + 1
    y = torch.full_like(x, float("nan"))
    if norm:
        at = (heads - kv) * d * x.element_size()
        call(lib.tcg_qk_norm_rope, y.data_ptr(), y.data_ptr() + at, x.data_ptr(), x.data_ptr() + at, wq.data_ptr(),
             wk.data_ptr(), 1e-5, pos.data_ptr(), C.byref(r), n, heads - kv, kv, heads * d, heads * d, heads * d, heads * d, code)
    else:
        call(lib.tcg_rope, y.data_ptr(), x.data_ptr(), pos.data_ptr(), C.byref(r), n, heads, heads * d, heads * d, code)
    z = x.double()
    if norm:
        z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + float(np.float32(1e-5)))
        z[:, :heads - kv] *= wq.double()
        z[:, heads - kv:] *= wk.double()
    want, mag = rotated(z, pos, r)
    tol = mag * (ROPE_U + (NORM_U if norm else 0)) * U + want.abs() * (half_step(dt) if t != "f32" else 0) + 1e-30
    tol += 2.0 ** -24 if t == "f16" else 0                               # half a step of fp16's subnormals is 2^-25
    assert ((y.double() - want).abs() <= tol).all()
    # in place, over rows with a stride, gives the same bits and leaves what lies between the rows
    if not norm:
        wide = torch.full((n, heads * d + 3), 7.0, dtype=dt, device="cuda")
        wide[:, :heads * d] = x.view(n, -1)
        call(lib.tcg_rope, wide.data_ptr(), wide.data_ptr(), pos.data_ptr(), C.byref(r), n, heads, heads * d + 3,
             heads * d + 3, code)
        assert torch.equal(wide[:, :heads * d], y.view(n, -1)) and (wide[:, heads * d:] == 7).all()


def test_rope_far_positions_and_plain_halves(lib):
    """The largest position: the fraction of a revolution is exact to 2^31 * 0.16 * 2^-53 turns (2e-7 radians, 4 u)."""
    r = plan(64, 64, True)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32).cuda()
    x = randn(gen(1), 3, 2, 64)
    y = torch.empty_like(x)
    call(lib.tcg_rope, y.data_ptr(), x.data_ptr(), pos.data_ptr(), C.byref(r), 3, 2, 128, 128, tcg.F32)
    want, mag = rotated(x.double(), pos, r)
    assert ((y.double() - want).abs() <= mag * (ROPE_U + 4) * U).all()
    assert torch.equal(y[2], x[2])                                       # position 0 turns nothing


def test_norm_of_one_side_and_none(lib):
    r = plan(64, 64, False)
    x, w = randn(gen(2), 4, 3, 64), randn(gen(3), 64)
    pos = torch.arange(4, dtype=torch.int32).cuda()
    both = torch.zeros_like(x)
    call(lib.tcg_qk_norm_rope, None, both.data_ptr(), None, x.data_ptr(), None, w.data_ptr(), 1e-6, pos.data_ptr(),
         C.byref(r), 4, 0, 3, 0, 192, 0, 192, tcg.F32)
    other = torch.zeros_like(x)
    call(lib.tcg_qk_norm_rope, other.data_ptr(), None, x.data_ptr(), None, w.data_ptr(), None, 1e-6, pos.data_ptr(),
         C.byref(r), 4, 3, 0, 192, 0, 192, 0, tcg.F32)
    assert torch.equal(both, other) and both.abs().sum() > 0
    call(lib.tcg_rope, both.data_ptr(), x.data_ptr(), pos.data_ptr(), C.byref(r), 0, 3, 192, 192, tcg.F32)
    call(lib.tcg_rope, both.data_ptr(), x.data_ptr(), pos.data_ptr(), C.byref(r), 4, 0, 192, 192, tcg.F32)
    assert torch.equal(both, other)                                      # no tokens, no heads: nothing written


# ------------------------------------------------------------------ the cache

class Pool:
    """A page pool, sequences with cached tokens in random pages, and garbage wherever no token lies."""

    def __init__(self, g, n_kv, d, kv, spare=3):
        self.n_kv, self.d, self.kv = n_kv, d, list(kv)
        pages = [-(-k // PAGE) for k in kv]
        self.n = sum(pages) + spare
        self.k = torch.randint(-127, 128, (self.n, n_kv, PAGE, d), generator=g, dtype=torch.int8).cuda()
        self.v = torch.randint(-127, 128, (self.n, n_kv, d, PAGE), generator=g, dtype=torch.int8).cuda()
        self.ks, self.vs = (torch.rand((self.n, n_kv), generator=g).cuda() * 0.03 + 0.01 for _ in range(2))
        order = torch.randperm(self.n, generator=g)
        self.ld = max(pages + [1]) + 1
        self.table = torch.full((len(kv), self.ld), -7, dtype=torch.int32)
        at = 0
        for b, p in enumerate(pages):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.free = order[at:].tolist()
        self.ks[self.free], self.vs[self.free] = float("nan"), float("inf")
        self.table = self.table.cuda()

    def cache(self):
        return tcg.Kv8(self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), self.n, self.n_kv, self.d)

    def step(self, new, kv=None, pad=0, max_new=None, max_kv=None):
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.keep = [torch.from_numpy(start).cuda(), torch.tensor(kv or self.kv, dtype=torch.int32).cuda()]
        return tcg.Kv8Step(self.keep[0].data_ptr(), self.keep[1].data_ptr(), self.table.data_ptr(), self.ld, len(new),
                           int(start[-1]) + pad, max(new) if max_new is None else max_new,
                           max(self.kv) if max_kv is None else max_kv)

    def values(self, b, n):
        """K and V of the first n tokens of sequence b: [heads, n, d] in 64 bits."""
        pages = self.table[b, :-(-n // PAGE)].long()
        k = (self.k[pages].double() * self.ks[pages].double()[..., None, None]).permute(1, 0, 2, 3)
        v = (self.v[pages].double() * self.vs[pages].double()[..., None, None]).permute(1, 0, 3, 2)
        return k.reshape(self.n_kv, -1, self.d)[:, :n], v.reshape(self.n_kv, -1, self.d)[:, :n]


def appended(codes, scale, page, lo, rows, dims_first):
    """The format's definition for one page, each step rounded to fp32 on the CPU: rows [n, heads, d] into slots lo..."""
    rows = rows.float().cpu().numpy()
    rows = np.clip(np.where(np.isnan(rows), np.float32(0), rows), -np.finfo(np.float32).max, np.finfo(np.float32).max)
    have = codes[page].cpu().numpy()
    if dims_first:
        have = have.transpose(0, 2, 1)
    have = have.copy()
    was = scale[page].cpu().numpy() if lo else np.zeros(have.shape[0], np.float32)
    now = np.maximum(was, np.abs(rows).max(axis=(0, 2)) / np.float32(127))
    for h in range(have.shape[0]):
        if lo and now[h] > was[h]:
            ratio = np.float32(was[h] / now[h])
            have[h, :lo] = np.rint(have[h, :lo].astype(np.float32) * ratio)
        q = np.rint(rows[:, h] / now[h]) if now[h] > 0 else np.zeros_like(rows[:, h])
        have[h, lo:lo + rows.shape[0]] = np.clip(q, -127, 127)
    return (have.transpose(0, 2, 1) if dims_first else have), now


APPENDS = [  # heads, d, [(new, kv)], type, padding of the stride
    (2, 64, [(1, 1)], "f32", 0), (1, 128, [(1, 64), (1, 65), (1, 100), (0, 70), (1, 128)], "f32", 0),
    (3, 16, [(64, 64), (65, 65), (63, 127), (128, 200), (2, 65)], "f16", 0), (2, 80, [(5, 5), (70, 133)], "bf16", 0),
    (8, 128, [(300, 300), (1, 640), (129, 1000)], "f32", 4), (1, 96, [(200, 263)], "f16", 1), (2, 112, [(9, 64), (7, 71)], "bf16", 2),
    (1, 48, [(3, 4)], "f32", 3), (4, 32, [(7, 9), (8, 72)], "f16", 4),
]


@pytest.mark.parametrize("heads,d,seqs,t,extra", APPENDS)
def test_append_and_read(lib, heads, d, seqs, t, extra):
    dt, code = TYPES[t]
    g = gen(heads * d + len(seqs))
    new, kv = [a for a, _ in seqs], [b for _, b in seqs]
    pool, n = Pool(g, heads, d, kv), sum(new)
    ld = heads * d + extra
    rows = [randn(g, n + 2, ld, dtype=dt, spread=s) for s in (1.0, 4.0)]  # V grows its pages' scales, K mostly not
    rows[0][0] = 0
    if n > 2:
        rows[1][1, :d] = 1e-30 if t != "f16" else 0
    before = [x.clone() for x in (pool.k, pool.v, pool.ks, pool.vs)]
    s = pool.step(new, pad=2)
    call(lib.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), rows[0].data_ptr(), rows[1].data_ptr(), ld, ld, code)
    want = [x.cpu().clone() for x in before]
    at = 0
    for b, (a, z) in enumerate(seqs):
        pos = z - a
        while pos < z:
            end = min(z, (pos // PAGE + 1) * PAGE)
            page = int(pool.table[b, pos // PAGE])
            for i in range(2):
                x = rows[i][at:at + end - pos, :heads * d].reshape(-1, heads, d)
                codes, now = appended(before[i], before[2 + i], page, pos % PAGE, x, i == 1)
                want[i][page], want[2 + i][page] = torch.from_numpy(codes), torch.from_numpy(now)
            at += end - pos
            pos = end
    for got, w in zip((pool.k, pool.v, pool.ks, pool.vs), want):
        # every byte of the pool: the step's slots, the older ones, and what must stay as it was
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=9e9), torch.nan_to_num(w.float(), nan=9e9))
    for t2, (dt2, code2) in TYPES.items():
        out = [torch.full((n + 2, ld), 7.0, dtype=dt2, device="cuda") for _ in range(2)]
        call(lib.tcg_kv8_read, out[0].data_ptr(), out[1].data_ptr(), C.byref(pool.cache()), C.byref(s), ld, ld, code2)
        at = 0
        for b, (a, z) in enumerate(seqs):
            for o, c, sc, last in ((out[0], pool.k, pool.ks, False), (out[1], pool.v, pool.vs, True)):
                pages = pool.table[b, :-(-z // PAGE)].long()
                x = (c[pages].transpose(2, 3) if last else c[pages]).float() * sc[pages][..., None, None]
                x = x.permute(0, 2, 1, 3).reshape(-1, heads * d)[z - a:z].to(dt2)
                assert torch.equal(o[at:at + a, :heads * d], x)
            at += a
        assert all((o[:, heads * d:] == 7).all() and (o[n:] == 7).all() for o in out)


def test_append_of_zeros_infinities_and_nan(lib):
    pool = Pool(gen(4), 1, 16, [5, 66])
    x = torch.zeros((7, 16), device="cuda")
    y = randn(gen(5), 7, 16)
    y[1, 3], y[2, 4], y[6, 0] = float("nan"), -float("inf"), float("nan")
    s = pool.step([5, 2])
    call(lib.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), x.data_ptr(), y.data_ptr(), 16, 16, tcg.F32)
    p, q = int(pool.table[0, 0]), int(pool.table[1, 1])
    assert pool.ks[p, 0] == 0 and pool.ks[q, 0] == 0 and (pool.k[p, 0, :5] == 0).all()
    big = np.float32(np.finfo(np.float32).max) / np.float32(127)
    assert pool.vs[p, 0].item() == big and pool.v[p, 0, 4, 2] == -127 and pool.v[p, 0, 3, 1] == 0
    assert pool.v[q, 0, 0, 1] == 0                                       # a NaN leaves the rest of its row alone
    codes, now = appended(pool.v, pool.vs, q, 0, y[5:].reshape(2, 1, 16), True)
    assert np.array_equal(codes, pool.v[q].cpu().numpy()) and pool.vs[q, 0].item() == now[0]


def test_append_token_by_token(lib):
    """One token at a time through two pages: the definition applied step by step, to the byte."""
    pool = Pool(gen(6), 2, 32, [100], spare=0)
    rows = randn(gen(7), 100, 64) * torch.linspace(0.1, 3, 100).cuda()[:, None]
    want_k, want_ks = pool.k.clone(), pool.ks.clone()
    for i in range(100):
        s = pool.step([1], kv=[i + 1])
        r = rows[i:i + 1]
        call(lib.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), r.data_ptr(), r.data_ptr(), 64, 64, tcg.F32)
        p = int(pool.table[0, i // PAGE])
        c, now = appended(want_k, want_ks, p, i % PAGE, r.reshape(1, 2, 32), False)
        want_k[p], want_ks[p] = torch.from_numpy(c).cuda(), torch.from_numpy(now).cuda()
    assert torch.equal(pool.k, want_k) and torch.equal(pool.ks, want_ks)
    for p in range(2):
        slots = 64 if p == 0 else 36
        i = int(pool.table[0, p])
        assert torch.equal(pool.v[i].transpose(1, 2)[:, :slots], pool.k[i][:, :slots])      # the same rows, dim-major
    assert torch.equal(pool.vs, pool.ks)


# ------------------------------------------------------------------ attention

def attention(pool, q, new, kv, group, scale, causal, window, t):
    """64-bit attention and the tolerance of each value. q [n, heads, d]."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    digits, weight = (2 * 8300000.0, 2.0 ** -24) if t == "f32" else (2 * 32512.0, 2.0 ** -17)
    at = 0
    for b, (n, k_n) in enumerate(zip(new, kv)):
        if n == 0:
            continue
        k, v = (x.cpu() for x in pool.values(b, k_n))
        pos, key = torch.arange(k_n - n, k_n)[:, None], torch.arange(k_n)[None]
        see = (key <= pos) if causal else torch.ones((n, k_n), dtype=torch.bool)
        if window:
            see &= key > pos - window
        x = q[at:at + n].double().cpu()
        for h in range(q.shape[1]):
            kk, vv = k[h // group], v[h // group]
            s = (x[:, h] @ kk.T * scale).masked_fill(~see, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            l = p.sum(-1, keepdim=True)
            out[at:at + n, h] = p @ vv / l
            # a score is off by half a digit of q against each |k|, by 10 roundings of fp32 (the two sums' conversions and
            # their join, the factor, the subtraction, the maximum raised by 2^-22) of the largest score (in exp2's units
            # 1.45 of it), and ex2 by 2^-22; a weight by half its digits' step, against the sum l. Both twice (sum and
            # division). Folding tiles into fp32 rounds once a tile, the merge of partial results 40 times at most.
            half_q = x[:, h].abs().amax(-1, keepdim=True) / digits * scale
            reach = half_q * kk.abs().sum(-1).max() + 20 * U * s.masked_fill(~see, 0).abs().amax(-1, keepdim=True) + 2.0 ** -22
            seen = see.sum(-1, keepdim=True)
            rel = 2 * (torch.expm1(reach) + seen * weight / l) + (k_n / PAGE + 40) * U
            tol[at:at + n, h] = rel * vv.abs().max()
        at += n
    return out, tol + out.abs() * half_step(TYPES[t][0])


def check_attention(lib, pool, new, heads, t, causal=True, window=0, seed=0, spread=1.0, pad=0, extra=0, offset=0, scale=None,
                    **kw):
    dt, code = TYPES[t]
    n, d = sum(new), pool.d
    scale = scale or 1 / math.sqrt(d)
    ld = heads * d + extra
    raw = randn(gen(seed), (n + pad) * ld + offset + 16, dtype=dt, spread=spread)
    q = raw[offset:offset + (n + pad) * ld].view(n + pad, ld)
    out = torch.full((raw.numel(),), 7.0, dtype=dt, device="cuda")
    o = out[offset:offset + (n + pad) * ld].view(n + pad, ld)
    s = pool.step(new, pad=pad, **kw)
    args = (C.byref(pool.cache()), C.byref(s), heads, ld, ld, scale, causal, window, code)
    call(lib.tcg_kv8_attention, o.data_ptr(), q.data_ptr(), *args)
    x = q[:n, :heads * d].reshape(n, heads, d)
    want, tol = attention(pool, x, new, kw.get("kv") or pool.kv, heads // pool.n_kv, scale, causal, window, t)
    got = o[:n, :heads * d].reshape(n, heads, d).double().cpu()
    over = (got - want).abs() - tol
    assert (over <= 0).all(), f"{over.max():.3g} over a tolerance of {tol.max():.3g}"
    assert (o[:, heads * d:] == 7).all() and (o[n:] == 7).all() and (out[:offset] == 7).all()
    first = o.clone()
    call(lib.tcg_kv8_attention, o.data_ptr(), q.data_ptr(), *args)
    assert torch.equal(first, o)                                         # the same bits again
    return got


ATTN = [  # n_kv, group, d, [(new, kv)], causal, window
    (1, 1, 64, [(1, 1)], True, 0), (2, 4, 128, [(1, 513)], True, 0), (1, 16, 128, [(1, 64), (1, 65), (1, 63), (1, 700)], True, 0),
    (8, 4, 128, [(1, 3000)], True, 0), (1, 8, 96, [(1, 4097), (1, 9)], True, 1000), (2, 1, 32, [(1, 130), (0, 40), (1, 1)], True, 0),
    (1, 5, 16, [(3, 3), (1, 100)], True, 0), (2, 2, 80, [(8, 8), (5, 77), (1, 64)], True, 3), (1, 17, 64, [(1, 500)], True, 0),
    (1, 32, 128, [(1, 900), (1, 2)], False, 0), (2, 4, 128, [(100, 100), (33, 200), (64, 64)], True, 0),
    (1, 1, 64, [(130, 130), (1, 1), (0, 0), (65, 1000)], True, 0), (1, 3, 112, [(70, 300)], True, 64),
    (2, 2, 64, [(40, 333), (7, 65)], False, 0), (1, 4, 48, [(257, 257)], True, 1), (1, 7, 128, [(20, 2100)], True, 0),
    (1, 1, 128, [(65, 65), (128, 129), (129, 400)], True, 0), (2, 3, 64, [(22, 3000), (1, 5)], True, 0),
    (150, 1, 64, [(33, 90)], True, 0), (1, 2, 32, [(16, 1000), (9, 64)], True, 100), (3, 24, 80, [(1, 1), (1, 1500)], True, 0),
]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("n_kv,group,d,seqs,causal,window", ATTN)
def test_attention(lib, n_kv, group, d, seqs, causal, window, t):
    new, kv = [a for a, _ in seqs], [b for _, b in seqs]
    pool = Pool(gen(d + n_kv), n_kv, d, kv)
    check_attention(lib, pool, new, n_kv * group, t, causal, window, seed=len(kv), pad=2)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("extra,offset", [(1, 0), (0, 1), (2, 2), (4, 4), (8, 8), (3, 5)])
def test_attention_strides_and_alignment(lib, extra, offset, t):
    for new, kv in (([1, 1], [200, 70]), ([30, 3], [200, 70])):
        check_attention(lib, Pool(gen(11), 2, 64, kv), new, 4, t, extra=extra, offset=offset, pad=1)


@pytest.mark.parametrize("t", list(TYPES))
def test_attention_of_peaked_and_huge_scores(lib, t):
    pool = Pool(gen(12), 1, 128, [777, 900])
    for spread in (0.0, 1e-4, 20.0, 400.0):                              # scores of 0, of 1e-4, of tens and of thousands
        check_attention(lib, pool, [1, 2], 4, t, spread=spread, seed=5)
    check_attention(lib, pool, [1, 60], 4, t, spread=30.0, seed=6)
    pool.ks[:], pool.vs[:] = 0.0, 1e-3                                   # keys of a page of zeros: equal weights
    check_attention(lib, pool, [3, 40], 4, t)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows", [[1, 1], [12, 5], [70, 33]])
def test_attention_of_pages_of_unlike_scales(lib, rows, t):
    """Scales spread over decades from page to page, some of them zero."""
    pool = Pool(gen(60), 2, 64, [1500, 700])
    g = gen(61)
    pool.ks = (10.0 ** (torch.rand(pool.ks.shape, generator=g) * 3 - 3)).cuda()
    pool.vs = (10.0 ** (torch.rand(pool.vs.shape, generator=g) * 5 - 3)).cuda()
    zero = pool.table[:, 3].long()
    pool.ks[zero[0]], pool.vs[zero[1]] = 0.0, 0.0
    check_attention(lib, pool, rows, 8, t, scale=0.02)
    pool.vs[pool.table[0, :24].long()] = 0.0                             # nothing but zeros to add up
    check_attention(lib, pool, rows, 8, t, scale=0.02)


@pytest.mark.parametrize("magnitude", [1e-36, 1e-25, 1e25, 1e36])
@pytest.mark.parametrize("rows", [[1, 1], [12, 5], [70, 33]])
def test_attention_of_tiny_and_huge_queries(lib, rows, magnitude):
    """Queries at the ends of fp32's range, with a scale that brings the scores back to ones of ordinary size."""
    pool = Pool(gen(62), 2, 64, [300, 200])
    if magnitude > 1:
        check_attention(lib, pool, rows, 4, "f32", spread=magnitude, scale=float(np.float32(0.125 / magnitude)))
    else:                                                                # the largest scale that is taken is 1e30
        pool.ks *= 1e6
        check_attention(lib, pool, rows, 4, "f32", spread=magnitude, scale=float(np.float32(min(1e30, 1e-7 / magnitude))))


def test_a_cache_past_32_bit_offsets(lib):
    """Pages behind the first 4 GB of codes."""
    n_pages, n_kv, d, n = 66100, 8, 128, 200                             # 4.3 GB of K codes, as much of V
    pool = Pool(gen(63), n_kv, d, [n])
    small = pool.k, pool.v, pool.ks, pool.vs, pool.table.clone()
    pool.k, pool.v = (torch.empty((n_pages,) + x.shape[1:], dtype=torch.int8, device="cuda") for x in small[:2])
    pool.ks, pool.vs = (torch.full((n_pages, n_kv), float("nan"), device="cuda") for _ in range(2))
    old = small[4][0, :4].long()
    far = torch.tensor([n_pages - 1, 65600, n_pages - 3, 65536], device="cuda")
    pool.k[far], pool.v[far], pool.ks[far], pool.vs[far] = (x[old] for x in small[:4])
    pool.table[0, :4], pool.n = far.to(torch.int32), n_pages
    assert int(far.min()) * n_kv * 64 * d >= 2 ** 32
    for rows in ([1], [30]):
        check_attention(lib, pool, rows, 16, "f32")
    x = randn(gen(64), 70, n_kv * d)
    s = pool.step([70])
    call(lib.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), x.data_ptr(), x.data_ptr(), n_kv * d, n_kv * d, tcg.F32)
    out = [torch.empty_like(x) for _ in range(2)]
    call(lib.tcg_kv8_read, out[0].data_ptr(), out[1].data_ptr(), C.byref(pool.cache()), C.byref(s), n_kv * d, n_kv * d, tcg.F32)
    for o, sc in zip(out, (pool.ks, pool.vs)):
        assert ((o - x).abs() <= sc[far].max() * 0.5001).all()          # half a step of the page's scale
    check_attention(lib, pool, [70], 16, "bf16")


def test_attention_contains_odd_queries(lib):
    """A NaN or an infinity in one query makes that row NaN and no other."""
    pool = Pool(gen(13), 2, 64, [300, 64])
    for new in ([1, 1], [40, 9]):
        q = randn(gen(14), sum(new), 8, 64)
        clean = q.clone()
        q[0, 1, 5], q[-1, 6, 63] = float("nan"), float("inf")
        s, out = pool.step(new), [torch.empty_like(q) for _ in range(2)]
        for x, o in zip((q, clean), out):
            call(lib.tcg_kv8_attention, o.data_ptr(), x.data_ptr(), C.byref(pool.cache()), C.byref(s), 8, 512, 512, 0.125,
                 True, 0, tcg.F32)
        bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
        bad[0, 1] = bad[-1, 6] = True
        assert out[0][bad].isnan().all() and torch.equal(out[0][~bad], out[1][~bad]) and not out[1].isnan().any()


def test_long_cache_and_launch_hints(lib):
    """max_kv only sizes the launch: any value gives the result, whatever the split over CTAs."""
    pool = Pool(gen(15), 1, 64, [20011])
    for hint in (0, 1, 5000, 20011, 2 ** 31 - 1):
        check_attention(lib, pool, [1], 4, "f32", max_kv=hint)
        check_attention(lib, pool, [30], 4, "bf16", max_kv=hint, max_new=31)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("group,d", [(1, 64), (4, 128), (20, 64)])
def test_attention_of_a_prompt_among_decode_steps(lib, group, d, t):
    """Sequences of unlike lengths: blocks of rows dealt out by the lengths, short sequences in a launch of their own."""
    g = torch.Generator().manual_seed(70)
    seqs = [(1, int(torch.randint(1, 900, (1,), generator=g))) for _ in range(90)]
    seqs[17], seqs[40], seqs[41], seqs[89] = (700, 900), (0, 33), (5, 70), (33, 33)
    pool = Pool(gen(71), 1, d, [b for _, b in seqs])
    check_attention(lib, pool, [a for a, _ in seqs], group, t, pad=3)
    check_attention(lib, pool, [a for a, _ in seqs], group, t, window=100)
    check_attention(lib, pool, [0] * 89 + [33], group, t, max_new=33)   # nothing but one


def test_bad_lengths_among_unlike_sequences(gpu):
    """A refused sequence is reported and the others are right, wherever the blocks of rows come from."""
    L = tcg.lib()
    tcg.check(L.tcg_clear_device_error())
    lens = [1] * 80
    lens[50] = 600
    kv = [40] * 80
    kv[50] = 640
    pool = Pool(gen(72), 1, 64, kv)
    q = randn(gen(73), sum(lens), 4, 64)
    want = torch.empty_like(q)
    s = pool.step(lens)
    args = (4, 256, 256, 0.125, True, 0, tcg.F32)
    call(L.tcg_kv8_attention, want.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), *args)
    assert L.tcg_device_error() == 0
    for bad in (0, 50, 79):
        kv2 = list(kv)
        kv2[bad] = 10 ** 6
        s, out = pool.step(lens, kv=kv2), torch.full_like(q, 7.0)
        call(L.tcg_kv8_attention, out.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), *args)
        assert L.tcg_device_error() == tcg.ERR_KV8_LENGTHS
        tcg.check(L.tcg_clear_device_error())
        at = sum(lens[:bad])
        mine = torch.zeros(len(q), dtype=torch.bool, device="cuda")
        mine[at:at + lens[bad]] = True
        assert (out[mine] == 7).all() and torch.equal(out[~mine], want[~mine])


def test_device_side_refusals(gpu):
    """Lengths and pages that cannot be: skipped on the device, reported, and everything else is right."""
    L = tcg.lib()
    tcg.check(L.tcg_clear_device_error())

    def error(code):
        torch.cuda.synchronize()
        assert L.tcg_device_error() == code
        tcg.check(L.tcg_clear_device_error())

    q = randn(gen(17), 6, 4, 64)
    x = randn(gen(18), 6, 128)
    bad_steps = [dict(kv=[100, 1, 100]), dict(kv=[100, 100000, 100]), dict(kv=[100, -5, 100]), dict(max_new=1)]
    for kw in bad_steps:
        pool = Pool(gen(16), 2, 64, [100, 100, 100])                     # anew: the same rows twice change nothing
        new = [1, 3, 1] if "max_new" in kw else [1, 2, 1]
        s = pool.step(new, **kw)
        good = [0, sum(new) - 1]
        out = torch.full_like(q, 7.0)
        call(L.tcg_kv8_attention, out.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), 4, 256, 256, 0.125, True,
             0, tcg.F32)
        error(tcg.ERR_KV8_LENGTHS)
        assert (out[1:sum(new) - 1] == 7).all() and (out[good] != 7).all()
        rows = [torch.full((6, 128), 7.0, device="cuda") for _ in range(2)]
        call(L.tcg_kv8_read, rows[0].data_ptr(), rows[1].data_ptr(), C.byref(pool.cache()), C.byref(s), 128, 128, tcg.F32)
        error(tcg.ERR_KV8_LENGTHS)
        assert (rows[0][1:sum(new) - 1] == 7).all() and (rows[0][good] != 7).any()
        k = pool.k.clone()
        mine = pool.table[1, :2].long()
        call(L.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), x.data_ptr(), x.data_ptr(), 128, 128, tcg.F32)
        error(tcg.ERR_KV8_LENGTHS)
        assert torch.equal(k[mine], pool.k[mine]) and not torch.equal(k, pool.k)

    # a page that does not exist: its 64 tokens are masked, read as zeros, not written
    for page in (-1, None, 2 ** 31 - 1, -2 ** 31):
        pool = Pool(gen(19), 2, 64, [100, 250, 100])
        pool.table[1, 2] = pool.n if page is None else page              # the first one behind the pool
        s = pool.step([1, 70, 1])
        q = randn(gen(20), 72, 4, 64)
        out = torch.full_like(q, 7.0)
        call(L.tcg_kv8_attention, out.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), 4, 256, 256, 0.125, True,
             0, tcg.F32)
        error(tcg.ERR_KV8_PAGE)
        pages = pool.table[1, :4].clone()
        pages[2] = pool.table[1, 0]
        k = (pool.k[pages.long()].double() * pool.ks[pages.long()].double()[..., None, None]).permute(1, 0, 2, 3).reshape(2, -1, 64)
        v = (pool.v[pages.long()].double() * pool.vs[pages.long()].double()[..., None, None]).permute(1, 0, 3, 2).reshape(2, -1, 64)
        pos, key = torch.arange(180, 250, device="cuda")[:, None], torch.arange(256, device="cuda")[None]
        hide = (key > pos) | ((key >= 128) & (key < 192))
        for h in range(4):
            w = torch.softmax((q[1:71, h].double() @ k[h // 2].T * 0.125).masked_fill(hide, -math.inf), -1) @ v[h // 2]
            assert (out[1:71, h].double() - w).abs().max() < 1e-4 * v.abs().max()
        rows = [torch.full((72, 128), 7.0, device="cuda") for _ in range(2)]
        call(L.tcg_kv8_read, rows[0].data_ptr(), rows[1].data_ptr(), C.byref(pool.cache()), C.byref(s), 128, 128, tcg.F32)
        error(tcg.ERR_KV8_PAGE)
        assert (rows[0][1:13] == 0).all() and (rows[0][13:71] != 0).any() and (rows[1][1:13] == 0).all()
        x = randn(gen(21), 72, 128)
        before = pool.k.clone()
        call(L.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), x.data_ptr(), x.data_ptr(), 128, 128, tcg.F32)
        error(tcg.ERR_KV8_PAGE)
        written = (pool.k != before).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(written) == {int(pool.table[0, 1]), int(pool.table[1, 3]), int(pool.table[2, 1])}
    # a query whose every key lies in such a page gets zeros
    pool = Pool(gen(22), 1, 64, [10])
    pool.table[0, 0] = -1
    s = pool.step([2])
    out = torch.full((2, 1, 64), 7.0, device="cuda")
    call(L.tcg_kv8_attention, out.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), 1, 64, 64, 0.125, True, 0, tcg.F32)
    error(tcg.ERR_KV8_PAGE)
    assert (out == 0).all()


def test_a_reported_page_leaves_other_operators_alone(gpu):
    """The word stays raised until it is cleared, and a host-buffer op, which would abort on a failed wait, still runs."""
    L = tcg.lib()
    tcg.check(L.tcg_clear_device_error())
    pool = Pool(gen(50), 1, 64, [10])
    pool.table[0, 0] = pool.n
    q = randn(gen(51), 1, 1, 64)
    out = torch.empty_like(q)
    s = pool.step([1])
    call(L.tcg_kv8_attention, out.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), 1, 64, 64, 0.125, True, 0, tcg.F32)
    assert L.tcg_device_error() == tcg.ERR_KV8_PAGE
    a, b, y = np.arange(8, dtype=np.float32), np.ones(8, np.float32), np.zeros(8, np.float32)
    L.tc_ref_add.restype = None
    L.tc_ref_add.argtypes = [C.c_void_p] * 3 + [C.c_size_t]
    L.tc_ref_add(y.ctypes.data, a.ctypes.data, b.ctypes.data, 8)
    assert np.array_equal(y, a + b)
    assert L.tcg_device_error() == tcg.ERR_KV8_PAGE
    tcg.check(L.tcg_clear_device_error())
    assert L.tcg_device_error() == 0


# ------------------------------------------------------------------ together

def test_a_run_of_them_in_a_graph(lib):
    """Prompt, then decode steps replayed from one captured graph on a caller's stream: norm and rotation, append,
    attention, against 64 bits over the unquantised keys up to the cache's own rounding."""
    heads, n_kv, d, eps = 8, 2, 64, 1e-6
    g = gen(30)
    pool = Pool(g, n_kv, d, [256, 256], spare=0)
    r = plan(d, d, True, 500000.0)
    wq, wk = randn(g, d) * 0.1 + 1, randn(g, d) * 0.1 + 1
    wide = (heads + 2 * n_kv) * d
    stream = torch.cuda.Stream()
    tcg.check(lib.tcg_set_stream(stream.cuda_stream))
    try:
        start, kv = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        cache = pool.cache()

        def step(rows, pos, out, n, max_new):
            s = tcg.Kv8Step(start.data_ptr(), kv.data_ptr(), pool.table.data_ptr(), pool.ld, 2, n, max_new, 256)
            size = rows.element_size()
            q, k, v = (rows.data_ptr() + i * d * size for i in (0, heads, heads + n_kv))
            tcg.check(lib.tcg_qk_norm_rope(q, k, q, k, wq.data_ptr(), wk.data_ptr(), eps, pos.data_ptr(), C.byref(r), n,
                                           heads, n_kv, wide, wide, wide, wide, tcg.F32))
            tcg.check(lib.tcg_kv8_append(C.byref(cache), C.byref(s), k, v, wide, wide, tcg.F32))
            tcg.check(lib.tcg_kv8_attention(out.data_ptr(), q, C.byref(cache), C.byref(s), heads, heads * d, wide,
                                            1 / math.sqrt(d), True, 0, tcg.F32))

        hist = [[], []]

        def exact(raw, pos, b):
            x = raw.double().view(-1, heads + 2 * n_kv, d)
            x, v = x[:, :heads + n_kv], x[:, heads + n_kv:]
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
            x = torch.cat([x[:, :heads] * wq.double(), x[:, heads:] * wk.double()], 1)
            x, _ = rotated(x, pos, r)
            hist[b].append((x[:, heads:], v))
            k, v = (torch.cat([h[i] for h in hist[b]]) for i in range(2))
            n, m = x.shape[0], k.shape[0]
            hide = torch.arange(m, device="cuda")[None] > torch.arange(m - n, m, device="cuda")[:, None]
            o = [torch.softmax((x[:, h] @ k[:, h // 4].T / math.sqrt(d)).masked_fill(hide, -math.inf), -1) @ v[:, h // 4]
                 for h in range(heads)]
            return torch.stack(o, 1)

        def near(got, want):
            # keys and values carry the cache's rounding, up to a step of max / 127 of a page each (half when written, half
            # when the page's scale grows): about 1% of a value, and of a score; 4% covers both
            assert (got.double() - want).norm() <= 0.04 * want.norm()

        lens = [70, 20]
        raw = randn(g, sum(lens), wide)
        pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).cuda()
        start.copy_(torch.tensor([0, 70, 90], dtype=torch.int32))
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        rows, out = raw.clone(), torch.empty((90, heads, d), device="cuda")
        torch.cuda.synchronize()
        step(rows, pos, out, 90, 70)
        torch.cuda.synchronize()
        near(out[:70], exact(raw[:70], pos[:70], 0))
        near(out[70:], exact(raw[70:], pos[70:], 1))

        # one token each, captured once, replayed with new rows and lengths
        rows1, pos1 = torch.zeros((2, wide), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        out1 = torch.empty((2, heads, d), device="cuda")
        start.copy_(torch.tensor([0, 1, 2], dtype=torch.int32))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(rows1, pos1, out1, 2, 1)
        for i in range(60):                                              # past the end of a page of each sequence
            raw = randn(g, 2, wide)
            rows1.copy_(raw)
            pos1.copy_(torch.tensor(lens, dtype=torch.int32))
            lens = [n + 1 for n in lens]
            kv.copy_(torch.tensor(lens, dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for b in range(2):
                near(out1[b:b + 1], exact(raw[b:b + 1], pos1[b:b + 1], b))
    finally:
        torch.cuda.synchronize()
        tcg.check(lib.tcg_set_stream(None))


CAPTURED_FIRST = """
import sys, torch
sys.path[:0] = sys.argv[1:3]
import tcg, test_gpu_lm as T
tcg.init(0)
L, g = tcg.lib(), T.gen(80)
pool = T.Pool(g, 2, 64, [300, 90])
for new in ([1, 1], [3, 20], [40, 33]):
    q, out = T.randn(g, sum(new), 8, 64), torch.zeros((sum(new), 8, 64), device="cuda")
    x = T.randn(g, sum(new), 128)
    pos, r = torch.arange(sum(new), dtype=torch.int32, device="cuda"), T.plan(64, 64, True)
    s = pool.step(new)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    tcg.check(L.tcg_set_stream(stream.cuda_stream))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        tcg.check(L.tcg_rope(x.data_ptr(), x.data_ptr(), pos.data_ptr(), T.C.byref(r), sum(new), 2, 128, 128, 0))
        tcg.check(L.tcg_kv8_append(T.C.byref(pool.cache()), T.C.byref(s), x.data_ptr(), x.data_ptr(), 128, 128, 0))
        tcg.check(L.tcg_kv8_attention(out.data_ptr(), q.data_ptr(), T.C.byref(pool.cache()), T.C.byref(s), 8, 512, 512,
                                      0.125, True, 0, 0))
    graph.replay()
    torch.cuda.synchronize()
    tcg.check(L.tcg_set_stream(None))
    want, tol = T.attention(pool, q, new, pool.kv, 4, 0.125, True, 0, "f32")
    assert ((out.double().cpu() - want).abs() <= tol).all()
assert L.tcg_device_error() == 0
print("captured")
"""


def test_first_calls_inside_a_capture():
    """A process whose first call of each operator is captured: nothing that a capture forbids happens in it."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    pkg = os.path.join(os.path.dirname(here), "roofline.c_b200")
    out = subprocess.run([sys.executable, "-c", CAPTURED_FIRST, here, pkg], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_two_streams_at_once(lib):
    """The operators keep nothing between calls: two streams' calls over one cache do not disturb each other."""
    pool = Pool(gen(40), 4, 128, [5000, 3000])
    s = pool.step([1, 1])
    q = [randn(gen(41 + i), 2, 16, 128) for i in range(2)]
    want = [torch.empty_like(x) for x in q]
    args = (C.byref(pool.cache()), C.byref(s), 16, 2048, 2048, 0.09, True, 0, tcg.F32)
    for x, o in zip(q, want):
        call(lib.tcg_kv8_attention, o.data_ptr(), x.data_ptr(), *args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(x) for _ in range(20)] for x in q]
    torch.cuda.synchronize()
    try:
        for i in range(20):
            for k in range(2):
                tcg.check(lib.tcg_set_stream(streams[k].cuda_stream))
                tcg.check(lib.tcg_kv8_attention(got[k][i].data_ptr(), q[k].data_ptr(), *args))
    finally:
        torch.cuda.synchronize()
        tcg.check(lib.tcg_set_stream(None))
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in got[k])
