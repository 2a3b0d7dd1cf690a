"""Attention over the 8-bit cache where softmax is far from broad: one key that
holds nearly all of the weight, a page's V beside one of another magnitude,
scores past what 24 bits resolve. Against 64 bits, with bounds that do not grow
with the number of keys but for the sums' own roundings.

u = 2^-24 is half a step of fp32, half_step(t) that of the output type.
"""
import ctypes as C
import math

import pytest
import torch

import tcg
from test_gpu_lm import PAGE, TYPES, U, Pool, call, gen, half_step, lib, randn  # noqa: F401

pytestmark = pytest.mark.gpu


def exact(pool, q, new, kv, group, scale, t, causal=True, window=0):
    """64-bit attention of q [n, heads, d] and the bound on each value's error, on the GPU."""
    few = max(new) * group <= 64
    f32 = t == "f32"
    out, tol = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        k, v = pool.values(b, m)
        pos, key = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        see = (key <= pos) if causal else torch.ones((n, m), dtype=torch.bool, device="cuda")
        if window:
            see &= key > pos - window
        x = q[at:at + n].double()
        for h in range(q.shape[1]):
            kk, vv = k[h // group], v[h // group]
            s = (x[:, h] @ kk.T * scale).masked_fill(~see, -math.inf)
            w = torch.exp(s - s.amax(-1, keepdim=True))
            l = w.sum(-1, keepdim=True)
            mass = w @ vv.abs() / l
            big = s.masked_fill(~see, 0).abs().amax(-1, keepdim=True)
            reach = kk.abs().sum(-1)[None].expand(n, -1).masked_fill(~see, 0).amax(-1, keepdim=True)
            top = x[:, h].abs().amax(-1, keepdim=True)
            # A score: few rows, half a digit of q (of its row's largest) against each |k|; many rows, q as it is (two
            # pieces of 11 bits with fp32) and a truncating sum, 2e-8 of its magnitude for each of at most 16 MMAs. Then
            # six roundings of the scaled score and ex2's 2^-22. Twice (weights and their sum).
            score = top / (2 * 8300000.0 if f32 else 2 * 32512.0) if few else top * (16 * 2e-8 + 2.0 ** -22)
            delta = score * scale * reach + 6 * U * big + 2.0 ** -22
            rel = 2 * torch.expm1(delta) + (m / PAGE + 40) * U
            if few:
                # Weights are whole numbers against the largest of their own tile, half a step off each: of 23 bits, or of
                # 16 where the inputs are and every 16 keys of the tile hold 1/16 of that weight (0.06: rounding).
                pad = -m % PAGE
                wt = torch.nn.functional.pad(w, (0, pad)).view(n, -1, 4, PAGE // 4)
                vt = torch.nn.functional.pad(vv.abs(), (0, 0, 0, pad)).view(-1, PAGE, vv.shape[1]).amax(1)
                top_w = wt.amax((-1, -2))
                coarse = (wt.sum(-1) >= 0.06 * top_w[..., None]).all(-1) & torch.tensor(not f32, device="cuda")
                lost = PAGE * (torch.where(coarse, 2.0 ** -17, 2.0 ** -24) * top_w) @ vt / l
            else:
                # Weights are fp16 under 2^8 (two of them with fp32): half a step, 2^-11 (2^-22), and that of fp16's
                # subnormals, 2^-25 / 2^8 of a reference at most 2^8 over the group's largest weight, of pages whose V scales
                # are within 2^3: six standard deviations (0.58 each) of as many roundings as a group has keys, against the
                # row's own sum of weights times |V| (the largest key's |V| a quarter of the page's or more), or, where
                # that key's V is 0, all of them against the key.
                rel += (2.0 ** -22 if f32 else 2.0 ** -11) + (64 if f32 else 256) * 2e-8
                group_keys = min(m, 512 if f32 else 4096)
                lost = torch.minimum(torch.minimum(w, torch.full_like(w, 2.0 ** -33)) @ vv.abs() / l,
                                     4 * 6 * 0.58 * math.sqrt(group_keys) * 2.0 ** -22 * mass)
            out[at:at + n, h] = w @ vv / l
            tol[at:at + n, h] = mass * rel + lost
        at += n
    return out, tol + out.abs() * half_step(TYPES[t][0])


def run(lib, pool, q, new, heads, scale, t, causal=True, window=0, **kw):
    out = torch.full_like(q, float("nan"))
    s = pool.step(new, **kw)
    ld = heads * pool.d
    call(lib.tcg_kv8_attention, out.data_ptr(), q.data_ptr(), C.byref(pool.cache()), C.byref(s), heads, ld, ld, scale, causal,
         window, TYPES[t][1])
    return out


def near(got, want, tol):
    if not got.numel():
        return
    over = (got.double() - want).abs() - tol
    worst = ((got.double() - want).abs() / want.abs().clamp(min=1e-300)).max().item()
    assert (over <= 0).all(), f"{over.max():.3g} over; relative error up to {worst:.3g}"


# ------------------------------------------------------------------ one key holds nearly all of the weight

def sink(seed, n_kv, d, keys, held, group, new, t):
    """Key 0 holds `held` of every row's weight and a V of zeros; the others' scores are normal, their V has one sign."""
    pool, g = Pool(gen(seed), n_kv, d, [keys], spare=0), gen(seed + 1)
    pool.ks[:], pool.vs[:] = 1 / 73.0, 0.01
    page, dims = int(pool.table[0, 0]), 16                               # dims that the sink's score comes from
    pool.k[..., :dims] = 0
    pool.k[page, :, 0] = 0
    pool.k[page, :, 0, :dims] = 127
    pool.v.copy_(torch.randint(32, 97, tuple(pool.v.shape), generator=g, dtype=torch.int8))
    pool.v[page, :, :, 0] = 0
    gap = math.log(keys * math.exp(0.5 * (d - dims) / d) * held / (1 - held))
    q = randn(g, new, n_kv * group, d, dtype=torch.float64)
    q[..., :dims] = gap * math.sqrt(d) / (dims * 127 / 73.0)
    return pool, q.to(TYPES[t][0])


SINKS = [  # tokens, query heads a key head, key heads, d: the shapes for 8, 16, 32 and 64 rows, and for many
    (1, 4, 1, 128), (4, 4, 1, 64), (7, 4, 1, 128), (5, 8, 1, 64), (16, 4, 1, 128), (16, 4, 160, 64), (70, 4, 1, 128),
]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("keys,held", [(2048, 0.99), (8192, 0.99), (131072, 0.9), (131072, 0.99)])
@pytest.mark.parametrize("new,group,n_kv,d", SINKS)
def test_attention_beside_a_sink(lib, new, group, n_kv, d, keys, held, t):
    if n_kv > 1:
        keys = min(keys, 2048)                                           # every SM has a key head: no split of the keys
    pool, q = sink(100, n_kv, d, keys, held, group, new, t)
    want, tol = exact(pool, q, [new], [keys], group, 1 / math.sqrt(d), t)
    assert (tol < 0.02 * want.abs()).all()                               # a lost tail does not fit under the bound
    near(run(lib, pool, q, [new], n_kv * group, 1 / math.sqrt(d), t), want, tol)


@pytest.mark.parametrize("new,group", [(1, 4), (7, 4), (16, 4), (70, 4)])
def test_a_row_does_not_depend_on_the_launch(lib, new, group):
    """The same rows over the same keys, whatever the split that the launch's hint leads to: alike to the bound's size."""
    pool, q = sink(110, 1, 64, 20000, 0.99, group, new, "bf16")
    want, tol = exact(pool, q, [new], [20000], group, 0.125, "bf16")
    for hint in (1, 700, 20000):
        near(run(lib, pool, q, [new], group, 0.125, "bf16", max_kv=hint), want, tol)


# ------------------------------------------------------------------ pages of unlike V scales

@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("low", [2.0 ** -7, 1e-6, 1e-12, 1e-30, 0.0])
@pytest.mark.parametrize("new,group", [(1, 4), (16, 4), (250, 4)])
@pytest.mark.parametrize("gap", [0.0, 20.0])
def test_attention_of_rows_whose_weight_lies_in_pages_of_small_v(lib, new, group, gap, low, t):
    """Every other page's V is `low` times its neighbours'. Rows that see the small one alone, or give it e^gap times the
    weight, are as right as any."""
    keys, d = 250, 128
    for first in (0, 1):
        pool = Pool(gen(130), 1, d, [keys])
        pool.ks[:] = 1 / 73.0
        for i in range(4):
            page = int(pool.table[0, i])
            small = i % 2 == first
            pool.vs[page] = 0.01 * (low if small else 1.0)
            pool.k[page, :, :, :16] = 127 if small else 0
        q = randn(gen(131), new, group, d, dtype=torch.float64)
        q[..., :16] = gap * math.sqrt(d) / (16 * 127 / 73.0)
        q = q.to(TYPES[t][0])
        want, tol = exact(pool, q, [new], [keys], group, 1 / math.sqrt(d), t)
        near(run(lib, pool, q, [new], group, 1 / math.sqrt(d), t), want, tol)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("new,group", [(3, 4), (140, 1), (190, 4)])
def test_attention_of_v_scales_at_the_ends_of_fp32(lib, new, group, t):
    """A later page of huge V leaves the rows before it alone; scales below fp32's normal numbers are scales."""
    pool = Pool(gen(140), 1, 64, [190])
    pages = pool.table[0, :3].long()
    q = randn(gen(141), new, group, 64, dtype=TYPES[t][0])
    for huge in (1e30, 1e36):
        pool.vs[pages] = torch.tensor([1e-3, 1e20, huge], device="cuda")[:, None]
        want, tol = exact(pool, q, [new], [190], group, 0.125, t)
        got = run(lib, pool, q, [new], group, 0.125, t)
        # the sum of weights times V passes fp32's range with the second one: 60 x 1.27e38 over rows that see that page
        sees = torch.arange(190 - new, 190) >= (128 if huge > 1e30 else 190)
        near(got[~sees], want[~sees], tol[~sees])
    pool.vs[pages] = torch.tensor([2e-39, 3e-40, 1e-38], device="cuda")[:, None]
    want, tol = exact(pool, q, [new], [190], group, 0.125, t)
    # a page's factor is rounded to 2^-150 and multiplied by its P V, below 64 * 127 * 2^23 at 2^11 for few rows, and
    # below 128 * 127 * 2^15 for many: 2^-123 for three pages
    near(run(lib, pool, q, [new], group, 0.125, t), want, tol + 2.0 ** -123)


# ------------------------------------------------------------------ scores past what 24 bits resolve

@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("size", [3e2, 1e4, 1e6, 1e8, 1e10, 1e20])
@pytest.mark.parametrize("new,group", [(1, 4), (7, 4), (16, 4), (70, 4)])
def test_attention_of_scores_of_any_size(lib, new, group, size, t):
    """Where the largest score is ahead by more than its own rounding, softmax is one: the row is that key's V."""
    keys, d = 1000, 64
    pool = Pool(gen(120), 2, d, [keys])
    pool.ks *= size / (100.0 * 73 * 0.025 * 8)                           # |q| about 100, |k| 73 codes, 8 = sqrt(d)
    q = randn(gen(121), new, 2 * group, d, dtype=TYPES[t][0], spread=100.0)
    got = run(lib, pool, q, [new], 2 * group, 1.0, t).double()
    k, v = pool.values(0, keys)
    hide = torch.arange(keys, device="cuda")[None] > torch.arange(keys - new, keys, device="cuda")[:, None]
    sure = 0
    for h in range(2 * group):
        s = (q[:, h].double() @ k[h // group].T).masked_fill(hide, -math.inf)
        two, at = s.topk(2, -1)
        # half a digit of q against each |k|, as in exact(), and eight roundings of the largest score; the keys e^40 behind
        # leave what `others` says of them
        slack = q[:, h].double().abs().amax(-1) / 65024 * k[h // group].abs().sum(-1).max() + 8 * U * s.masked_fill(hide, 0).abs().amax(-1)
        ahead = two[:, 0] - two[:, 1] > 2 * slack + 40
        sure += int(ahead.sum())
        want = v[h // group][at[:, 0]]
        others = keys * math.exp(-40) * v.abs().max()
        bad = (got[:, h] - want).abs() > want.abs() * (half_step(TYPES[t][0]) + 2.0 ** -11) + others
        assert not bad[ahead].any(), f"{int(bad[ahead].any(-1).sum())} of {int(ahead.sum())} rows"
        assert got[:, h].isfinite().all()
    assert size < 1e4 or sure > new * group                              # half of the rows and more


# ------------------------------------------------------------------ infinities

@pytest.mark.parametrize("n", [2, 70])
def test_an_infinity_is_read_back_as_the_largest_finite_value(lib, n):
    """Stored by both forms of the append (few rows, many), with fp32's largest value itself, in K and in V."""
    biggest = torch.finfo(torch.float32).max
    pool = Pool(gen(150), 1, 64, [n])
    x = [randn(gen(151 + i), n, 64) for i in range(2)]
    for i in range(2):
        x[i][0, 3], x[i][n - 1, 5 + i], x[i][n - 1, 9] = math.inf, -math.inf, -biggest
    s = pool.step([n])
    call(lib.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), x[0].data_ptr(), x[1].data_ptr(), 64, 64, tcg.F32)
    for dt, code in TYPES.values():
        out = [torch.empty((n, 64), dtype=dt, device="cuda") for _ in range(2)]
        call(lib.tcg_kv8_read, out[0].data_ptr(), out[1].data_ptr(), C.byref(pool.cache()), C.byref(s), 64, 64, code)
        want = torch.tensor(biggest, device="cuda").to(dt)
        for i in range(2):
            assert out[i][0, 3] == want and out[i][n - 1, 5 + i] == -want and out[i][n - 1, 9] == -want
            rest = out[i].clone()
            rest[0, 3] = rest[n - 1, 5 + i] = rest[n - 1, 9] = 0
            assert (rest == 0).all()                                     # half a step of those pages is 1.3e36


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("new,group", [(1, 4), (30, 2), (90, 4)])
def test_attention_over_an_infinite_key(lib, new, group, t):
    """A K with an infinity decides each row that sees it, one way or the other; the rows before it never see it."""
    pool = Pool(gen(160), 1, 64, [200])
    x = randn(gen(161), 1, 64)
    x[0, 7] = math.inf
    v = pool.values(0, 200)[1].clone()
    kv = torch.tensor([171], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    s = tcg.Kv8Step(start.data_ptr(), kv.data_ptr(), pool.table.data_ptr(), pool.ld, 1, 1, 1, 171)
    call(lib.tcg_kv8_append, C.byref(pool.cache()), C.byref(s), x.data_ptr(), x.data_ptr(), 64, 64, tcg.F32)
    pool.v[pool.table[0, 2].long()], pool.vs[pool.table[0, 2].long()] = 0, 0.01      # its V too was infinite
    v = pool.values(0, 200)[1]
    q = randn(gen(162), new, group, 64, dtype=TYPES[t][0])
    q[..., 7] = torch.where(q[..., 7] >= 0, 1.0, -1.0).to(q.dtype)
    got = run(lib, pool, q, [new], group, 0.125, t).double()
    assert got.isfinite().all()
    for i in range(new):
        pos = 200 - new + i
        for h in range(group):
            if pos >= 170 and q[i, h, 7] > 0:                            # the older keys of its page moved to codes of 0
                assert (got[i, h] - v[0, 170]).abs().max() <= 1e-6


# ------------------------------------------------------------------ beside other kernels

def test_attention_between_gemms(lib):
    """Chunks of few blocks, whose kernel lets the next one start early, between GEMMs that take TMEM before they wait for
    it: the chain finishes and gives what the calls give one by one."""
    rows, heads, d = 150, 4, 128
    pool = Pool(gen(170), 1, d, [600])
    s = pool.step([rows])
    w = randn(gen(171), heads * d, heads * d) * 0.05
    x = randn(gen(172), rows, heads * d)
    out, y = torch.empty_like(x), torch.empty_like(x)

    def step(src, sync):
        tcg.check(lib.tcg_kv8_attention(out.data_ptr(), src.data_ptr(), C.byref(pool.cache()), C.byref(s), heads, heads * d,
                                        heads * d, 0.09, True, 0, tcg.F32))
        if sync:
            tcg.check(lib.tcg_sync())
        tcg.check(lib.tcg_linear(y.data_ptr(), out.data_ptr(), w.data_ptr(), None, rows, heads * d, heads * d))
        if sync:
            tcg.check(lib.tcg_sync())

    torch.cuda.synchronize()
    got = []
    for sync in (True, False):
        y.copy_(x)
        torch.cuda.synchronize()
        for i in range(40):
            step(y, sync)
        tcg.check(lib.tcg_sync())
        got.append(y.clone())
    assert torch.equal(*got) and got[0].isfinite().all() and got[0].abs().sum() > 0


THREADS_FIRST = """
import sys, threading, torch
sys.path[:0] = sys.argv[1:3]
import tcg, test_gpu_lm as T
L, g, N = tcg.lib(), T.gen(180), 8
tcg.init(0)
pool = T.Pool(g, 2, 64, [700, 90])
news = ([1, 1], [3, 20], [40, 33])
steps = [pool.step(new) for new in news]
keep = []
for new, s in zip(news, steps):                    # each step's lengths in memory of its own
    keep.append((torch.tensor([0, new[0], sum(new)], dtype=torch.int32).cuda(), torch.tensor(pool.kv, dtype=torch.int32).cuda()))
    s.tok_start, s.kv_len = (x.data_ptr() for x in keep[-1])
qs = [T.randn(g, sum(new), 8, 64) for new in news]
outs = [[torch.zeros_like(q) for q in qs] for _ in range(N)]
cache, wall, bad = pool.cache(), threading.Barrier(N), []
torch.cuda.synchronize()

def work(i):
    try:
        tcg.init(0)
        for q, s, o in zip(qs, steps, outs[i]):
            wall.wait(60)
            tcg.check(L.tcg_kv8_attention(o.data_ptr(), q.data_ptr(), T.C.byref(cache), T.C.byref(s), 8, 512, 512, 0.125, True,
                                          0, 0))
        tcg.check(L.tcg_sync())
    except Exception as e:
        bad.append(e)
        wall.abort()

threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert not bad, bad
for q, s, new, *got in zip(qs, steps, news, *outs):
    want, tol = T.attention(pool, q, new, pool.kv, 4, 0.125, True, 0, "f32")
    for o in got:
        assert torch.equal(o, got[0]) and ((o.double().cpu() - want).abs() <= tol).all()
print("together")
"""


def test_first_calls_of_several_threads_at_once():
    """What a kernel's first call on a device finds out is found by threads that come together, and none of them runs without."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    pkg = os.path.join(os.path.dirname(here), "roofline.c_b200")
    out = subprocess.run([sys.executable, "-c", THREADS_FIRST, here, pkg], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "together" in out.stdout, out.stderr[-2000:]


# ------------------------------------------------------------------ in place

@pytest.mark.parametrize("d,n_rot,half,heads,kv,n,t", [(128, 128, True, 32, 8, 3, "f32"), (64, 32, False, 5, 1, 129, "bf16"),
                                                      (80, 80, True, 7, 2, 17, "f16"), (256, 256, False, 3, 3, 40, "f32"),
                                                      (6, 4, True, 2, 1, 5, "bf16"), (128, 64, True, 40, 8, 6001, "bf16")])
def test_norm_and_rotation_in_place(lib, d, n_rot, half, heads, kv, n, t):
    """Over a fused row's queries and keys, where they lie: the bits of the call out of place, and the values beside them kept."""
    dt, code = TYPES[t]
    g = gen(190)
    r = tcg.Rope()
    tcg.check(lib.tcg_rope_init(C.byref(r), d, n_rot, int(half), 10000.0))
    for ld in ((heads + 2 * kv) * d, (heads + 2 * kv) * d + 3):
        rows = randn(g, n, ld, dtype=dt)
        wq, wk = randn(g, d) + 1, randn(g, d) + 1
        pos = torch.randint(0, 1 << 17, (n,), generator=g, dtype=torch.int32).cuda()
        at, size = heads * d, rows.element_size()
        apart = [torch.empty((n, h * d), dtype=dt, device="cuda") for h in (heads, kv)]
        x = rows.data_ptr()
        call(lib.tcg_qk_norm_rope, apart[0].data_ptr(), apart[1].data_ptr(), x, x + at * size, wq.data_ptr(), wk.data_ptr(), 1e-6,
             pos.data_ptr(), C.byref(r), n, heads, kv, heads * d, kv * d, ld, ld, code)
        place = rows.clone()
        x = place.data_ptr()
        call(lib.tcg_qk_norm_rope, x, x + at * size, x, x + at * size, wq.data_ptr(), wk.data_ptr(), 1e-6, pos.data_ptr(),
             C.byref(r), n, heads, kv, ld, ld, ld, ld, code)
        if ld % 4 == 0:                                                  # else by single values, in another order of sums
            assert torch.equal(place[:, :at], apart[0]) and torch.equal(place[:, at:at + kv * d], apart[1])
        else:
            # two sums of d squares in fp32 and the steps after them, twice: 2 x 25 u of each value, and a step of the type
            for a, b in ((place[:, :at], apart[0]), (place[:, at:at + kv * d], apart[1])):
                pair = b.double().abs().view(n, -1, d).amax(-1, keepdim=True).expand(-1, -1, d).reshape(n, -1)
                assert ((a.double() - b.double()).abs() <= 50 * U * pair + 2 * half_step(dt) * b.double().abs() + 2.0 ** -23 * (t == "f16")).all()
        assert torch.equal(place[:, at + kv * d:], rows[:, at + kv * d:])


# ------------------------------------------------------------------ the shape for a device full of rows, and NaN beside others

@pytest.mark.parametrize("t", list(TYPES))
def test_many_key_heads_of_huge_scores_and_small_v(lib, t):
    """40 rows of each of 150 key heads: warps of 16 rows. As above, one key decides; then V below fp32's normal numbers."""
    pool = Pool(gen(200), 150, 64, [300])
    q = randn(gen(201), 40, 150, 64, dtype=TYPES[t][0], spread=100.0)
    pool.ks *= 1e8 / (100.0 * 73 * 0.025 * 8)
    got = run(lib, pool, q, [40], 150, 1.0, t).double()
    k, v = pool.values(0, 300)
    hide = torch.arange(300, device="cuda")[None] > torch.arange(260, 300, device="cuda")[:, None]
    s = torch.einsum("nhd,hkd->hnk", q.double(), k).masked_fill(hide, -math.inf)
    two, at = s.topk(2, -1)
    slack = (q.double().abs().amax(-1).T / 65024 * k.abs().sum(-1).amax(-1)[:, None]
             + 8 * U * s.masked_fill(hide, 0).abs().amax(-1))            # as in the test of scores of any size
    ahead = two[..., 0] - two[..., 1] > 2 * slack + 40
    want = torch.gather(v, 1, at[..., :1].expand(-1, -1, 64))
    bad = (got.transpose(0, 1) - want).abs() > want.abs() * (half_step(TYPES[t][0]) + 2.0 ** -11) + 300 * math.exp(-40) * v.abs().max()
    assert ahead.float().mean() > 0.8 and not bad[ahead].any()
    if t != "f16":
        pool = Pool(gen(202), 150, 64, [150])
        pool.vs *= 1e-37
        q = randn(gen(203), 40, 150, 64, dtype=TYPES[t][0])
        want, tol = exact(pool, q, [40], [150], 1, 0.125, t)
        near(run(lib, pool, q, [40], 150, 0.125, t), want, tol + 2.0 ** -123)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("new,group", [(2, 4), (4, 4), (8, 4), (16, 4), (40, 4)])
def test_a_nan_query_leaves_the_rows_beside_it_alone(lib, new, group, t):
    pool = Pool(gen(210), 1, 64, [300])
    q = randn(gen(211), new, group, 64, dtype=TYPES[t][0])
    clean = run(lib, pool, q, [new], group, 0.125, t)
    odd = q.clone()
    odd[0, 1, 5], odd[new - 1, 2, 63] = math.nan, -math.inf
    got = run(lib, pool, odd, [new], group, 0.125, t)
    hit = torch.zeros((new, group), dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[new - 1, 2] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit]) and not clean.isnan().any()
