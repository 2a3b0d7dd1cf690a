"""Cases for timing the language-model operators of libtcg: rotary positions, head norms with the rotation in the same
pass, the 8-bit key/value cache and the attention that reads it.

Each case runs in two ways on the same state: as plain torch operations (`own` false), or through the library's entry
points (`own` true). Lengths are fixed by the case; values, pages and positions come from the seed.

The cache holds pages of 64 tokens. K codes are [n_pages, n_kv, 64, d], V codes [n_pages, n_kv, d, 64] (int8), with one
scale per (page, head) each: value = code * scale. Pages that no sequence uses hold garbage codes and NaN scales, as
freed memory does.
"""
import ctypes
import math
import os
import random
import sys

import numpy as np
import torch

own = False

PAGE = 64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ------------------------------------------------------------------ cases

def _rope(name, t, n_tok, n_head, d, n_rot, layout, base, scaling, factor, ctx, norm=False, n_kv=0):
    return {"name": name, "op": "norm_rope" if norm else "rope", "type": t, "n_tok": n_tok, "n_head": n_head,
            "n_kv": n_kv, "d": d, "n_rot": n_rot, "layout": layout, "base": base, "scaling": scaling,
            "factor": factor, "ctx": ctx}


def _append(name, t, n_seq, max_new, max_kv, n_kv, d):
    return {"name": name, "op": "append", "type": t, "n_seq": n_seq, "max_new": max_new, "max_kv": max_kv,
            "n_kv": n_kv, "d": d}


def _attn(name, t, n_seq, max_new, max_kv, n_head, n_kv, d, causal=True, window=0):
    return {"name": name, "op": "attn", "type": t, "n_seq": n_seq, "max_new": max_new, "max_kv": max_kv,
            "n_head": n_head, "n_kv": n_kv, "d": d, "causal": causal, "window": window}


def listed():
    return [
        # one decoded token's queries and keys, rotated in place of the fp32 rows that the K-quant matvec writes
        _rope("rope_token", "f32", 1, 40, 128, 128, "interleaved", 500000.0, "bands", 8.0, 8192),
        # a long document's rows, a part of each head, positions far beyond the trained context
        _rope("rope_far", "bf16", 6001, 36, 128, 64, "half", 10000.0, "yarn", 32.0, 4096),
        # one decode step of 48 sequences: head norms and rotation of 32 query and 8 key heads
        _rope("norm_rope_step", "bf16", 48, 32, 128, 128, "half", 1000000.0, "none", 1.0, 32768, norm=True, n_kv=8),
        # a prompt's rows, fp32 as the GEMM leaves them
        _rope("norm_rope_prompt", "f32", 4096, 32, 128, 128, "half", 1000000.0, "linear", 4.0, 32768, norm=True, n_kv=8),
        # a decode step writes one token of each of 33 sequences into pages that are partly full
        _append("append_step", "f32", 33, 1, 4096, 8, 128),
        # five prompts of different lengths written at once, some behind a cached prefix
        _append("append_prompt", "f16", 5, 2048, 5000, 8, 128),
        # one conversation, one token, a few hundred tokens of context: latency
        _attn("attn_token", "f32", 1, 1, 513, 32, 8, 128),
        # a serving batch's decode step, contexts of all lengths up to 8192
        _attn("attn_serve", "bf16", 64, 1, 8192, 32, 8, 128),
        # one token against a very long context
        _attn("attn_long", "f16", 1, 1, 131071, 32, 8, 128),
        # a whole prompt, causal, fp32
        _attn("attn_prompt", "f32", 1, 4096, 4096, 32, 8, 128),
        # chunks of prompts behind cached prefixes, smaller heads
        _attn("attn_chunk", "bf16", 3, 700, 6100, 16, 4, 64),
        # a few drafted tokens of each of 17 sequences to verify, a sliding window, one key head
        _attn("attn_draft", "f16", 17, 5, 3001, 10, 1, 96, True, 1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    t = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["rope", "norm_rope", "append", "attn", "attn", "attn"])
    if op in ("rope", "norm_rope"):
        d = rng.choice([32, 64, 80, 96, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 7])
        return {k: v for k, v in _rope(
            "", t, _log(rng, 1, 4096), heads, d, rng.choice([d, d // 2, 16]), rng.choice(["interleaved", "half"]),
            rng.choice([10000.0, 500000.0]), rng.choice(["none", "linear", "yarn", "bands"]),
            rng.choice([2.0, 8.0, 32.0]), rng.choice([2048, 8192]), op == "norm_rope",
            kv if op == "norm_rope" else 0).items() if k != "name"}
    d = rng.choice([32, 64, 80, 96, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == "append":
        n_seq = _log(rng, 1, 64)
        new = rng.choice([1, 1, _log(rng, 1, max(2, 8192 // n_seq))])
        return {k: v for k, v in _append("", t, n_seq, new, new + _log(rng, 1, 4000), kv, d).items() if k != "name"}
    n_seq = _log(rng, 1, 64)
    heads = kv * rng.choice([1, 2, 4, 5, 8])
    new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, max(17, 2048 // n_seq))])
    most = min(65536, 200_000_000 // (n_seq * new * heads), 400_000 // n_seq)
    window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
    causal = rng.random() < 0.85
    return {k: v for k, v in _attn("", t, n_seq, new, new + _log(rng, 1, max(2, most)), heads, kv, d, causal,
                                   window if causal else 0).items() if k != "name"}


def _lengths(case):
    """New tokens and cached tokens (the new ones included) of each sequence: the first one has the most of both."""
    r = random.Random("%(n_seq)d %(max_new)d %(max_kv)d" % case)
    new, kv = [case["max_new"]], [case["max_kv"]]
    while len(new) < case["n_seq"]:
        new.append(r.randint(1, case["max_new"]))
        kv.append(new[-1] + r.randint(0, max(0, case["max_kv"] - new[-1])))
    return new, kv


def _pairs(case):
    """Visible (query, key) pairs, and keys that some query sees, over all sequences."""
    pairs = keys = 0
    for n, kv in zip(*_lengths(case)):
        if not case["causal"]:
            pairs += n * kv
            keys += kv
            continue
        w = case["window"] or kv
        pos = np.arange(kv - n, kv)
        pairs += int((np.minimum(pos + 1, w)).sum())
        keys += kv - max(0, kv - n - w + 1)
    return pairs, keys


def work(case):
    size, d = SIZE[case["type"]], case["d"]
    if case["op"] in ("rope", "norm_rope"):
        n = case["n_tok"] * (case["n_head"] + case["n_kv"]) * d
        return {"bytes": 2 * n * size + 4 * case["n_tok"], "flops": (7 if case["n_kv"] else 3) * n}
    if case["op"] == "append":
        new, kv = _lengths(case)
        wide = case["n_kv"] * d * 2
        back = sum(k - (k - n) // PAGE * PAGE for n, k in zip(new, kv))     # tokens of the pages written, read back
        return {"bytes": sum(new) * wide * (size + 1) + back * wide * 5, "flops": 4 * sum(new) * wide + back * wide}
    pairs, keys = _pairs(case)
    n = sum(_lengths(case)[0])
    return {"bytes": 2 * n * case["n_head"] * d * size + keys * case["n_kv"] * (2 * d + 8 / PAGE),
            "flops": 4 * pairs * case["n_head"] * d}


# ------------------------------------------------------------------ states

def _turns(case):
    """Revolutions per position of each rotated pair, and the factor on the rotated values (64 bits)."""
    half = case["n_rot"] // 2
    freq = case["base"] ** (-np.arange(half) * 2.0 / case["n_rot"])
    s, ctx, m = case["factor"], case["ctx"], 1.0
    if case["scaling"] == "linear":
        freq = freq / s
    elif case["scaling"] == "yarn":
        # between the pair that turns 32 times over the trained context and the one that turns once: from kept to stretched
        def at(turns):
            return case["n_rot"] * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))
        low, high = max(0.0, math.floor(at(32.0))), min(case["n_rot"] - 1.0, math.ceil(at(1.0)))
        ramp = np.clip((np.arange(half) - low) / max(high - low, 0.001), 0, 1)
        freq = freq * (1 - ramp) + freq / s * ramp
        m = 0.1 * math.log(s) + 1
    elif case["scaling"] == "bands":
        # waves longer than the context are stretched, those shorter than a quarter of it kept, between them both by turns
        wave = 2 * math.pi / freq
        mix = np.clip((ctx / wave - 1.0) / (4.0 - 1.0), 0, 1)
        freq = freq * mix + freq / s * (1 - mix)
    return freq / (2 * math.pi), m


def _values(g, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)


def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "roofline.c_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tcg
    tcg.init(torch.cuda.current_device())
    return tcg


def _rope_state(case, g):
    dt, d = TYPES[case["type"]], case["d"]
    n, h, kv = case["n_tok"], case["n_head"], case["n_kv"]
    far = int(case["ctx"] * case["factor"])
    first = torch.randint(0, far, (1,), generator=g, device="cuda")
    s = {"case": case, "pos": ((first + torch.arange(n, device="cuda")) % far).to(torch.int32),
         "x": _values(g, (n, (h + kv) * d), dt)}                # rows as a fused projection leaves them
    turns, m = _turns(case)
    s["turns"], s["mscale"] = torch.tensor(turns, device="cuda"), m
    s["out"] = torch.empty_like(s["x"])
    if kv:
        s["wq"], s["wk"] = (_values(g, (d,), torch.float32, 0.1) + 1 for _ in range(2))
    if own:
        tcg = _library()
        r = tcg.Rope()
        lib = tcg.lib()
        tcg.check(lib.tcg_rope_init(ctypes.byref(r), d, case["n_rot"], int(case["layout"] == "half"), case["base"]))
        if case["scaling"] == "linear":
            tcg.check(lib.tcg_rope_scale_linear(ctypes.byref(r), case["factor"]))
        elif case["scaling"] == "yarn":
            tcg.check(lib.tcg_rope_scale_yarn(ctypes.byref(r), case["factor"], case["ctx"], 32.0, 1.0, 0.0))
        elif case["scaling"] == "bands":
            tcg.check(lib.tcg_rope_scale_bands(ctypes.byref(r), case["factor"], case["ctx"], 1.0, 4.0))
        s["tcg"], s["rope"] = tcg, r
    return s


def _cache_state(case, g, seed):
    """A page pool with every sequence's cached tokens in it, and the step's rows."""
    new, kv = _lengths(case)
    n_kv, d = case["n_kv"], case["d"]
    pages = [-(-k // PAGE) for k in kv]
    n_pages = sum(pages) + 2
    k = (torch.randn((n_pages, n_kv, PAGE, d), generator=g, device="cuda") * 36).round_().clamp_(-127, 127).to(torch.int8)
    v = (torch.randn((n_pages, n_kv, d, PAGE), generator=g, device="cuda") * 36).round_().clamp_(-127, 127).to(torch.int8)
    ks, vs = (torch.exp(torch.randn((n_pages, n_kv), generator=g, device="cuda") * 0.15) * 0.0276 for _ in range(2))
    order = np.random.RandomState(seed).permutation(n_pages)
    ld = max(pages)
    table = np.full((case["n_seq"], ld), -1, np.int32)          # behind a sequence's last page: nothing
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    ks[order[at:]], vs[order[at:]] = float("nan"), float("nan")  # pages of nobody
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    s = {"case": case, "k": k, "v": v, "ks": ks, "vs": vs, "n_tok": int(start[-1]),
         "start": torch.from_numpy(start).cuda(), "kv": torch.tensor(kv, dtype=torch.int32, device="cuda"),
         "table": torch.from_numpy(table).cuda()}
    if own:
        tcg = _library()
        s["tcg"] = tcg
        s["cache"] = tcg.Kv8(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), n_pages, n_kv, d)
        s["step"] = tcg.Kv8Step(s["start"].data_ptr(), s["kv"].data_ptr(), s["table"].data_ptr(), ld, case["n_seq"],
                                s["n_tok"], case["max_new"], case["max_kv"])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("rope", "norm_rope"):
        return _rope_state(case, g)
    s = _cache_state(case, g, seed)
    dt, d = TYPES[case["type"]], case["d"]
    if case["op"] == "attn":
        s["q"] = _values(g, (s["n_tok"], case["n_head"], d), dt, 1.5)
        s["out"] = torch.empty_like(s["q"])
        return s
    s["new_k"], s["new_v"] = (_values(g, (s["n_tok"], case["n_kv"], d), dt) for _ in range(2))
    # the pages that the step writes are read back, as a program does that moves or checks them
    new, kv = _lengths(case)
    back = [b - (b - a) // PAGE * PAGE for a, b in zip(new, kv)]
    rows = np.concatenate([[0], np.cumsum(back)]).astype(np.int32)
    s["back"], s["n_back"], s["max_back"] = torch.from_numpy(rows).cuda(), int(rows[-1]), max(back)
    s["out_k"], s["out_v"] = (torch.empty((s["n_back"], case["n_kv"], d), device="cuda") for _ in range(2))
    if own:
        st = s["step"]
        s["back_step"] = s["tcg"].Kv8Step(s["back"].data_ptr(), st.kv_len, st.table, st.table_ld, st.n_seq,
                                          s["n_back"], s["max_back"], st.max_kv)
    return s


# ------------------------------------------------------------------ plain forms

def _angles(s):
    t = s["pos"].double()[:, None] * s["turns"]                  # far positions need the 64 bits
    a = (t - torch.round(t)) * (2 * math.pi)
    return (torch.cos(a) * s["mscale"]).float()[:, None], (torch.sin(a) * s["mscale"]).float()[:, None]


def _rotated(x, cos, sin, n_rot, layout):
    half = n_rot // 2
    if layout == "half":
        a, b = x[..., :half], x[..., half:n_rot]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., n_rot:]], -1)
    a, b = x[..., 0:n_rot:2], x[..., 1:n_rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), x[..., n_rot:]], -1)


def _run_rope(s):
    c = s["case"]
    x = s["x"].float().view(c["n_tok"], c["n_head"] + c["n_kv"], c["d"])
    cos, sin = _angles(s)
    if c["n_kv"]:
        w = torch.cat([s["wq"].expand(c["n_head"], -1), s["wk"].expand(c["n_kv"], -1)])
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    return _rotated(x, cos, sin, c["n_rot"], c["layout"]).to(s["out"].dtype).view(c["n_tok"], -1)


def _rows(start, kv, n):
    """Of each of n rows dealt out by `start`: its sequence and its token's position (the rows are the sequence's last)."""
    i = torch.arange(n, device="cuda", dtype=torch.int32)
    b = torch.bucketize(i, start[1:], right=True)
    return b, (kv[b] - (start[b + 1] - start[b]) + (i - start[b])).long()


def _append_codes(s, x, codes, scale, tokens_last):
    """Writes x's rows into codes / scale: a page's scale grows to its largest magnitude / 127, older codes follow it."""
    c = s["case"]
    b, pos = _rows(s["start"], s["kv"], s["n_tok"])
    page, slot = s["table"][b, pos // PAGE].long(), pos % PAGE
    x = x.float()
    step = x.abs().amax(-1) / torch.full((1,), 127.0, device="cuda")     # [rows, heads]; by a plain number torch multiplies
    # the pages that the step touches: of each sequence as many as its longest run of new tokens can reach
    first = s["kv"].long() - (s["start"][1:] - s["start"][:-1]).long()
    reach = torch.arange((c["max_new"] + PAGE - 1) // PAGE + 1, device="cuda")
    at = first[:, None] // PAGE + reach
    used = at * PAGE < s["kv"].long()[:, None]
    slots = (first[:, None] - at * PAGE).clamp(0, PAGE)          # older tokens in each of these pages
    p = s["table"].gather(1, at.clamp(max=s["table"].shape[1] - 1)).long()[used]
    old_n = slots[used]
    grown = torch.zeros_like(scale).index_reduce_(0, page, step, "amax", include_self=True)[p]
    old = torch.where((old_n > 0)[:, None], scale[p], torch.zeros((), device="cuda"))
    now = torch.maximum(old, grown)
    ratio = torch.where(now > 0, old / now, torch.zeros((), device="cuda"))
    moved = torch.round(codes[p].float() * ratio[:, :, None, None]).to(torch.int8)
    token = torch.arange(PAGE, device="cuda")
    older = token < old_n[:, None]
    older = older[:, None, None, :] if tokens_last else older[:, None, :, None]
    codes[p] = torch.where(older, moved, codes[p])
    scale[p] = now
    fine = scale[page]
    q = torch.where(fine[..., None] > 0, torch.round(x / fine[..., None]), torch.zeros((), device="cuda"))
    q = q.clamp(-127, 127).to(torch.int8)
    if tokens_last:
        codes[page, :, :, slot] = q
    else:
        codes[page, :, slot, :] = q


def _read_back(s, codes, scale, tokens_last):
    b, pos = _rows(s["back"], s["kv"], s["n_back"])
    page, slot = s["table"][b, pos // PAGE].long(), pos % PAGE
    x = codes[page, :, :, slot] if tokens_last else codes[page, :, slot, :]
    return x.float() * scale[page][..., None]


def _run_append(s):
    _append_codes(s, s["new_k"], s["k"], s["ks"], False)
    _append_codes(s, s["new_v"], s["v"], s["vs"], True)
    return _read_back(s, s["k"], s["ks"], False), _read_back(s, s["v"], s["vs"], True)


def _run_attn(s):
    c = s["case"]
    n_seq, n_kv, d, group = c["n_seq"], c["n_kv"], c["d"], c["n_head"] // c["n_kv"]
    page = s["table"].clamp(min=0).long()
    used = (s["table"] >= 0)[:, :, None]
    zero = torch.zeros((), device="cuda")
    k = s["k"][page].float() * torch.where(used, s["ks"][page], zero)[..., None, None]     # [seq, pages, heads, 64, d]
    v = s["v"][page].float() * torch.where(used, s["vs"][page], zero)[..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, -1, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(n_seq, n_kv, -1, d)
    # queries in rows of equal number, [seq, kv heads, group * tokens, d]
    i = torch.arange(c["max_new"], device="cuda")
    new = (s["start"][1:] - s["start"][:-1]).long()
    row = (s["start"][:-1].long()[:, None] + i).clamp(max=s["n_tok"] - 1)
    q = s["q"].float()[row].view(n_seq, -1, n_kv, group, d).permute(0, 2, 3, 1, 4).reshape(n_seq, n_kv, -1, d)
    score = (q @ k.transpose(-1, -2)).view(n_seq, n_kv, group, c["max_new"], -1) / math.sqrt(d)
    key = torch.arange(k.shape[2], device="cuda")
    kv = s["kv"].long()[:, None, None]
    see = key < kv
    if c["causal"]:
        pos = (kv[..., 0] - new[:, None] + i)[..., None]
        see = see & (key <= pos)
        if c["window"]:
            see = see & (key > pos - c["window"])
    score = score.masked_fill(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, zero))
    total = p.sum(-1, keepdim=True)
    o = (p.view(n_seq, n_kv, -1, k.shape[2]) @ v).view(n_seq, n_kv, group, c["max_new"], d)
    o = torch.where(total > 0, o / total, zero).permute(0, 3, 1, 2, 4).reshape(n_seq, c["max_new"], n_kv * group, d)
    b, _ = _rows(s["start"], s["kv"], s["n_tok"])
    at = torch.arange(s["n_tok"], device="cuda") - s["start"][b].long()
    return o[b, at].to(s["out"].dtype)


# ------------------------------------------------------------------ one pass

def run(s):
    c = s["case"]
    if not own:
        return {"rope": _run_rope, "norm_rope": _run_rope, "append": _run_append, "attn": _run_attn}[c["op"]](s)
    tcg, t = s["tcg"], GGML[c["type"]]
    lib = tcg.lib()
    if c["op"] == "rope":
        ld = c["n_head"] * c["d"]
        tcg.check(lib.tcg_rope(s["out"].data_ptr(), s["x"].data_ptr(), s["pos"].data_ptr(), ctypes.byref(s["rope"]),
                               c["n_tok"], c["n_head"], ld, ld, t))
        return s["out"]
    if c["op"] == "norm_rope":
        ld, k_at = (c["n_head"] + c["n_kv"]) * c["d"], c["n_head"] * c["d"] * SIZE[c["type"]]
        x, out = s["x"].data_ptr(), s["out"].data_ptr()
        tcg.check(lib.tcg_qk_norm_rope(out, out + k_at, x, x + k_at, s["wq"].data_ptr(), s["wk"].data_ptr(), EPS,
                                       s["pos"].data_ptr(), ctypes.byref(s["rope"]), c["n_tok"], c["n_head"], c["n_kv"],
                                       ld, ld, ld, ld, t))
        return s["out"]
    cache, step = ctypes.byref(s["cache"]), ctypes.byref(s["step"])
    if c["op"] == "append":
        ld = c["n_kv"] * c["d"]
        tcg.check(lib.tcg_kv8_append(cache, step, s["new_k"].data_ptr(), s["new_v"].data_ptr(), ld, ld, t))
        tcg.check(lib.tcg_kv8_read(s["out_k"].data_ptr(), s["out_v"].data_ptr(), cache, ctypes.byref(s["back_step"]),
                                   ld, ld, GGML["f32"]))
        return s["out_k"], s["out_v"]
    ld = c["n_head"] * c["d"]
    tcg.check(lib.tcg_kv8_attention(s["out"].data_ptr(), s["q"].data_ptr(), cache, step, c["n_head"], ld, ld,
                                    1.0 / math.sqrt(c["d"]), c["causal"], c["window"], t))
    return s["out"]


# ------------------------------------------------------------------ in 64 bits

def _exact_rope(s):
    c = s["case"]
    n, heads, d, n_rot = c["n_tok"], c["n_head"] + c["n_kv"], c["d"], c["n_rot"]
    x = s["x"].double().view(n, heads, d)
    if c["n_kv"]:
        x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS)
        x[:, :c["n_head"]] *= s["wq"].double()
        x[:, c["n_head"]:] *= s["wk"].double()
    turns, m = _turns(c)
    out = x.clone()
    for i in range(n_rot // 2):
        lo, hi = (i, i + n_rot // 2) if c["layout"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.full((n,), m, dtype=torch.float64, device="cuda"),
                           torch.remainder(s["pos"].double() * turns[i], 1.0) * (2 * math.pi))[:, None]
        z = torch.complex(x[..., lo], x[..., hi]) * turn
        out[..., lo], out[..., hi] = z.real, z.imag
    return out.view(n, heads * d)


def _exact_append(s, x, codes, scale, tokens_last):
    """The cache's values after the step, page by page. Scales, quotients and codes are rounded to 32 bits as the format
    says, from results in 64 bits."""
    start, kv, table = s["start"].tolist(), s["kv"].tolist(), s["table"].tolist()
    x = x.double()
    back = []
    for b in range(len(kv)):
        n = start[b + 1] - start[b]
        begin = kv[b] - n
        for p in range(begin // PAGE, -(-kv[b] // PAGE)):
            lo, hi = max(begin, p * PAGE), min(kv[b], (p + 1) * PAGE)
            rows = x[start[b] + lo - begin:start[b] + hi - begin]
            page, older = table[b][p], lo - p * PAGE
            sc = (rows.abs().amax(dim=(0, 2)) / 127).float().double()
            have = codes[page].double()                          # [heads, 64, d] or [heads, d, 64]
            have = (have.transpose(1, 2) if tokens_last else have)[:, :older]
            if older:
                was = scale[page].double()
                sc = torch.maximum(sc, was)
                have = (have * (was / sc).float().double()[:, None, None]).float().double().round()
            q = (rows / sc[None, :, None]).float().double().round().clamp(-127, 127)
            back.append(torch.cat([have.transpose(0, 1), q]) * sc[None, :, None])
    return torch.cat(back)


def _exact_attn(s):
    c = s["case"]
    group, d = c["n_head"] // c["n_kv"], c["d"]
    start, kv = s["start"].tolist(), s["kv"].tolist()
    out = torch.zeros((s["n_tok"], c["n_head"], d), dtype=torch.float64, device="cuda")
    for b in range(c["n_seq"]):
        n, pages = start[b + 1] - start[b], s["table"][b, :-(-kv[b] // PAGE)].long()
        pos = torch.arange(kv[b] - n, kv[b], device="cuda")[:, None]
        key = torch.arange(kv[b], device="cuda")[None]
        hide = torch.zeros((n, kv[b]), dtype=torch.bool, device="cuda")
        if c["causal"]:
            hide |= key > pos
            if c["window"]:
                hide |= pos - key >= c["window"]
        for h in range(c["n_kv"]):
            k = (s["k"][pages, h].double() * s["ks"][pages, h].double()[:, None, None]).reshape(-1, d)[:kv[b]]
            v = (s["v"][pages, h].double() * s["vs"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:kv[b]]
            for j in range(h * group, (h + 1) * group):
                w = s["q"][start[b]:start[b + 1], j].double() @ k.T * d ** -0.5
                out[start[b]:start[b + 1], j] = torch.softmax(w.masked_fill_(hide, -math.inf), -1) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rope", "norm_rope"):
        return _exact_rope(s)
    if case["op"] == "append":
        return (_exact_append(s, s["new_k"], s["k"], s["ks"], False), _exact_append(s, s["new_v"], s["v"], s["vs"], True))
    return _exact_attn(s)
