"""Cases for timing the microscaled operators of libtcg: quantisation to 4 and 8 bits in blocks of 32 with a power of two
each, the residual's addition with the root-mean-square norm whose rows come out in 8 bits, and the product of such rows
with weights held in 4 bits.

Each case runs in two ways on the same state: as plain torch operations (`own` false), or through the library's entry
points (`own` true). Sizes are fixed by the case; values come from the seed.

A matrix [rows, cols] is held as
  codes  [rows, P] in 4 bits (E2M1, two in a byte, the even column in the low half) or 8 bits (E4M3), P = cols rounded up
         to 128; columns behind the last are 0;
  scales one byte s for 32 columns, value = code * 2^(s - 127), s = 255: the block is NaN. The bytes of 128 rows and 128
         columns stand together: row r, block b at ((r / 128) * (P / 128) + b / 4) * 512 + r % 32 * 16 + r / 32 % 4 * 4 + b % 4.
A block's scale is 2^(floor(log2(its largest magnitude)) - m), m = 2 (E2M1) or 8 (E4M3); codes are the nearest values, ties
to the even code, at most the format's largest (6 or 448).
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
# exponent of the largest binade, bits of the mantissa, smallest normal exponent, largest value
FORMAT = {4: (2, 1, 0, 6.0), 8: (8, 3, -6, 448.0)}


# ------------------------------------------------------------------ cases

def _norm(name, t, rows, cols, bits, residual=True, pad=0):
    return {"name": name, "op": "norm", "type": t, "rows": rows, "cols": cols, "bits": bits, "residual": residual, "pad": pad}


def _quant(name, t, rows, cols, bits, pad=0):
    return {"name": name, "op": "quant", "type": t, "rows": rows, "cols": cols, "bits": bits, "pad": pad}


def _linear(name, t, rows, cols, outs, bits, bias=False):
    return {"name": name, "op": "linear", "type": t, "rows": rows, "cols": cols, "outs": outs, "bits": bits, "bias": bias}


def listed():
    return [
        # one decoded token between two blocks of a model: residual, norm, 8-bit row for the next product
        _norm("norm_token", "f32", 1, 4096, 8),
        # a serving batch's decode step
        _norm("norm_step", "bf16", 64, 4096, 8),
        # a prompt's rows, fp32 as the GEMM leaves them
        _norm("norm_prompt", "f32", 4096, 4096, 8),
        # the last norm before the logits: rows of an odd width inside wider ones, in their own type, no addition
        _norm("norm_last", "f16", 777, 2571, 0, False, 5),
        # a weight matrix taken from its GGUF tensor into 4 bits
        _quant("quant_weights", "f32", 14336, 4096, 4),
        # the activations of a step's wide layer
        _quant("quant_rows", "bf16", 64, 14336, 8),
        # rows whose last block is not whole, inside wider rows
        _quant("quant_ragged", "f16", 1501, 4100, 4, 3),
        # one decoded token through the up projection, fp32 result
        _linear("mx_token", "f32", 1, 4096, 14336, 8),
        # a decode step of 64 sequences through the down projection
        _linear("mx_step", "bf16", 64, 14336, 4096, 8),
        # a prompt through the up projection, rows in 4 bits too
        _linear("mx_prompt", "bf16", 4096, 4096, 14336, 4),
        # a chunk of a prompt through the down projection, rows in 8 bits, fp32 result
        _linear("mx_prompt_f32", "f32", 2048, 14336, 4096, 8),
        # odd sizes all over, with a bias
        _linear("mx_ragged", "f16", 333, 1100, 5003, 4, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    t = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["norm", "quant", "linear", "linear"])
    cols = rng.choice([_log(rng, 32, 14336), 32 * _log(rng, 1, 448), 256 * _log(rng, 1, 56)])
    pad = rng.choice([0, 0, 0, _log(rng, 1, 64)])
    if op == "norm":
        c = _norm("", t, _log(rng, 1, 4096), cols, rng.choice([0, 4, 8, 8]), rng.random() < 0.8, pad)
    elif op == "quant":
        c = _quant("", t, _log(rng, 1, 14336), min(cols, 8192), rng.choice([4, 4, 8]), pad)
    else:
        rows, outs = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 4096), _log(rng, 64, 4096)]), _log(rng, 16, 16384)
        while rows * cols * outs > 4096 * 4096 * 14336:
            rows = max(1, rows // 2)
        c = _linear("", t, rows, cols, outs, rng.choice([4, 8]), rng.random() < 0.3)
    del c["name"]
    return c


def _held(rows, cols, bits):
    """Bytes of a matrix's codes and scales."""
    return rows * cols * bits / 8 + rows * -(-cols // 32)


def work(case):
    rows, cols, bits, size = case["rows"], case["cols"], case["bits"], SIZE[case["type"]]
    n = rows * cols
    # what is held in few bits is written once, and read back once as bf16 values
    back = 2 * _held(rows, cols, bits) + 2 * n if bits else 0
    if case["op"] == "norm":
        wide = (3 if case["residual"] else 1) * size + (0 if bits else size)
        return {"bytes": wide * n + 4 * cols + back, "flops": 5 * n}
    if case["op"] == "quant":
        return {"bytes": size * n + back, "flops": 3 * n}
    outs = case["outs"]
    return {"bytes": _held(rows, cols, bits) + _held(outs, cols, 4) + size * rows * outs + (4 * outs if case["bias"] else 0),
            "flops": 2 * rows * cols * outs}


# ------------------------------------------------------------------ the format in plain form

def _power(e):
    """2^e of whole numbers e, in 64 bits and exactly: by the exponent's own bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantised(v, bits):
    """v [rows, cols] -> multiples of each block's scale [rows, blocks, 32] and scale bytes [rows, blocks]."""
    top, mant, low, most = FORMAT[bits]
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % 32)).view(rows, -1, 32)
    largest = v.abs().amax(-1)
    fine = torch.isfinite(largest)
    _, e = torch.frexp(torch.where(fine, largest, torch.zeros_like(largest)))
    s = torch.where(largest > 0, (e - 1 - top).clamp(-127, 127), torch.full_like(e, -127))
    q = v.double() * _power(-s)[..., None]
    _, e = torch.frexp(q)
    step = _power((e - 1).clamp(min=low) - mant)
    q = (torch.round(q / step) * step).clamp(-most, most)
    q = torch.where(fine[..., None], q, torch.zeros_like(q))
    return q, torch.where(fine, s + 127, torch.full_like(s, 255)).to(torch.uint8)


def _values(q, scale, cols):
    """Multiples and scale bytes as bf16 values, which hold them exactly."""
    p = torch.where(scale == 255, torch.full((), math.nan, dtype=torch.float64, device=q.device), _power(scale.int() - 127))
    return (q.double() * p[..., None]).flatten(1)[:, :cols].to(torch.bfloat16)


def _codes(q, bits):
    """[rows, blocks, 32] multiples as codes [rows, P * bits / 8] of bytes."""
    q = q.flatten(1)
    q = torch.nn.functional.pad(q, (0, -q.shape[1] % 128)).float()
    if bits == 8:
        return q.to(torch.float8_e4m3fn).view(torch.uint8)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    c = torch.bucketize(q.abs(), grid).to(torch.uint8) + 8 * torch.signbit(q).to(torch.uint8)
    return (c[:, 0::2] + 16 * c[:, 1::2]).contiguous()


def _tiled(scale):
    """Scale bytes [rows, blocks] in the order that they are held in."""
    rows, blocks = scale.shape
    s = torch.nn.functional.pad(scale, (0, -blocks % 4, 0, -rows % 128))
    return s.view(s.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _decoded(m):
    """A held matrix as fp32 values [rows, cols]."""
    rows, cols, bits = m["rows"], m["cols"], m["bits"]
    if bits == 8:
        q = m["codes"].view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
        q = table[torch.stack([m["codes"] & 15, m["codes"] >> 4], -1).flatten(1).int()]
    s = m["scales"].view(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)[:rows]
    p = torch.where(s == 255, torch.full((), math.nan, device="cuda"), _power(s.int() - 127).float())
    return (q.view(rows, -1, 32) * p[..., None]).flatten(1)[:, :cols]


# ------------------------------------------------------------------ states

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _matrix(v, bits):
    q, s = _quantised(v, bits)
    return {"rows": v.shape[0], "cols": v.shape[1], "bits": bits, "codes": _codes(q, bits), "scales": _tiled(s)}


def _room(rows, cols, bits):
    wide = -(-cols // 128) * 128
    return {"rows": rows, "cols": cols, "bits": bits,
            "codes": torch.empty((rows, wide * bits // 8), dtype=torch.uint8, device="cuda"),
            "scales": torch.empty(-(-rows // 128) * wide * 4, dtype=torch.uint8, device="cuda")}


def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "roofline.c_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tcg
    tcg.init(torch.cuda.current_device())
    return tcg


def _activations(g, rows, cols):
    """Rows of unlike sizes with a few large columns, as a model's hidden states have them."""
    wide = torch.exp(_randn(g, cols) * 0.3) * torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    return _randn(g, rows, cols) * wide * torch.exp(_randn(g, rows, 1) * 0.2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows, cols, bits = TYPES[case["type"]], case["rows"], case["cols"], case["bits"]
    s = {"case": case}
    if case["op"] == "linear":
        s["x"] = _matrix(_activations(g, rows, cols), bits)
        s["w"] = _matrix(_randn(g, case["outs"], cols) * 0.02, 4)
        s["bias"] = _randn(g, case["outs"]) if case["bias"] else None
        s["y"] = torch.empty((rows, case["outs"]), dtype=dt, device="cuda")
    else:
        wide = cols + case["pad"]
        s["x"] = _activations(g, rows, wide).to(dt)
        if bits:
            s["mx"], s["back"] = _room(rows, cols, bits), torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
        if case["op"] == "norm":
            s["w"] = _randn(g, cols) * 0.1 + 1
            s["r"] = (_randn(g, rows, wide) * 0.5).to(dt) if case["residual"] else None
            s["h"] = torch.empty((rows, cols), dtype=dt, device="cuda") if case["residual"] else None
            s["y"] = None if bits else torch.empty((rows, cols), dtype=dt, device="cuda")
    if own:
        s["tcg"] = _library()
        for name in ("x", "w", "mx"):
            m = s.get(name)
            if isinstance(m, dict):
                m["held"] = s["tcg"].Mx(m["codes"].data_ptr(), m["scales"].data_ptr(), m["rows"], m["cols"], m["bits"])
    return s


# ------------------------------------------------------------------ plain forms

def _run_norm(s):
    c = s["case"]
    h = s["x"][:, :c["cols"]]
    if c["residual"]:
        h = (h.float() + s["r"][:, :c["cols"]].float()).to(h.dtype)
    v = h.double() if c["bits"] else h.float()                   # codes next to a border need the 64 bits
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * s["w"]
    out = [h] if c["residual"] else []
    if c["bits"]:
        return out + [_values(*_quantised(y, c["bits"]), c["cols"])]
    return out + [y.to(h.dtype)]


def _run_quant(s):
    c = s["case"]
    return [_values(*_quantised(s["x"][:, :c["cols"]].float(), c["bits"]), c["cols"])]


def _run_linear(s):
    y = _decoded(s["x"]) @ _decoded(s["w"]).T
    if s["bias"] is not None:
        y = y + s["bias"]
    return [y.to(s["y"].dtype)]


# ------------------------------------------------------------------ one pass

def _at(t):
    return None if t is None else t.data_ptr()


def run(s):
    c = s["case"]
    if not own:
        return {"norm": _run_norm, "quant": _run_quant, "linear": _run_linear}[c["op"]](s)
    tcg, t = s["tcg"], GGML[c["type"]]
    lib = tcg.lib()
    if c["op"] == "linear":
        tcg.check(lib.tcg_mx_linear(s["y"].data_ptr(), ctypes.byref(s["x"]["held"]), ctypes.byref(s["w"]["held"]), _at(s["bias"]),
                                    c["outs"], t))
        return [s["y"]]
    mx = ctypes.byref(s["mx"]["held"]) if c["bits"] else None
    ld, out = c["cols"] + c["pad"], []
    if c["op"] == "quant":
        tcg.check(lib.tcg_mx_quantize(mx, s["x"].data_ptr(), ld, t))
    else:
        tcg.check(lib.tcg_add_rms_norm(_at(s["h"]), _at(s["y"]), mx, s["x"].data_ptr(), _at(s["r"]), s["w"].data_ptr(), EPS,
                                       c["rows"], c["cols"], c["cols"], c["cols"], ld, ld, t))
        out = [o for o in (s["h"], s["y"]) if o is not None]
    if c["bits"]:
        # read back, as a program does that checks or unpacks them
        tcg.check(lib.tcg_mx_dequantize(s["back"].data_ptr(), mx, c["cols"], GGML["bf16"]))
        out.append(s["back"])
    return out


# ------------------------------------------------------------------ in 64 bits

def _nearest(v, bits):
    """Values of v [rows, cols] (64 bits) in the format, by search in the list of its codes' values."""
    top, mant, low, most = FORMAT[bits]
    grid = sorted({m * 2.0 ** (e - mant) for e in range(low, top + 1) for m in range(2 ** mant if e > low else 0, 2 ** (mant + 1))})
    grid = torch.tensor([x for x in grid if x <= most], dtype=torch.float64, device="cuda")
    powers = torch.tensor([2.0 ** e for e in range(-300, 301)], dtype=torch.float64, device="cuda")     # pow() may be off by a bit
    between = (grid[1:] + grid[:-1]) / 2
    rows, cols = v.shape
    out = torch.empty((rows, cols), dtype=torch.float64, device="cuda")
    for at in range(0, cols, 32):
        b = v[:, at:at + 32]
        big = b.abs().max(dim=1, keepdim=True).values
        e = torch.floor(torch.log2(big.clamp(2.0 ** -200, 2.0 ** 200))).long()
        e = e + (powers[e + 301] <= big).long() - (powers[e + 300] > big).long()
        scale = powers[(e - top).clamp(-127, 127) + 300]
        a = b.abs() / scale
        i = torch.searchsorted(between, a.contiguous())          # the middles below a
        tie = (i < between.numel()) & (between[i.clamp(max=between.numel() - 1)] == a) & (i % 2 == 1)
        near = torch.sign(b) * grid[i + tie.long()] * scale
        out[:, at:at + 32] = torch.where(torch.isfinite(big), near, math.nan)
    return out


def _unheld(m):
    """A held matrix's values in 64 bits, scales taken one block of columns at a time."""
    rows, cols, bits = m["rows"], m["cols"], m["bits"]
    raw = m["codes"].cpu().numpy()
    if bits == 4:
        raw = np.stack([raw & 15, raw >> 4], -1).reshape(rows, -1)
        sign, e, f = raw >> 3, (raw >> 1) & 3, raw & 1
        q = np.where(e == 0, f * 0.5, (1 + f * 0.5) * np.exp2(e - 1.0))
    else:
        sign, e, f = raw >> 7, (raw >> 3) & 15, raw & 7
        q = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8.0) * np.exp2(e - 7.0))
    q = torch.from_numpy(np.where(sign, -q, q)).cuda()
    wide = q.shape[1] // 128
    r = torch.arange(rows, device="cuda")
    for b in range(wide * 4):
        at = (r // 128 * wide + b // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + b % 4
        power = torch.from_numpy(np.ldexp(1.0, m["scales"][at].cpu().numpy().astype(np.int64) - 127)).cuda()
        q[:, b * 32:b * 32 + 32] *= power[:, None]
    return q[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    c, cols = case, case["cols"]
    if c["op"] == "linear":
        y = _unheld(s["x"]) @ _unheld(s["w"]).T
        return [y + s["bias"].double() if c["bias"] else y]
    x = s["x"][:, :cols].double()
    if c["op"] == "quant":
        return [_nearest(x, c["bits"])]
    out = []
    if c["residual"]:
        x = (x + s["r"][:, :cols].double()).to(s["x"].dtype).double()      # the row as it is written
        out = [x]
    y = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / cols + EPS) * s["w"].double()
    return out + [_nearest(y, c["bits"]) if c["bits"] else y]
