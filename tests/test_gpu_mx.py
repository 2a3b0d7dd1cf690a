"""Microscaled operators on the GPU against their formulas in 64 bits: quantisation (bytes compared exactly), values read
back, the residual's addition with the root-mean-square norm, the product, and a run of them together.

Tolerances are sums of the roundings each kernel makes, written beside them; u = 2^-24 is half a step of fp32.
"""
import ctypes as C
import math

import pytest
import torch

import tcg

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, tcg.F32), "f16": (torch.float16, tcg.F16), "bf16": (torch.bfloat16, tcg.BF16)}
U = 2.0 ** -24
TOP = {4: 2, 8: 8}                       # exponent of the largest value's binade


def half_step(dt):
    return torch.finfo(dt).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, spread=1.0):
    return (torch.randn(shape, generator=g, dtype=torch.float64) * spread).to(dtype).cuda()


@pytest.fixture()
def lib(gpu):
    """The library with a stream of its own: tests synchronise around calls."""
    L = tcg.lib()
    tcg.check(L.tcg_clear_device_error())
    yield L
    torch.cuda.synchronize()
    assert L.tcg_device_error() == 0


def call(fn, *args):
    torch.cuda.synchronize()
    tcg.check(fn(*args))
    torch.cuda.synchronize()


# ------------------------------------------------------------------ the format

def code_values(bits):
    """The value of each code without its sign."""
    mant, bias = (1, 1) if bits == 4 else (3, 7)
    v = []
    for c in range(1 << (bits - 1)):
        e, m = c >> mant, c & ((1 << mant) - 1)
        v.append(m * 2.0 ** (1 - bias - mant) if e == 0 else (1 + m / 2 ** mant) * 2.0 ** (e - bias))
    return torch.tensor(v[:8] if bits == 4 else v[:127], dtype=torch.float64, device="cuda")


POWERS = [2.0 ** e for e in range(-300, 301)]


def power(e):
    return torch.tensor(POWERS, dtype=torch.float64, device="cuda")[(e + 300).long()]


def quantised(v, bits):
    """v [rows, cols] in 64 bits -> codes [rows, wide] and scale bytes [rows, wide / 32], wide = cols up to 128s."""
    rows, cols = v.shape
    b = torch.nn.functional.pad(v, (0, -cols % 128)).view(rows, -1, 32)
    top = b.abs().amax(-1)
    fine = torch.isfinite(top)
    _, e = torch.frexp(torch.where(fine & (top > 0), top, torch.ones_like(top)))
    s = torch.where(top > 0, (e - 1 - TOP[bits]).clamp(-127, 127), torch.full_like(e, -127))
    a = b.abs() * power(-s)[..., None]
    grid = code_values(bits)
    mid = (grid[1:] + grid[:-1]) / 2
    i = torch.searchsorted(mid, a.contiguous())
    tie = (i < mid.numel()) & (mid[i.clamp(max=mid.numel() - 1)] == a) & (i % 2 == 1)
    code = (i + tie.long()) + (torch.signbit(b).long() << (bits - 1))
    return code.flatten(1), torch.where(fine, s + 127, torch.full_like(s, 255))


class Held:
    """A microscaled matrix in device memory, with bytes of 0xAB behind its codes and 0xCD where no scale is written."""

    def __init__(self, rows, cols, bits):
        self.rows, self.cols, self.bits = rows, cols, bits
        self.wide = -(-cols // 128) * 128
        n, m = tcg.lib().tcg_mx_code_bytes(rows, cols, bits), tcg.lib().tcg_mx_scale_bytes(rows, cols)
        assert n == rows * self.wide * bits // 8
        self.codes = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((m + 64,), 0xCD, dtype=torch.uint8, device="cuda")
        self.n, self.m = n, m

    def mx(self):
        return tcg.Mx(self.codes.data_ptr(), self.scales.data_ptr(), self.rows, self.cols, self.bits)

    def code(self):
        c = self.codes[:self.n].view(self.rows, -1).long()
        return c if self.bits == 8 else torch.stack([c & 15, c >> 4], -1).flatten(1)

    def scale(self):
        """[rows up to 128s, wide / 32]"""
        s = self.scales[:self.m].view(-(-self.rows // 128), self.wide // 128, 32, 4, 4)
        return s.permute(0, 3, 2, 1, 4).reshape(-(-self.rows // 128) * 128, -1).long()

    def put(self, code, scale):
        """Codes [rows, wide] and scale bytes [rows, wide / 32]; the scales of rows that there are not are NaN."""
        c = code.to(torch.uint8)
        self.codes[:self.n] = (c if self.bits == 8 else c[:, 0::2] + 16 * c[:, 1::2]).flatten()
        s = torch.full((-(-self.rows // 128) * 128, self.wide // 32), 255, dtype=torch.uint8, device="cuda")
        s[:self.rows] = scale.to(torch.uint8)
        self.scales[:self.m] = s.view(-1, 4, 32, self.wide // 128, 4).permute(0, 3, 2, 1, 4).flatten()
        return self

    def values(self):
        """[rows, cols] in 64 bits"""
        code, s, half = self.code(), self.scale()[:self.rows], 1 << (self.bits - 1)
        v = code_values(self.bits)[(code % half).clamp(max=126)] * torch.where(code >= half, -1.0, 1.0)
        v = v * torch.where(s == 255, torch.full((), math.nan, dtype=torch.float64, device="cuda"), power(s - 127)).repeat_interleave(32, 1)
        return v[:, :self.cols]

    def check(self, code, scale):
        """Whether exactly these are held: codes of NaN blocks aside, nothing else written."""
        fine = (scale != 255).repeat_interleave(32, 1)
        assert torch.equal(self.scale()[:self.rows], scale)
        assert (self.scale()[self.rows:] == 0xCD).all()
        assert torch.equal(self.code()[fine], code[fine])
        assert (self.codes[self.n:] == 0xAB).all() and (self.scales[self.m:] == 0xCD).all()


def random_held(g, rows, cols, bits, center, spread=3):
    """Codes of all values, scales 2^(center - spread .. center + spread)."""
    m = Held(rows, cols, bits)
    g = torch.Generator(device="cuda").manual_seed(int(torch.randint(1 << 30, (1,), generator=g)))
    code = torch.randint(0, 1 << bits, (rows, m.wide), generator=g, device="cuda")
    if bits == 8:
        code = torch.where(code % 128 == 127, code - 1, code)            # the format's NaN
    code[:, cols:] = 0
    return m.put(code, torch.randint(127 + center - spread, 128 + center + spread, (rows, m.wide // 32), generator=g, device="cuda"))


# ------------------------------------------------------------------ quantisation and back

def rows_of(v, pad, offset):
    """v inside an array whose rows are `pad` longer and whose first element is the offset-th: (array, view, pointer, stride)."""
    rows, cols = v.shape
    flat = torch.full((offset + rows * (cols + pad),), 7.0, dtype=v.dtype, device="cuda")
    view = flat[offset:].view(rows, cols + pad)[:, :cols]
    view.copy_(v)
    return flat, view, flat.data_ptr() + offset * v.element_size(), cols + pad


QUANTS = [  # rows, cols, pad, offset
    (1, 1, 0, 0), (1, 32, 0, 0), (3, 33, 0, 0), (1, 4096, 0, 0), (2, 127, 1, 0), (5, 130, 0, 3), (31, 260, 4, 0), (32, 256, 0, 8),
    (33, 257, 0, 1), (97, 1001, 3, 2), (130, 512, 8, 0), (300, 4100, 3, 0), (1, 20001, 0, 5), (129, 300, 2, 1), (4, 7, 0, 0),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cols,pad,offset", QUANTS)
def test_quantise_and_read_back(lib, rows, cols, pad, offset, t, bits):
    dt, code = TYPES[t]
    g = gen(rows + cols)
    x = randn(g, rows, cols, dtype=torch.float64) * torch.exp(randn(g, rows, 1, dtype=torch.float64) * 2)
    x = torch.where(torch.rand((rows, cols), generator=g).cuda() < 0.02, x * 1e-4, x).to(dt)
    flat, view, ptr, ld = rows_of(x, pad, offset)
    m = Held(rows, cols, bits)
    call(lib.tcg_mx_quantize, C.byref(m.mx()), ptr, ld, code)
    m.check(*quantised(x.double(), bits))
    # back, into rows of the same layout: every value exactly, rounded once to f16; what lies between stays
    for u, (du, cu) in TYPES.items():
        flat, view, ptr, ld = rows_of(torch.zeros((rows, cols), dtype=du, device="cuda"), pad, offset)
        call(lib.tcg_mx_dequantize, ptr, C.byref(m.mx()), ld, cu)
        assert torch.equal(view, m.values().to(du))
        assert (flat[:offset] == 7).all() and (flat[offset:].view(rows, -1)[:, cols:] == 7).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_quantise_at_borders(lib, bits):
    """Values in the middle between two codes, at powers of two, beyond the largest code, next to each of them."""
    grid = code_values(bits)
    mid = (grid[1:] + grid[:-1]) / 2
    top = 2.0 ** TOP[bits]
    near = torch.cat([grid, mid, torch.tensor([grid[-1] * 1.05, top * 2 - 0.01], dtype=torch.float64, device="cuda")])
    near = torch.cat([near, near * (1 + 2.0 ** -23), near * (1 - 2.0 ** -23)])
    near = torch.cat([near, -near])
    near = near[near.abs() < 2 * top]
    rows = []
    for e in (0, -1, 5, -100, 110, -126 - TOP[bits], -135):              # the block's scale, where it can be
        b = torch.nn.functional.pad(near, (0, -near.numel() % 31)).view(-1, 31)
        b = torch.cat([torch.full_like(b[:, :1], top), b], 1) * 2.0 ** e  # each block's largest binade is the format's
        rows.append(b.flatten())
    for big in (1.0, 1.5, 1.75, 1.9999999, 2.0):                         # the largest magnitude itself
        rows.append(torch.nn.functional.pad(torch.full((1,), big, dtype=torch.float64, device="cuda"), (0, rows[0].numel() - 1)))
    x = torch.stack(rows).float()
    m = Held(*x.shape, bits)
    call(lib.tcg_mx_quantize, C.byref(m.mx()), x.data_ptr(), x.shape[1], tcg.F32)
    m.check(*quantised(x.double(), bits))


@pytest.mark.parametrize("bits", [4, 8])
def test_quantise_of_zeros_infinities_and_nan(lib, bits):
    x = torch.zeros((8, 96), device="cuda")
    x[1] = -0.0
    x[2, 40] = math.nan                  # the middle block only
    x[3, 0], x[3, 95] = math.inf, -math.inf
    x[4, :32] = torch.finfo(torch.float32).max
    x[5, :32] = 2.0 ** -149
    x[5, 32:] = 2.0 ** -126
    x[6, 5], x[6, 70] = 1e38, 1e-38
    x[7] = randn(gen(1), 96)
    m = Held(8, 96, bits)
    call(lib.tcg_mx_quantize, C.byref(m.mx()), x.data_ptr(), 96, tcg.F32)
    m.check(*quantised(x.double(), bits))
    y = torch.empty_like(x)
    call(lib.tcg_mx_dequantize, y.data_ptr(), C.byref(m.mx()), 96, tcg.F32)
    v = m.values()
    assert torch.equal(torch.isnan(y), torch.isnan(v)) and torch.isnan(v).sum() == 96
    assert torch.equal(torch.nan_to_num(y.double()), torch.nan_to_num(v))
    half = torch.empty((8, 96), dtype=torch.float16, device="cuda")      # beyond the type: infinities and zeros
    call(lib.tcg_mx_dequantize, half.data_ptr(), C.byref(m.mx()), 96, tcg.F16)
    assert torch.isinf(half[4, :32]).all() and (half[5] == 0).all()


def test_arrays_past_32_bits(lib):
    """2.2e9 values of 2 bytes, 1.1e9 bytes of codes as weights: rows from both ends are right, and so is their product."""
    rows, cols = 270_001, 8192
    x = torch.empty((rows, cols), dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    part = torch.randn((4096, cols), generator=g, device="cuda").half()
    for i in range(0, rows, 4096):
        x[i:i + 4096] = part[:rows - i] * (1 + i // 4096 % 7)
    m = Held(rows, cols, 4)
    call(lib.tcg_mx_quantize, C.byref(m.mx()), x.data_ptr(), cols, tcg.F16)
    at = torch.tensor([0, 1, 127, 128, 131072, 262143, 262144, rows - 2, rows - 1], device="cuda")
    code, scale = quantised(x[at].double(), 4)
    held = m.codes[:m.n].view(rows, -1)[at].long()
    assert torch.equal(torch.stack([held & 15, held >> 4], -1).flatten(1), code)
    r = at[:, None]
    b = torch.arange(cols // 32, device="cuda")[None]
    assert torch.equal(m.scales[(r // 128 * (cols // 128) + b // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + b % 4].long(), scale)
    back = torch.zeros((rows, cols), dtype=torch.float16, device="cuda")
    call(lib.tcg_mx_dequantize, back.data_ptr(), C.byref(m.mx()), cols, tcg.F16)
    w = code_values(4)[code % 8] * torch.where(code >= 8, -1.0, 1.0) * power(scale - 127).repeat_interleave(32, 1)
    assert torch.equal(back[at].double(), w)
    v = random_held(gen(4), 2, cols, 8, -8)
    y = torch.zeros((2, rows), device="cuda")
    call(lib.tcg_mx_linear, y.data_ptr(), C.byref(v.mx()), C.byref(m.mx()), None, rows, tcg.F32)
    want, tol = product(v.values(), w, "f32", 8)
    assert ((y[:, at].double() - want).abs() <= tol).all()


# ------------------------------------------------------------------ residual and norm

NORMS = [  # rows, cols, type, pad, offset
    (1, 1, "f32", 0, 0), (3, 32, "bf16", 0, 0), (1, 4096, "f32", 0, 0), (2, 4096, "f16", 0, 0), (70, 100, "f16", 0, 0),
    (301, 256, "f32", 0, 0), (300, 300, "bf16", 4, 0), (310, 777, "f16", 3, 1), (299, 1024, "f32", 1, 3), (400, 2571, "bf16", 0, 0),
    (600, 4096, "bf16", 8, 0), (296, 4104, "f32", 0, 0), (5, 8192, "bf16", 0, 0), (2, 8193, "f32", 2, 2), (3, 16384, "f16", 0, 0),
    (2, 16500, "f32", 0, 1), (1, 32768, "f32", 0, 0), (297, 8000, "f16", 0, 0),
]


def normed(h, w, eps):
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("rows,cols,t,pad,offset", NORMS)
def test_add_and_norm(lib, rows, cols, t, pad, offset):
    dt, code = TYPES[t]
    g = gen(rows * 3 + cols)
    eps = float(torch.tensor(1e-5))                                      # as the call takes it: fp32
    x, r = randn(g, rows, cols, dtype=dt, spread=2.0), randn(g, rows, cols, dtype=dt)
    w = randn(g, cols) * 0.2 + 1
    x_rows, _, xp, ld = rows_of(x, pad, offset)
    r_rows, _, rp, _ = rows_of(r, pad, offset)
    h = (x.float() + r.float()).to(dt)
    # the product of three fp32 factors, each rounded, and the root's rounding: 3 u, then the type's
    def near(y, v):
        return ((y.double() - v).abs() <= v.abs() * (4 * U + (half_step(dt) if t != "f32" else 0)) + (2.0 ** -24 if t == "f16" else 0)).all()
    for bits in (0, 4, 8):
        m = Held(rows, cols, bits) if bits else None
        flat, hv, hp, _ = rows_of(torch.zeros_like(x), pad, offset)
        y_rows, yv, yp, _ = rows_of(torch.zeros_like(x), pad, offset)
        call(lib.tcg_add_rms_norm, hp, yp, C.byref(m.mx()) if m else None, xp, rp, w.data_ptr(), eps, rows, cols, ld, ld, ld, ld, code)
        want = normed(h.double(), w, eps)
        assert torch.equal(hv, h) and near(yv, want)
        assert (flat[:offset] == 7).all() and (flat[offset:].view(rows, -1)[:, cols:] == 7).all()
        if m:
            m.check(*quantised(want, bits))
    # no residual; in place of x; only the sum; only codes
    own_rows, iv, ip, _ = rows_of(x, pad, offset)
    call(lib.tcg_add_rms_norm, None, ip, None, ip, None, w.data_ptr(), eps, rows, cols, ld, ld, ld, ld, code)
    assert near(iv, normed(x.double(), w, eps))
    m = Held(rows, cols, 8)
    own_rows, iv, ip, _ = rows_of(x, pad, offset)
    call(lib.tcg_add_rms_norm, ip, None, C.byref(m.mx()), ip, rp, w.data_ptr(), eps, rows, cols, ld, ld, ld, ld, code)
    assert torch.equal(iv, h)
    m.check(*quantised(normed(h.double(), w, eps), 8))
    own_rows, iv, ip, _ = rows_of(r, pad, offset)
    call(lib.tcg_add_rms_norm, ip, None, None, xp, ip, None, eps, rows, cols, ld, ld, ld, ld, code)
    assert torch.equal(iv, h)


LAYOUTS = [  # of x and r, of h and y: (elements a row is longer, the first one's offset), 16-byte boundaries unless odd; of w
    ((8, 0), (3, 0), 0), ((0, 8), (0, 1), 0), ((3, 1), (8, 0), 0), ((8, 8), (1, 3), 4), ((8, 0), (8, 0), 1), ((5, 2), (2, 5), 3),
]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(3, 200), (300, 256), (1, 2571), (310, 512), (777, 2571), (300, 4104), (297, 8000), (2, 9001), (2, 20000)])
def test_norm_with_unlike_layouts(lib, rows, cols, t):
    """Rows that are read and rows that are written on unlike boundaries, weights off their own; one token's and many rows'
    kernels of each width."""
    dt, code = TYPES[t]
    g, eps = gen(rows * 7 + cols), float(torch.tensor(1e-5))
    x, r = randn(g, rows, cols, dtype=dt, spread=2.0), randn(g, rows, cols, dtype=dt)
    h = (x.float() + r.float()).to(dt)
    cols_up = -(-cols // 8) * 8
    for i, ((in_pad, in_off), (out_pad, out_off), w_off) in enumerate(LAYOUTS):
        in_pad, out_pad = in_pad + cols_up - cols, out_pad + cols_up - cols
        x_rows, _, xp, ldx = rows_of(x, in_pad, in_off)
        r_rows, _, rp, ldr = rows_of(r, in_pad, in_off)
        w_all = randn(g, cols + w_off) * 0.2 + 1
        w, wp = w_all[w_off:], w_all.data_ptr() + 4 * w_off
        for residual in (True, False):
            want_h = h if residual else x
            want = normed(want_h.double(), w, eps)
            for bits in ((0, 4, 8) if i % 2 else (0, 8)):
                m = Held(rows, cols, bits) if bits else None
                h_rows, hv, hp, ldh = rows_of(torch.zeros_like(x), out_pad, out_off)
                y_rows, yv, yp, ldy = rows_of(torch.zeros_like(x), out_pad + 8, out_off)
                call(lib.tcg_add_rms_norm, hp, yp, C.byref(m.mx()) if m else None, xp, rp if residual else None, wp, eps, rows, cols,
                     ldh, ldy, ldx, ldr, code)
                assert torch.equal(hv, want_h)
                # three fp32 factors and the root, each rounded, then the type's rounding
                tol = want.abs() * (4 * U + (half_step(dt) if t != "f32" else 0)) + (2.0 ** -24 if t == "f16" else 0)
                assert ((yv.double() - want).abs() <= tol).all()
                for flat in (h_rows, y_rows):
                    wide = (flat.numel() - out_off) // rows
                    assert (flat[:out_off] == 7).all() and (flat[out_off:].view(rows, wide)[:, cols:] == 7).all()
                if m:
                    m.check(*quantised(want, bits))
            # the sum alone, or a copy of x where there is none to add
            h_rows, hv, hp, ldh = rows_of(torch.zeros_like(x), out_pad, out_off)
            call(lib.tcg_add_rms_norm, hp, None, None, xp, rp if residual else None, None, eps, rows, cols, ldh, 0, ldx, ldr, code)
            assert torch.equal(hv, want_h)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 256), (2, 4096), (5, 20000), (400, 300), (300, 4096)])
def test_the_sum_alone_reads_no_weights(lib, rows, cols):
    """With h alone asked for, w may be any address: one that is not there, one that no float stands at."""
    g = gen(cols)
    x, r, h = randn(g, rows, cols), randn(g, rows, cols), torch.zeros((rows, cols), device="cuda")
    for w in (None, 1, 4096, h.data_ptr() + 2):
        h.zero_()
        call(lib.tcg_add_rms_norm, h.data_ptr(), None, None, x.data_ptr(), r.data_ptr(), w, 1e-6, rows, cols, cols, 0, cols, cols, tcg.F32)
        assert torch.equal(h, x + r)


@pytest.mark.parametrize("bits", [4, 8])
def test_norm_codes_next_to_borders(lib, bits):
    """Weights that put every value within an fp32 step of a border between codes, or of a power of two for the scale: the
    codes are those of the formula in 64 bits all the same."""
    g = gen(bits)
    grid = code_values(bits)
    mid = (grid[1:] + grid[:-1]) / 2
    cols, eps = 4096, float(torch.tensor(1e-6))
    x = randn(g, 40, cols)
    inv = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)
    # row 0's values at borders; the other rows share the weights and land anywhere
    pick = mid[torch.randint(0, mid.numel(), (cols,), generator=g).cuda()]
    pick[::32] = 2.0 ** TOP[bits] * torch.where(torch.rand(cols // 32, generator=g).cuda() < 0.5, 1.0, 2.0)
    w = (pick / (x[0].double() * inv[0])).float()
    w = torch.where(torch.rand(cols, generator=g).cuda() < 0.3, torch.nextafter(w, torch.zeros_like(w)), w)
    m = Held(40, cols, bits)
    call(lib.tcg_add_rms_norm, None, None, C.byref(m.mx()), x.data_ptr(), None, w.data_ptr(), eps, 40, cols, 0, 0, cols, 0, tcg.F32)
    m.check(*quantised(normed(x.double(), w, eps), bits))


def test_norm_of_odd_rows(lib):
    """Rows of zeros, of tiny and of huge values, with an infinity or a NaN: the others stay as they are."""
    g, eps = gen(9), float(torch.tensor(1e-6))
    x = randn(g, 8, 300)
    x[1] = 0
    x[2] *= 1e-30
    x[3] *= 1e34
    x[4, 17] = math.inf
    x[5, 3] = math.nan
    x[6] *= 1e-44
    w = randn(g, 300) * 0.1 + 1
    m, y = Held(8, 300, 8), torch.empty_like(x)
    call(lib.tcg_add_rms_norm, None, y.data_ptr(), C.byref(m.mx()), x.data_ptr(), None, w.data_ptr(), eps, 8, 300, 0, 300, 300, 0, tcg.F32)
    want = normed(x.double(), w, eps)
    assert torch.isnan(y[4, 17]) and torch.isnan(y[5]).all() and (y[1] == 0).all()
    assert (y[4, torch.arange(300, device="cuda") != 17] == 0).all()     # x / infinity
    for i in (0, 1, 2, 3, 7):
        assert ((y[i].double() - want[i]).abs() <= want[i].abs() * 4 * U).all()
    assert ((y[6].double() - want[6]).abs() <= 2.0 ** -149).all()        # subnormals
    code, scale = quantised(want, 8)
    got, sc = m.code(), m.scale()
    for i in (0, 1, 2, 3, 7):
        assert torch.equal(got[i], code[i]) and torch.equal(sc[i], scale[i])
    assert (sc[5, :10] == 255).all() and sc[4, 0] == 255 and (sc[4, 1:] == 0).all()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(3, 256), (2, 4096), (310, 700), (300, 6000), (2, 20000)])
def test_norm_of_rows_of_unlike_values(lib, rows, cols, t):
    """Values 40 orders below their own row's size, which large weights bring back to ordinary numbers: the factor between is
    below fp32's normal numbers, and the results and their codes are those of the formula all the same."""
    dt, code = TYPES[t]
    g, eps = gen(rows + cols), float(torch.tensor(1e-6))
    col = torch.arange(cols, device="cuda")
    small = col // 32 % 3 == 1
    x = randn(g, rows, cols, dtype=torch.float64)
    x = torch.where(x.abs() < 0.05, 0.05, x) * torch.where(small, 1e-22, 1e20)
    x[:, 64:96] = torch.where(col[64:96] % 5 == 0, 1e-25, 1e18) * x[:, 64:96].sign()     # one block holds both
    x[:, 70] = 0
    x = x.to(dt)
    w = ((randn(g, cols) * 0.1 + 1) * torch.where(small | (col // 32 == 2), 1e10, 1.0)).float()
    want = normed(x.double(), w, eps)
    y = torch.zeros_like(x)
    for bits in (4, 8):
        m = Held(rows, cols, bits)
        call(lib.tcg_add_rms_norm, None, y.data_ptr(), C.byref(m.mx()), x.data_ptr(), None, w.data_ptr(), eps, rows, cols, 0, cols, cols, 0, code)
        assert want.abs()[want != 0].min() > 2.0 ** -126
        assert ((y.double() - want).abs() <= want.abs() * (4 * U + (half_step(dt) if t == "bf16" else 0))).all()
        m.check(*quantised(want, bits))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shift", [-121, 0, 118])
def test_norm_codes_at_the_ends_of_the_range(lib, bits, shift):
    """Borders between codes as in test_norm_codes_next_to_borders, down to fp32's smallest normal numbers, where what is left
    of a product falls below fp32 altogether, and up to the largest, where its fp32 form is an infinity."""
    g, cols, eps = gen(bits + shift), 4096, float(torch.tensor(1e-6))
    grid = code_values(bits)
    mid = (grid[1:] + grid[:-1]) / 2
    mid = mid[mid > 2.0 ** -5]
    x = randn(g, 3, cols)
    x = torch.where(x.abs() < 0.05, 0.05, x)
    inv = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)
    pick = mid[torch.randint(0, mid.numel(), (cols,), generator=g).cuda()]
    pick[::32] = 2.0 ** TOP[bits] * torch.where(torch.rand(cols // 32, generator=g).cuda() < 0.5, 1.0, 2.0)
    if shift > 0:                                                        # next to the largest number, from below
        x = torch.where(x.abs() < 1, x.sign() * 1.25, x)
        inv = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + eps)
        pick = torch.where(torch.rand(cols, generator=g).cuda() < 0.5, torch.finfo(torch.float32).max, pick.clamp(max=64) * 2.0 ** shift)
        w = (pick / (x[0].double().abs() * inv[0])).clamp(max=3e38).float()
        w = torch.nextafter(w, torch.zeros_like(w))
        x = x[:1]
    else:
        w = (pick * 2.0 ** shift / (x[0].double() * inv[0])).float()
        w = torch.where(torch.rand(cols, generator=g).cuda() < 0.3, torch.nextafter(w, torch.zeros_like(w)), w)
    want = normed(x.double(), w, eps)
    assert want[0].abs().min() >= 2.0 ** -126 and want.abs().max() <= torch.finfo(torch.float32).max
    m = Held(len(x), cols, bits)
    call(lib.tcg_add_rms_norm, None, None, C.byref(m.mx()), x.data_ptr(), None, w.data_ptr(), eps, len(x), cols, 0, cols, cols, 0, tcg.F32)
    code, scale = quantised(want, bits)
    sure = (want.abs() >= 2.0 ** -126).all(-1)                            # rows whose values are all normal numbers
    assert sure[0] and torch.equal(m.code()[:len(x)][sure], code[sure]) and torch.equal(m.scale()[:len(x)][sure], scale[sure])


# ------------------------------------------------------------------ the product

def product(x, w, t, bits, bias=None):
    """x w^T + bias in 64 bits, and how far the kernel may be off: each step of 32 (8 bits) or 64 columns (4 bits) adds to an
    fp32 sum that the tensor core may cut instead of rounding (2 u of the largest partial sum, which is at most the sum of
    magnitudes), once for the alignment of the step's own products and once for the sum; the parts of a split and the bias
    are rounded (u each, at most 12 of them); then the type's rounding."""
    want, mag = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    dt = TYPES[t][0]
    steps = -(-x.shape[1] // (32 if bits == 8 else 64))
    tol = mag * (4 * steps + 12) * U
    return want, tol + (want.abs() + tol) * (half_step(dt) if t != "f32" else U) + (2.0 ** -25 if t == "f16" else 0)


LINEARS = [  # rows, cols, outs
    (1, 1, 1), (1, 32, 128), (1, 33, 129), (1, 4096, 1000), (7, 100, 130), (8, 4096, 200), (9, 256, 128), (16, 1000, 300), (17, 128, 64),
    (32, 5000, 257), (33, 700, 500), (64, 14336, 130), (65, 520, 140), (100, 2080, 500), (127, 4000, 333), (128, 1024, 1024),
    (129, 300, 1000), (200, 4096, 4096), (300, 129, 5003), (513, 4224, 2500), (1024, 9000, 4096), (1025, 640, 4100), (2047, 384, 3001),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,cols,outs", LINEARS)
def test_linear(lib, rows, cols, outs, bits):
    g = gen(rows + cols + outs + bits)
    x, w = random_held(g, rows, cols, bits, -8 if bits == 8 else -2), random_held(g, outs, cols, 4, -4)
    xv, wv = x.values(), w.values()
    bias = randn(g, outs)
    for i, (t, (dt, code)) in enumerate(TYPES.items()):
        b = bias if (rows + i) % 2 else None
        pad = (0, 1, 2)[(rows + i) % 3]
        flat, view, ptr, ld = rows_of(torch.zeros((rows, outs), dtype=dt, device="cuda"), pad, (rows + i) % 2)
        call(lib.tcg_mx_linear, ptr, C.byref(x.mx()), C.byref(w.mx()), b.data_ptr() if b is not None else None, ld, code)
        want, tol = product(xv, wv, t, bits, b)
        assert want.abs().max() < 60000                                  # within f16
        assert ((view.double() - want).abs() <= tol).all()
        first = view.clone()
        assert (flat[:(rows + i) % 2] == 7).all() and (flat[(rows + i) % 2:].view(rows, -1)[:, outs:] == 7).all()
        call(lib.tcg_mx_linear, ptr, C.byref(x.mx()), C.byref(w.mx()), b.data_ptr() if b is not None else None, ld, code)
        assert torch.equal(view, first)                                  # the same bits again


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows,cols,outs", [(1, 70000, 300), (64, 262144, 130), (128, 100000, 200), (600, 70000, 1024), (2000, 66000, 4100)])
def test_linear_of_long_sums_of_one_sign(lib, rows, cols, outs, bits):
    """Where the tensor core's cuts add up: results stay within what the header gives for a step (2^-22 of the sum), whatever
    the type, and 16-bit ones within two of their own roundings up to the columns that it names."""
    g = gen(rows + cols)
    x, w = random_held(g, rows, cols, bits, -12 if bits == 8 else -6), random_held(g, outs, cols, 4, -8)
    for m in (x, w):
        m.put(m.code() % (1 << (m.bits - 1)), m.scale()[:m.rows])
    xv, wv = x.values(), w.values()
    for t, (dt, code) in TYPES.items():
        y = torch.zeros((rows, outs), dtype=dt, device="cuda")
        call(lib.tcg_mx_linear, y.data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, outs, code)
        want, tol = product(xv, wv, t, bits)
        assert want.min() > 1 and want.max() < 60000
        assert ((y.double() - want).abs() <= tol).all()
        if t == "bf16" or (t == "f16" and cols <= (65536 if bits == 8 else 131072)):
            assert ((y.double() - want).abs() <= 2 * half_step(dt) * want).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("outs", [20011, 40000])
@pytest.mark.parametrize("rows,cols", [(1, 128), (1, 1100), (12, 128), (12, 1100), (30, 300), (30, 1100), (64, 128), (64, 1100), (100, 700)])
def test_linear_of_few_rows_in_several_waves(lib, rows, cols, outs, bits):
    """More tiles than SMs: CTAs that share an SM's memory and TMEM (up to 32 rows of x), or take turns at TMEM (up to 64)."""
    g = gen(rows + cols + outs + bits)
    x, w = random_held(g, rows, cols, bits, -8 if bits == 8 else -2), random_held(g, outs, cols, 4, -4)
    xv, wv = x.values(), w.values()
    for t in ("f32", "bf16"):
        dt, code = TYPES[t]
        want, tol = product(xv, wv, t, bits)
        out = []
        for _ in range(3):
            flat, view, ptr, ld = rows_of(torch.zeros((rows, outs), dtype=dt, device="cuda"), 1, 1)
            call(lib.tcg_mx_linear, ptr, C.byref(x.mx()), C.byref(w.mx()), None, ld, code)
            assert ((view.double() - want).abs() <= tol).all()
            assert flat[0] == 7 and (flat[1:].view(rows, -1)[:, outs:] == 7).all()
            out.append(view.clone())
        assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def test_linear_of_nothing(lib):
    x, w = random_held(gen(1), 3, 64, 8, -8), random_held(gen(2), 5, 64, 4, -4)
    none = tcg.Mx(None, None, 0, 64, 8)
    no_out = tcg.Mx(None, None, 0, 64, 4)
    y = torch.full((3, 5), 7.0, device="cuda")
    call(lib.tcg_mx_linear, y.data_ptr(), C.byref(none), C.byref(w.mx()), None, 5, tcg.F32)
    call(lib.tcg_mx_linear, y.data_ptr(), C.byref(x.mx()), C.byref(no_out), None, 5, tcg.F32)
    call(lib.tcg_mx_quantize, C.byref(none), None, 64, tcg.F32)
    call(lib.tcg_mx_dequantize, None, C.byref(none), 64, tcg.F32)
    call(lib.tcg_add_rms_norm, None, None, C.byref(none), None, None, None, 1e-6, 0, 64, 64, 64, 64, 64, tcg.F32)
    assert (y == 7).all()


@pytest.mark.parametrize("rows,outs", [(5, 300), (600, 4096)])
@pytest.mark.parametrize("bits", [4, 8])
def test_linear_with_nan_blocks(lib, rows, outs, bits):
    """A NaN block reaches its row of x, or its weight's column, and nothing else."""
    x, w = random_held(gen(5), rows, 640, bits, -6), random_held(gen(6), outs, 640, 4, -4)
    code, s = x.code(), x.scale()[:rows]
    s[3, 7] = 255
    x.put(code, s)
    code, s = w.code(), w.scale()[:outs]
    s[outs - 1, 0] = s[17, 19] = 255
    w.put(code, s)
    y = torch.zeros((rows, outs), device="cuda")
    call(lib.tcg_mx_linear, y.data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, outs, tcg.F32)
    bad = torch.zeros((rows, outs), dtype=torch.bool, device="cuda")
    bad[3], bad[:, outs - 1], bad[:, 17] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    want, tol = product(torch.nan_to_num(x.values()), torch.nan_to_num(w.values()), "f32", bits)
    assert ((y.double() - want).abs() <= tol)[~bad].all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows", [3, 700])
def test_linear_with_far_scales(lib, rows, bits):
    """Scales at both ends whose products are ordinary; and blocks of unlike sizes, the large ones first or last."""
    x, w = random_held(gen(7), rows, 512, bits, -115, 5), random_held(gen(8), 4096, 512, 4, 110, 5)
    y = torch.zeros((rows, 4096), device="cuda")
    call(lib.tcg_mx_linear, y.data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, 4096, tcg.F32)
    want, tol = product(x.values(), w.values(), "f32", bits)
    assert ((y.double() - want).abs() <= tol).all()
    x, w = random_held(gen(9), rows, 4096, bits, 0, 0), random_held(gen(10), 4096, 4096, 4, 0, 0)
    ramp = torch.linspace(115, 139, 128, device="cuda").long()
    for s in (ramp, ramp.flip(0)):
        x.put(x.code(), s.expand(rows, -1))
        call(lib.tcg_mx_linear, y.data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, 4096, tcg.F32)
        want, tol = product(x.values(), w.values(), "f32", bits)
        assert ((y.double() - want).abs() <= tol).all()


WITHHELD = [  # rows, cols, outs, bits, type, stages that are loaded
    (1, 4096, 14336, 8, "f32", 0), (40, 4096, 14336, 4, "bf16", 7),      # K undivided
    (1, 14336, 4096, 8, "f32", 1), (64, 14336, 4096, 4, "f16", 0), (100, 14336, 4096, 8, "f32", 7),      # split over clusters
    (1024, 4096, 4096, 4, "bf16", 0), (1024, 4096, 4096, 8, "f32", 7), (3000, 2304, 5000, 8, "bf16", 1), (3000, 2304, 5000, 4, "f32", 0),
]


@pytest.mark.parametrize("rows,cols,outs,bits,t,stages", WITHHELD)
def test_waits_that_give_up(lib, rows, cols, outs, bits, t, stages):
    """Loading warps that stop asking after some stages: the waits for the next one run out after their second, the kernel
    returns without a store and reports it, and the next call is right."""
    dt, code = TYPES[t]
    g = gen(rows + stages)
    x, w = random_held(g, rows, cols, bits, -8 if bits == 8 else -2), random_held(g, outs, cols, 4, -4)
    flat, view, ptr, ld = rows_of(torch.full((rows, outs), 7.0, dtype=dt, device="cuda"), 2, 4)
    args = (ptr, C.byref(x.mx()), C.byref(w.mx()), None, ld, code)
    assert lib.tcg_test_mx_withhold_loads(stages) == -1
    try:
        call(lib.tcg_mx_linear, *args)
    finally:
        assert lib.tcg_test_mx_withhold_loads(-1) == stages
    assert lib.tcg_device_error() == tcg.ERR_MX_WAIT
    assert (flat == 7).all()
    tcg.check(lib.tcg_clear_device_error())
    call(lib.tcg_mx_linear, *args)
    want, tol = product(x.values(), w.values(), t, bits)
    assert ((view.double() - want).abs() <= tol).all() and lib.tcg_device_error() == 0


# ------------------------------------------------------------------ together

class Layer:
    """A feed-forward block on microscaled rows: add and norm, product, GELU, quantisation, product; then add and norm."""

    def __init__(self, g, n, d, f, bits):
        self.n, self.d, self.f, self.bits, self.eps = n, d, f, bits, float(torch.tensor(1e-5))
        self.up, self.down = Held(f, d, 4), Held(d, f, 4)
        for m, s in ((self.up, 0.05), (self.down, 0.03)):
            v = randn(g, m.rows, m.cols, spread=s)
            call(tcg.lib().tcg_mx_quantize, C.byref(m.mx()), v.data_ptr(), m.cols, tcg.F32)
        self.w = [randn(g, d) * 0.1 + 1 for _ in range(2)]
        self.b = randn(g, f) * 0.1
        self.x, self.r = torch.zeros((n, d), device="cuda"), torch.zeros((n, d), device="cuda")
        self.h, self.out = torch.zeros_like(self.x), torch.zeros_like(self.x)
        self.a, self.c = Held(n, d, bits), Held(n, f, bits)
        self.mid, self.act, self.back = torch.zeros((n, f), device="cuda"), torch.zeros((n, f), device="cuda"), torch.zeros((n, d), device="cuda")

    def run(self):
        L, ck, p, n, d, f = tcg.lib(), tcg.check, lambda t: t.data_ptr(), self.n, self.d, self.f
        ck(L.tcg_add_rms_norm(p(self.h), None, C.byref(self.a.mx()), p(self.x), p(self.r), p(self.w[0]), self.eps, n, d, d, d, d, d, 0))
        ck(L.tcg_mx_linear(p(self.mid), C.byref(self.a.mx()), C.byref(self.up.mx()), p(self.b), f, 0))
        ck(L.tcg_gelu(p(self.act), p(self.mid), n * f))
        ck(L.tcg_mx_quantize(C.byref(self.c.mx()), p(self.act), f, 0))
        ck(L.tcg_mx_linear(p(self.back), C.byref(self.c.mx()), C.byref(self.down.mx()), None, d, 0))
        ck(L.tcg_add_rms_norm(None, p(self.out), None, p(self.back), p(self.h), p(self.w[1]), self.eps, n, d, d, d, d, d, 0))

    def check(self):
        """Every step against the formula on what the step before it left."""
        h = self.x + self.r
        assert torch.equal(self.h, h)
        self.a.check(*quantised(normed(h.double(), self.w[0], self.eps), self.bits))
        want, tol = product(self.a.values(), self.up.values(), "f32", self.bits, self.b)
        assert ((self.mid.double() - want).abs() <= tol).all()
        m = self.mid.double()
        assert (self.act.double() - 0.5 * m * (1 + torch.erf(m / math.sqrt(2)))).abs().max() <= 1e-6 * (1 + m.abs().max())
        self.c.check(*quantised(self.act.double(), self.bits))
        want, tol = product(self.c.values(), self.down.values(), "f32", self.bits)
        assert ((self.back.double() - want).abs() <= tol).all()
        out = normed((self.back + self.h).double(), self.w[1], self.eps)
        assert ((self.out.double() - out).abs() <= out.abs() * 4 * U).all()


@pytest.mark.parametrize("n,bits", [(1, 8), (5, 4), (40, 8), (300, 4)])
def test_a_run_of_them_in_a_graph(lib, n, bits):
    g = gen(n)
    layer = Layer(g, n, 512, 1408, bits)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    tcg.check(lib.tcg_set_stream(stream.cuda_stream))
    try:
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            layer.run()
        for i in range(5):
            layer.x.copy_(randn(g, n, 512, spread=2.0))
            layer.r.copy_(randn(g, n, 512))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            layer.check()
        layer.run()                                                      # and as plain calls on the caller's stream
        torch.cuda.synchronize()
        layer.check()
    finally:
        torch.cuda.synchronize()
        tcg.check(lib.tcg_set_stream(None))


CAPTURED_FIRST = """
import sys, torch
sys.path[:0] = sys.argv[1:3]
import tcg, test_gpu_mx as T
tcg.init(0)
L = tcg.lib()
for n, bits in ((1, 8), (12, 4), (33, 8), (70, 4), (1500, 8), (1500, 4)):
    layer = T.Layer(T.gen(n), n, 512, 2816, bits)
    layer.x.copy_(T.randn(T.gen(n + 1), n, 512))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    tcg.check(L.tcg_set_stream(stream.cuda_stream))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        layer.run()
    graph.replay()
    torch.cuda.synchronize()
    tcg.check(L.tcg_set_stream(None))
    layer.check()
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


def test_streams_at_once(lib):
    """The operators keep nothing between calls: calls of three streams, of split, whole and paired kinds, do not disturb
    one another."""
    shapes = [(1, 4096, 4096), (64, 8192, 2048), (100, 4096, 1024), (1024, 1024, 4096)]
    jobs = []
    for i, (rows, cols, outs) in enumerate(shapes):
        bits = 4 if i % 2 else 8
        x, w = random_held(gen(i), rows, cols, bits, -8), random_held(gen(i + 9), outs, cols, 4, -4)
        want = torch.zeros((rows, outs), device="cuda")
        call(lib.tcg_mx_linear, want.data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, outs, tcg.F32)
        jobs.append((x, w, want, [torch.zeros_like(want) for _ in range(12)]))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    try:
        for i in range(12):
            for k, (x, w, want, got) in enumerate(jobs):
                tcg.check(lib.tcg_set_stream(streams[(i + k) % 3].cuda_stream))
                tcg.check(lib.tcg_mx_linear(got[i].data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, want.shape[1], tcg.F32))
    finally:
        torch.cuda.synchronize()
        tcg.check(lib.tcg_set_stream(None))
    for x, w, want, got in jobs:
        assert all(torch.equal(o, want) for o in got)


THREADS_FIRST = """
import sys, threading, torch
sys.path[:0] = sys.argv[1:3]
import tcg, test_gpu_mx as T
L, g, N = tcg.lib(), T.gen(31), 8
tcg.init(0)
C, jobs = T.C, []
for rows, cols, outs, bits in ((1, 14336, 4096, 8), (40, 4096, 2000, 4), (100, 2080, 500, 8), (700, 640, 4100, 4)):
    v = T.randn(g, rows, cols)
    x, w = T.Held(rows, cols, bits), T.random_held(g, outs, cols, 4, -6)
    jobs.append((v, torch.ones(cols, device="cuda"), x, w, T.normed(v.double(), torch.ones(cols, device="cuda"), 0.0)))
mine = [[(T.Held(x.rows, x.cols, x.bits), torch.zeros((x.rows, w.rows), device="cuda"), torch.zeros_like(v)) for v, _, x, w, _ in jobs]
        for _ in range(N)]
wall, bad = threading.Barrier(N), []
torch.cuda.synchronize()

def work(i):
    try:
        tcg.init(0)
        for (v, one, x, w, _), (m, y, back) in zip(jobs, mine[i]):
            wall.wait(60)
            tcg.check(L.tcg_add_rms_norm(None, None, C.byref(m.mx()), v.data_ptr(), None, one.data_ptr(), 0.0, x.rows, x.cols, 0, 0, x.cols, 0, 0))
            tcg.check(L.tcg_mx_linear(y.data_ptr(), C.byref(m.mx()), C.byref(w.mx()), None, w.rows, 0))
            tcg.check(L.tcg_mx_dequantize(back.data_ptr(), C.byref(m.mx()), x.cols, 0))
        tcg.check(L.tcg_sync())
        assert L.tcg_device_error() == 0
    except Exception as e:
        bad.append(e)
        wall.abort()

threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert not bad, bad
for k, (v, one, x, w, norm) in enumerate(jobs):
    for i in range(N):
        m, y, back = mine[i][k]
        m.check(*T.quantised(norm, x.bits))
        want, tol = T.product(m.values(), w.values(), "f32", x.bits)
        assert ((y.double() - want).abs() <= tol).all() and torch.equal(y, mine[0][k][1]) and torch.equal(back.double(), m.values())
print("together")
"""


def test_first_calls_of_several_threads_at_once():
    """Threads whose first calls of each operator come together: each has a context of its own, none runs unprepared."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    pkg = os.path.join(os.path.dirname(here), "roofline.c_b200")
    out = subprocess.run([sys.executable, "-c", THREADS_FIRST, here, pkg], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "together" in out.stdout, out.stderr[-2000:]


@pytest.mark.parametrize("kind", ["Q4_K", "Q6_K"])
def test_weights_of_a_gguf_tensor(lib, kind):
    """From a tensor's K-quant blocks over its values to 4 bits and into a product: the codes are those of the values, each
    within a quarter of itself or of its block's unit, and the product is that of what is held."""
    import numpy as np
    import oracle
    import tcg_gguf as G
    outs, cols, qt = 512, 2048, getattr(G, kind)
    raw = G.make_kquant_like(qt, outs, cols, 17, 1e-3)
    v = torch.from_numpy(np.ascontiguousarray(oracle.dequant(raw, outs * cols, qt))).view(outs, cols).cuda().double()
    blocks, f32 = torch.from_numpy(raw).cuda(), torch.zeros((outs, cols), device="cuda")
    call(lib.tcg_dequant, f32.data_ptr(), blocks.data_ptr(), outs * cols, qt)
    assert torch.equal(f32.double(), v)
    w = Held(outs, cols, 4)
    call(lib.tcg_mx_quantize, C.byref(w.mx()), f32.data_ptr(), cols, tcg.F32)
    w.check(*quantised(v, 4))
    unit = power(w.scale()[:outs] - 127).repeat_interleave(32, 1)
    assert ((w.values() - v).abs() <= torch.maximum(v.abs(), unit) / 4).all()
    for rows, bits in ((1, 8), (70, 4)):
        x = Held(rows, cols, bits)
        a = randn(gen(rows), rows, cols)
        call(lib.tcg_mx_quantize, C.byref(x.mx()), a.data_ptr(), cols, tcg.F32)
        y = torch.zeros((rows, outs), device="cuda")
        call(lib.tcg_mx_linear, y.data_ptr(), C.byref(x.mx()), C.byref(w.mx()), None, outs, tcg.F32)
        want, tol = product(x.values(), w.values(), "f32", bits)
        assert ((y.double() - want).abs() <= tol).all()
