"""Microscaled rows on the GPU against their definition in 64 bits: quantisation and read-back bit for bit, the norm
and the products within bounds that follow from the roundings."""
import numpy as np
import pytest

from mx_ref import (BF16, F16, F32, FP4, FP8, HALF, VALUES, Mx, buf, from_type, quantize, random_rows, scale_bytes, to_type, unit,
                    values)

pytestmark = pytest.mark.gpu


def _quantize(F, x, t, fmt, ldx=0, **kw):
    m = Mx(F, fmt, x.shape[0], kw.pop("n", x.shape[1]), **kw)
    d = buf(F, x)
    F.mx_quantize_dev(t, d, m.mx, ldx)
    F.synchronize()
    return m


def _rows(rng, rows, n, t):
    x = rng.standard_normal((rows, n)) * np.repeat(np.exp2(rng.uniform(-20, 10, (rows, n // 32))), 32, 1)
    x[rng.random(x.shape) < 0.1] = 0
    return to_type(x.astype(np.float32), t)


@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(1, 32), (3, 64), (7, 96), (2, 5120), (33, 544), (1, 2080), (130, 160), (5, 65536)])
def test_quantize_and_read_back(gpu, rows, n, t, fmt):
    x = _rows(np.random.default_rng(rows * 7 + n), rows, n, t)
    m = _quantize(gpu, x, t, fmt)
    want = quantize(from_type(x, t), fmt)
    got = m.read()
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    for back in (F32, F16, BF16):
        ref = to_type(values(*want, fmt).astype(np.float32), back)
        d = buf(gpu, np.full((rows, n), 7, ref.dtype))
        gpu.mx_dequant_dev(m.mx, back, d)
        gpu.synchronize()
        assert np.array_equal(d.download(ref.dtype, ref.shape), ref)


@pytest.mark.parametrize("fmt", [FP4, FP8])
def test_quantize_ties_and_borders(gpu, fmt):
    """Every midpoint between two codes, the numbers beside it, and largest values at and beside every scale's border."""
    half = len(VALUES[fmt]) // 2
    grid = VALUES[fmt][:half if fmt == FP4 else half - 1].astype(np.float32)
    mid = ((grid[1:] + grid[:-1]) / 2).astype(np.float32)
    pts = np.concatenate([grid, mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))])
    pts = np.concatenate([pts, -pts])
    pts = np.pad(pts, (0, -len(pts) % 31))
    top = np.float32(grid[-1])
    blocks = np.concatenate([np.full((len(pts) // 31, 1), top, np.float32), pts.reshape(-1, 31)], 1)   # scale 1 in each
    blocks[:, 1:] = np.clip(blocks[:, 1:], -top, top)
    tops = []
    for e in (-149, -140, -130, -127, -126, -100, -1, 0, 1, 60, 119, 120, 125, 127):
        for v in (1.0, 1.5, 1.75, 1.9999):
            v = np.float32(np.ldexp(v, e))
            tops += [v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(0))]
    tops = np.array([v for v in tops if np.isfinite(v)], np.float32)
    border = tops[:, None] * np.linspace(-1, 1, 32, dtype=np.float32)[None]
    border[:, 5] = tops
    x = np.concatenate([blocks, border]).astype(np.float32)
    m = _quantize(gpu, x, F32, fmt)
    want, got = quantize(x, fmt), m.read()
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])


@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_quantize_non_finite_blocks(gpu, t, fmt):
    """A NaN or infinity takes its own block to NaN, scale 255 and codes 0, and no other."""
    x = from_type(_rows(np.random.default_rng(3), 6, 160, t), t)
    x[1, 40], x[2, 0], x[3, 159], x[4, 64:96] = np.nan, np.inf, -np.inf, np.nan
    m = _quantize(gpu, to_type(x.astype(np.float32), t), t, fmt)
    got, want = m.read(), quantize(x, fmt)
    assert np.array_equal(got[1], want[1]) and (got[1] == 255).sum() == 4
    assert np.array_equal(got[0], want[0])
    d = gpu.DeviceBuffer(6 * 160 * 4)
    gpu.mx_dequant_dev(m.mx, F32, d)
    gpu.synchronize()
    back = d.download(np.float32, (6, 160))
    assert np.array_equal(np.isnan(back), np.repeat(got[1] == 255, 32, 1))


@pytest.mark.parametrize("fmt", [FP4, FP8])
def test_quantize_strides(gpu, fmt):
    """Rows with gaps everywhere: gaps stay as they were, and what stands in them is not read."""
    rng = np.random.default_rng(5)
    x = _rows(rng, 19, 224, BF16)
    wide = np.concatenate([x, np.full((19, 24), 0x7FC0, x.dtype)], 1)
    m = _quantize(gpu, wide, BF16, fmt, ldx=248, n=224, gap=48, gap_scales=8, pad=0xA5)
    got, want = m.read(), quantize(from_type(x, BF16), fmt)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    out = np.full((19, 240), 9, np.float32)
    d = buf(gpu, out)
    gpu.mx_dequant_dev(m.mx, F32, d, 240)
    gpu.synchronize()
    back = d.download(np.float32, out.shape)
    assert np.array_equal(back[:, :224], values(*want, fmt).astype(np.float32)) and (back[:, 224:] == 9).all()


def test_read_back_every_code_and_scale(gpu):
    """All codes under all scales, as each type: rounded once, infinite where the type ends."""
    for fmt in (FP4, FP8):
        half = len(VALUES[fmt])
        codes = np.tile(np.arange(half, dtype=np.uint8), (256, max(1, 32 // half)))
        s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], codes.shape[1] // 32, 1)
        m = Mx(gpu, fmt, 256, codes.shape[1], codes, s)
        with np.errstate(over="ignore"):
            want = values(codes, s, fmt).astype(np.float32)
        for t in (F32, F16, BF16):
            with np.errstate(over="ignore"):
                ref = from_type(to_type(want, t), t)
            d = gpu.DeviceBuffer(codes.size * 4)
            gpu.mx_dequant_dev(m.mx, t, d)
            gpu.synchronize()
            got = from_type(d.download(to_type(want, t).dtype, want.shape), t)
            assert np.array_equal(got, ref, equal_nan=True)


# ---------------------------------------------------------------------------
# Norm
# ---------------------------------------------------------------------------
def _check_quantized(got, exact, fmt, rel):
    """Codes and scales of values that are known within rel: scales as the formula's, or where its largest value is
    that near the border between two; each value within half a step of its scale's grid."""
    codes, s = got
    amax = np.abs(exact).reshape(exact.shape[0], -1, 32).max(-1)
    lo, hi = scale_bytes(amax * (1 - rel), fmt), scale_bytes(amax * (1 + rel), fmt)
    assert ((s >= lo) & (s <= hi)).all()
    v = values(codes, s, fmt)
    u = np.repeat(unit(s), 32, 1)
    half = np.maximum(np.abs(exact) * (2.0 ** -2 if fmt == FP4 else 2.0 ** -4), (0.25 if fmt == FP4 else 2.0 ** -10) * u)
    off = np.abs(v - exact)
    assert (off <= half * (1 + 4 * rel) + rel * np.abs(exact)).all(), float((off / half).max())


def _norm(F, t, x, w, eps, fmt, add=None, sum_to=None, shift=None, scale=None, gap=0):
    rows, n = x.shape
    ld = n + gap
    wide = lambda a: np.concatenate([a, np.zeros((rows, gap), a.dtype)], 1)  # noqa: E731
    m = Mx(F, fmt, rows, n, gap=16 if gap else 0, gap_scales=4 if gap else 0)
    dx, da = buf(F, wide(x)), None if add is None else buf(F, wide(add))
    ds = {None: None, "x": dx, "add": da}.get(sum_to, buf(F, np.full((rows, ld), 3, x.dtype)))
    keep = [buf(F, a.astype(np.float32)) if a is not None else None for a in (w, shift, scale)]
    F.mx_norm_dev(t, dx, keep[0], eps, m.mx, d_add=da, d_sum=ds, d_shift=keep[1], d_scale=keep[2], ldx=ld if gap else 0,
                  ldadd=ld if gap else 0, ldsum=ld if gap else 0)
    F.synchronize()
    h = None if ds is None else ds.download(x.dtype, (rows, ld))[:, :n]
    return m.read(), h


def _norm_exact(x, w, eps, shift=None, scale=None):
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return n if shift is None else n * (1 + scale.astype(np.float64)) + shift


# everything up to a value's one rounding is in 64 bits: relative to its largest term about 10 * 2^-53
NORM_REL = 2.0 ** -49


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n", [(1, 32), (3, 96), (5, 5120), (17, 544), (2, 8224), (1, 32768), (300, 256), (2, 16416), (4, 14336)])
def test_norm(gpu, rows, n, t, fmt):
    rng = np.random.default_rng(rows + n)
    x, add = (to_type(rng.standard_normal((rows, n)).astype(np.float32), t) for _ in range(2))
    w = 1 + 0.1 * rng.standard_normal(n).astype(np.float32)
    got, h = _norm(gpu, t, x, w, 1e-6, fmt, add=add, sum_to="new")
    want = to_type((from_type(x, t) + from_type(add, t)).astype(np.float32), t)
    assert np.array_equal(h, want)
    _check_quantized(got, _norm_exact(from_type(want, t).astype(np.float64), w.astype(np.float64), 1e-6), fmt, NORM_REL)


@pytest.mark.parametrize("sum_to", ["x", "add", "new"])
@pytest.mark.parametrize("modulate", [False, True])
@pytest.mark.parametrize("gap", [0, 16])
def test_norm_in_place_modulated_strided(gpu, sum_to, modulate, gap):
    rng = np.random.default_rng(8)
    x, add = (to_type(rng.standard_normal((9, 352)).astype(np.float32), BF16) for _ in range(2))
    w = 1 + 0.1 * rng.standard_normal(352).astype(np.float32)
    shift, scale = ((0.5 + 0.1 * rng.standard_normal((9, 352))).astype(np.float32) for _ in range(2)) if modulate else (None, None)
    got, h = _norm(gpu, BF16, x, w, 1e-5, FP8, add, sum_to, shift, scale, gap)
    want = to_type((from_type(x, BF16) + from_type(add, BF16)).astype(np.float32), BF16)
    assert np.array_equal(h, want)
    exact = _norm_exact(from_type(want, BF16).astype(np.float64), w.astype(np.float64), 1e-5, shift, scale)
    codes, s = got
    # half a step, and the arithmetic's share of the two terms' sizes where they cancel
    size = np.abs(_norm_exact(from_type(want, BF16).astype(np.float64), w.astype(np.float64), 1e-5))
    size = size * (1 + np.abs(scale)) + np.abs(shift) if modulate else size
    half = np.maximum(np.abs(exact) * 2.0 ** -4, 2.0 ** -10 * np.repeat(unit(s), 32, 1))
    assert (np.abs(values(codes, s, FP8) - exact) <= half + NORM_REL * size).all()


def test_norm_without_addition(gpu):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((4, 1056)).astype(np.float32)
    w = np.ones(1056, np.float32)
    for sum_to in (None, "new"):
        got, h = _norm(gpu, F32, x, w, 0.0, FP8, sum_to=sum_to)
        _check_quantized(got, _norm_exact(x.astype(np.float64), w, 0.0), FP8, NORM_REL)
        assert h is None or np.array_equal(h, x)


def test_norm_of_any_size(gpu):
    """Rows of 10^-38 to 3 * 10^38 and rows of zeros; a NaN or an infinity changes no other row."""
    rng = np.random.default_rng(10)
    x = rng.uniform(0.5, 1, (9, 96)).astype(np.float32)
    for i, f in enumerate((1e-38, 1e-30, 1e-15, 1.0, 1e15, 1e30, 3e38)):
        x[i] *= np.float32(f)
    x[7] = 0
    w = np.ones(96, np.float32)
    got, _ = _norm(gpu, F32, x, w, 0.0, FP8)
    _check_quantized((got[0][:7], got[1][:7]), _norm_exact(x[:7].astype(np.float64), w, 0.0), FP8, NORM_REL)
    bad = x.copy()
    bad[2, 5], bad[4, 40] = np.nan, np.inf
    other, _ = _norm(gpu, F32, bad, w, 1e-6, FP8)
    clean, _ = _norm(gpu, F32, x, w, 1e-6, FP8)
    rest = [0, 1, 3, 5, 6, 7, 8]
    assert np.array_equal(other[0][rest], clean[0][rest]) and np.array_equal(other[1][rest], clean[1][rest])
    assert (other[1][2] == 255).all() and other[1][4, 1] == 255 and (clean[1][7] == 0).all()


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------
def _product_bound(xv, wv, t, fp8, exact_y):
    """Sums in fp32: each step of 128 values adds a rounding of at most 2^-23 (the instruction may cut rather than
    round) of the terms' sizes, and so does each join of parts (fewer than one to a step), bias and residual.  FP8 rows
    to 16 bits: of eight products up to seven lose less than 2^-13 of the largest's power of two.  Then the output's
    rounding."""
    size = np.abs(xv) @ np.abs(wv).T
    b = size * (2 * (xv.shape[1] // 128 + 1) + 4) * 2.0 ** -23
    if fp8 and t != F32:
        b = b + size * 7 * 2.0 ** -13
    return b, HALF[t] * np.abs(exact_y)


class Case:
    def __init__(self, seed, rows, n, out, fmt, bias=False, gate=False, res=False, spread=2.0):
        rng = np.random.default_rng(seed)
        self.rows, self.n, self.out, self.fmt = rows, n, out, fmt
        self.x, self.w = random_rows(rng, rows, n, fmt, spread), random_rows(rng, out, n, FP4, spread)
        self.bias = rng.standard_normal(out).astype(np.float32) if bias else None
        self.gate = rng.standard_normal((rows, out)).astype(np.float32) if gate else None
        self.res = rng.standard_normal((rows, out)).astype(np.float32) if res or gate else None

    def exact(self, t):
        y = self.x[2] @ self.w[2].T
        y = y if self.bias is None else y + self.bias
        if self.res is None:
            return y
        r = from_type(to_type(self.res, t), t).astype(np.float64)
        return r + (y if self.gate is None else self.gate * y)

    def run(self, F, t, gap=0, off=0, ldy=0, in_place=False, mx_gap=0, stream=None):
        """The product, into a buffer off values past its start with ldy values to a row; returns y and checks the gaps."""
        self.mx = Mx(F, self.fmt, self.rows, self.n, *self.x[:2], gap=mx_gap, gap_scales=mx_gap // 4), Mx(F, FP4, self.out, self.n, *self.w[:2])
        x, w = self.mx[0].mx, self.mx[1].mx
        kind = to_type(np.zeros(1, np.float32), t).dtype
        ld = max(ldy, self.out)
        full = np.full(off + self.rows * ld, 77, kind)
        if in_place:
            full[off:].reshape(self.rows, ld)[:, :self.out] = to_type(self.res, t)
        dy = buf(F, full)
        at = dy.ptr + off * kind.itemsize
        dr = None if self.res is None else (at if in_place else buf(F, to_type(self.res, t)))
        db = None if self.bias is None else buf(F, self.bias)
        dg = None if self.gate is None else buf(F, self.gate)
        need = F.mx_matmul_workspace_bytes(w, x)
        ws = F.DeviceBuffer(max(1, need))
        ws.fill(0xFF)
        F.mx_matmul_dev(w, x, t, at, ws, need, d_bias=db, d_gate=dg, d_res=dr, ldres=ld if in_place else 0, ldy=ld, stream_ptr=stream)
        F.synchronize()
        got = dy.download(kind, full.shape)
        rows = got[off:].reshape(self.rows, ld)
        assert (got[:off] == 77).all() and (rows[:, self.out:] == 77).all()
        return rows[:, :self.out]

    def check(self, y, t):
        want = self.exact(t)
        b, r = _product_bound(self.x[2], self.w[2], t, self.fmt == FP8, want)
        f = 1.0 if self.gate is None else np.abs(self.gate)
        got = from_type(y, t).astype(np.float64)
        extra = 2.0 ** -22 * (np.abs(want) + (0 if self.res is None else np.abs(self.res)))
        off = np.abs(got - want)
        assert np.isfinite(got).all()
        assert (off <= b * f + extra + r).all(), float((off / (b * f + extra + r)).max())


SIZES = [(1, 32, 1), (1, 64, 16), (2, 96, 17), (1, 5120, 130), (3, 160, 257), (8, 544, 100), (15, 256, 15), (16, 1024, 384), (17, 288, 33),
         (31, 5120, 96), (33, 832, 65), (64, 512, 128), (65, 128, 129), (100, 2080, 200), (128, 256, 128), (130, 1056, 260), (257, 416, 300),
         (300, 64, 520), (520, 1184, 257), (5, 25600, 64), (1, 13824, 48)]


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("rows,n,out", SIZES)
def test_product_fp32(gpu, rows, n, out, fmt):
    c = Case(rows + n + out, rows, n, out, fmt)
    c.check(c.run(gpu, F32), F32)


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("rows,n,out", [(1, 256, 48), (7, 5120, 50), (16, 288, 33), (40, 544, 160), (70, 1024, 70), (129, 320, 257), (400, 512, 384)])
def test_product_16_bit(gpu, rows, n, out, t, fmt):
    c = Case(rows + n + out, rows, n, out, fmt, bias=True)
    c.check(c.run(gpu, t), t)


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n,out", [(1, 512, 130), (20, 352, 64), (70, 256, 257), (300, 1024, 256)])
@pytest.mark.parametrize("bias,gate", [(False, False), (True, False), (False, True), (True, True)])
def test_product_bias_residual_gate(gpu, rows, n, out, t, fmt, bias, gate):
    c = Case(rows + n + out, rows, n, out, fmt, bias, gate, res=True)
    y = c.run(gpu, t)
    c.check(y, t)
    assert np.array_equal(c.run(gpu, t, in_place=True), y)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,out", [(3, 61), (19, 64), (200, 193), (260, 512)])
@pytest.mark.parametrize("off,more", [(0, 0), (1, 3), (3, 0), (4, 8), (8, 8)])
def test_product_strides(gpu, rows, out, t, off, more):
    """Rows of y at any stride and alignment, gaps in the codes and scales (which hold 255): the same bits, gaps stay."""
    c = Case(rows + out, rows, 736, out, FP8, bias=True, gate=True)
    y = c.run(gpu, t)
    assert np.array_equal(c.run(gpu, t, off=off, ldy=out + more, mx_gap=48), y)
    assert np.array_equal(c.run(gpu, t, off=off, ldy=out + more, in_place=True), y)


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("rows", [1, 12, 50, 140, 600])
def test_product_scales_of_any_size(gpu, rows, fmt):
    """Scales from 2^-120 to 2^120 that meet their inverses, blocks of zeros among them."""
    rng = np.random.default_rng(rows)
    c = Case(rows, rows, 640, 90, fmt)
    e = rng.integers(-100, 100, 20)
    for part, sign in ((c.x, 1), (c.w, -1)):
        s = np.clip(part[1].astype(np.int64) + sign * e[None], 0, 254).astype(np.uint8)
        part[1][:] = s
        part[0][:, 64:96] = 0
        part[2][:] = values(part[0], s, fmt if part is c.x else FP4)
    c.check(c.run(gpu, F32), F32)


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("rows,n,out", [(1, 512, 40), (14, 96, 33), (40, 1024, 70), (130, 288, 130), (300, 800, 300)])
def test_product_nan_rows(gpu, rows, n, out, fmt):
    """A NaN scale (in x or in W) or code makes its own row or column NaN; every other output keeps its bits."""
    c = Case(rows, rows, n, out, fmt)
    clean = c.run(gpu, F32)
    c.x[1][rows // 2, n // 32 - 1] = 255
    c.w[1][out - 2, 0] = 255
    if fmt == FP8:
        c.x[0][0, n - 1] = 0x7F
    bad = c.run(gpu, F32)
    nan = np.zeros((rows, out), bool)
    nan[rows // 2], nan[:, out - 2] = True, True
    if fmt == FP8:
        nan[0] = True
    assert np.array_equal(np.isnan(bad), nan)
    assert np.array_equal(bad[~nan], clean[~nan])


def test_fp32_output_of_fp8_rows_is_exact(gpu):
    """Eight products of very different sizes: what the single instruction would cut is there."""
    n, rows, out = 256, 300, 64
    for rows in (1, 300):
        codes = np.zeros((rows, n), np.uint8)
        codes[:, ::8], codes[:, 1::8], codes[:, 2::8] = 0x7E, 0x01, 0x09   # 448, 2^-9, 2^-6 * 1.125
        w = np.zeros((out, n), np.uint8)
        w[:, ::8], w[:, 1::8], w[:, 2::8] = 2, 1, 7
        w[:, 8::16] = 10                                                     # -1: the large ones cancel
        one = np.full((rows, n // 32), 127, np.uint8)
        c = Case(0, rows, n, out, FP8)
        c.x, c.w = (codes, one, values(codes, one, FP8)), (w, one[:1].repeat(out, 0), values(w, one[:1].repeat(out, 0), FP4))
        want = c.x[2] @ c.w[2].T
        assert np.array_equal(c.run(gpu, F32).astype(np.float64), want)


# ---------------------------------------------------------------------------
# SwiGLU
# ---------------------------------------------------------------------------
def _swiglu(F, c, fmt, gap=0):
    x, w = Mx(F, c.fmt, c.rows, c.n, *c.x[:2]), Mx(F, FP4, c.out, c.n, *c.w[:2])
    y = Mx(F, fmt, c.rows, c.out // 2, gap=gap, gap_scales=gap // 4)
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx, True)
    ws = F.DeviceBuffer(max(1, need))
    ws.fill(0xFF)
    db = None if c.bias is None else buf(F, c.bias)
    F.mx_matmul_swiglu_dev(w.mx, x.mx, y.mx, ws, need, d_bias=db)
    F.synchronize()
    return y


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("to", [FP8, FP4])
@pytest.mark.parametrize("rows,n,out", [(1, 512, 128), (5, 96, 384), (20, 1024, 640), (70, 288, 256), (130, 544, 384), (300, 512, 1280)])
def test_swiglu(gpu, rows, n, out, to, fmt):
    c = Case(rows + n, rows, n, out, fmt, bias=rows % 2 == 0)
    codes, s = _swiglu(gpu, c, to, gap=16 if rows == 5 else 0).read()
    y = c.exact(F32)
    val, gate = y[:, :out // 2], y[:, out // 2:]
    act = val * gate / (1 + np.exp(-gate))
    # the products' error (FP8 rows are summed as for 16 bits), through silu (slope at most 1.1) and val, and six roundings
    b, _ = _product_bound(c.x[2], c.w[2], BF16, fmt == FP8, y)
    b = b + 2.0 ** -23 * np.abs(y)
    tol = np.abs(gate) * b[:, :out // 2] + 1.1 * np.abs(val) * b[:, out // 2:] + 1.1 * b[:, :out // 2] * b[:, out // 2:]
    tol = tol + np.abs(act) * (8 + np.abs(gate)) * 2.0 ** -23
    amax, blocks = np.abs(act).reshape(rows, -1, 32), tol.reshape(rows, -1, 32)
    lo, hi = scale_bytes(np.maximum(amax - blocks, 0).max(-1), to), scale_bytes((amax + blocks).max(-1), to)
    assert ((s >= lo) & (s <= hi)).all()
    half = np.maximum(np.abs(act) * (2.0 ** -2 if to == FP4 else 2.0 ** -4), (0.25 if to == FP4 else 2.0 ** -10) * np.repeat(unit(s), 32, 1))
    off = np.abs(values(codes, s, to) - act)
    assert (off <= half + 1.25 * tol).all(), float((off - half - 1.25 * tol).max())
