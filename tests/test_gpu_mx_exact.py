"""Products of microscaled rows where every partial sum, in whatever order, has an fp32 number of its own: outputs of each
type are then the exact sums, rounded once, whichever kernel serves the call.  Within a group of eight the largest codes
cancel beside the smallest ones of both parts that FP8 codes are split into (448 * 6 beside 2.25 * 0.5, and 2^-9 * 0.5),
so sums that keep fewer bits come out wrong."""
import numpy as np
import pytest

from mx_ref import BF16, F16, F32, FP4, FP8, Mx, buf, from_type, quantize, to_type, values
from test_gpu_mx_calls import test_swiglu_codes_are_those_of_exact_sums as codes_of_exact_sums

pytestmark = pytest.mark.gpu

GATES = 8          # codes of a row that SwiGLU's gates are made of: the second group of eight


def _base(rng, rows, n, out, fmt, swiglu):
    """Codes of a few rows of x and W.  FP8: all sums of magnitudes stay below 2^14, and every product is a multiple of 2^-10:
    24 bits.  FP4: below 2^20, multiples of 2^-2."""
    wv = out // 2 if swiglu else out
    w = rng.integers(0, 16, (wv, n)).astype(np.uint8)
    if fmt == FP4:
        x = rng.integers(0, 16, (rows, n)).astype(np.uint8)
    else:
        x = (rng.integers(0, 16, (rows, n)) | rng.integers(0, 2, (rows, n)) << 7).astype(np.uint8)       # up to 1.875 * 2^-6
        top = rng.choice(np.array([0x7E, 0x7D, 0x7C, 0x78], np.uint8), (rows, 1))
        v = rng.choice(np.array([7, 6, 5], np.uint8), (wv, 1))
        for k, at in enumerate((0, n - 8)):
            x[:, at:at + 2] = top
            w[:, at + k:at + k + 1], w[:, at + 1 - k:at + 2 - k] = v, v | 8
            x[:, at + 2:at + 4] = rng.integers(0x40, 0x48, (rows, 2))          # 2 to 3.75
            w[:, at + 2:at + 4] = rng.choice(np.array([1, 9, 3, 11], np.uint8), (wv, 2))
            x[:, at + 4:at + 8] = rng.integers(0x01, 0x40, (rows, 4))          # up to 1.875
    if swiglu:
        x[:, GATES:GATES + 8] = 0x58 if fmt == FP8 else 6                      # 16, 4
        w[:, GATES:GATES + 8] = 0
        g = np.zeros((wv, n), np.uint8)
        g[:, GATES:GATES + 8] = 6                                              # 4: sums of 512, 128
        w = np.concatenate([w, g])
    return x, w


class Exact:
    """rows x n -> out: base rows again and again, copy k of those of x with 2^(k % 5) times the scales (W: % 7)."""

    def __init__(self, F, rows, n, out, fmt, swiglu=False, base=40):
        rng = np.random.default_rng(rows + n + out)
        self.F, self.rows, self.n, self.out, self.fmt = F, rows, n, out, fmt
        half = out // 2 if swiglu else out
        bx, bw = min(rows, base), min(half, base)
        x, w = _base(rng, bx, n, 2 * bw if swiglu else bw, fmt, swiglu)
        e = rng.integers(-30, 30, n // 32)
        xv, wv = values(x, np.full((len(x), n // 32), 127), fmt), values(w, np.full((len(w), n // 32), 127), FP4)
        size, step = (np.abs(xv) @ np.abs(wv).T).max(), 2.0 ** (-10 if fmt == FP8 else -2)
        assert size < step * 2 ** 24
        down = 0 if swiglu else 10
        ix, iw = np.arange(rows) % bx, np.arange(half) % bw
        px, pw = np.arange(rows) // bx % 5, np.arange(half) // bw % 7
        if swiglu:
            iw, pw = np.concatenate([iw, iw + bw]), np.concatenate([pw, pw])
        y = xv @ wv.T
        self.y = y[np.ix_(ix, iw)] * np.exp2(px[:, None] + pw[None] - down)
        self.x = Mx(F, fmt, rows, n, x[ix], (127 + e[None] + px[:, None] - down).astype(np.uint8))
        self.w = Mx(F, FP4, out, n, w[iw], (127 - e[None] + pw[:, None]).astype(np.uint8))

    def workspace(self, swiglu):
        need = self.F.mx_matmul_workspace_bytes(self.w.mx, self.x.mx, swiglu)
        ws = self.F.DeviceBuffer(max(1, need))
        ws.fill(0xFF)
        return ws, need


# few rows with one, two and four tiles of tokens, one to four of weight rows, with and without a window loaded ahead; streamed weights,
# whole and in parts of the rows' length; tiles of 128 and of 256, whole, in parts, and with a last round of smaller ones
SIZES = [(1, 32, 1), (1, 512, 40), (3, 8224, 300), (5, 544, 5003), (16, 288, 9700), (20, 352, 64), (30, 1056, 4900), (50, 544, 70),
         (1, 5088, 15361), (17, 5088, 15361), (40, 5088, 15361), (40, 1056, 130001), (1, 25632, 5130), (17, 25632, 5130), (40, 25632, 5130), (64, 2080, 40003),
         (70, 352, 100), (300, 1056, 260), (600, 4128, 520), (422, 16480, 5532), (154, 19040, 12387), (1930, 1824, 4401), (2100, 1824, 8101)]


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("rows,n,out", SIZES)
def test_products(gpu, rows, n, out, t, fmt):
    c = Exact(gpu, rows, n, out, fmt)
    kind = to_type(np.zeros(1, np.float32), t).dtype
    y, (ws, need) = buf(gpu, np.full((rows, out), 77, kind)), c.workspace(False)
    gpu.mx_matmul_dev(c.w.mx, c.x.mx, t, y, ws, need)
    gpu.synchronize()
    with np.errstate(over="ignore"):
        got, want = from_type(y.download(kind, (rows, out)), t), from_type(to_type(c.y.astype(np.float32), t), t)
    assert np.array_equal(got, want), (np.argwhere(got != want)[:3], (got != want).mean())


SWIGLU = [(1, 512, 128), (5, 96, 384), (20, 1024, 640), (50, 544, 512), (1, 5088, 40064), (19, 5088, 40064), (40, 5088, 40064),
          (64, 2080, 40064), (1, 13856, 20096), (12, 13856, 20096), (30, 13856, 20096), (60, 13856, 20096), (70, 352, 128), (130, 1056, 640),
          (300, 4096, 1280), (422, 16480, 5504), (154, 19040, 12416), (1930, 1824, 4480), (2100, 1824, 8192)]


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("to", [FP8, FP4])
@pytest.mark.parametrize("rows,n,out", SWIGLU)
def test_swiglu(gpu, rows, n, out, to, fmt):
    """Gates of 128 and more, powers of two, where silu(g) is g: codes and scales are those of the exact products."""
    c = Exact(gpu, rows, n, out, fmt, swiglu=True)
    val, gate = c.y[:, :out // 2], c.y[:, out // 2:]
    assert (gate >= 128).all() and (np.frexp(gate)[0] == 0.5).all()
    y, (ws, need) = Mx(gpu, to, rows, out // 2), c.workspace(True)
    gpu.mx_matmul_swiglu_dev(c.w.mx, c.x.mx, y.mx, ws, need)
    gpu.synchronize()
    got, want = y.read(), quantize(val * gate, to)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])


# gates from where exp(g) leaves fp32's normal numbers on, beside values that bring the result back among the codes
FAR = [(1.0, -87.4, 4.0), (-3.0, -92.0, 3.0), (2.0 ** 40, -110.0, 20.0), (-(2.0 ** 100), -150.0, 20.0), (3e38, -186.0, 30.0), (1.0, -20.0, 40.0),
       (2.0 ** -20, -80.0, 12.0), (1e38, -400.0, 100.0)]


@pytest.mark.parametrize("to", [FP8, FP4])
@pytest.mark.parametrize("rows,n,out", [(1, 96, 1024), (19, 5088, 40064), (12, 13856, 20096), (130, 1056, 1280), (300, 4096, 1280), (1930, 1824, 4480)])
def test_swiglu_of_far_negative_gates(gpu, rows, n, out, to):
    """Rows of zeros and a bias that holds values and gates.  Relative errors: exp2 and the reciprocal a unit in the last place
    (2^-23) each, seven roundings of 2^-24; below 2^-126 two steps of 2^-149."""
    f, rng = out // 2, np.random.default_rng(out)
    kind = np.arange(f) // 32 % len(FAR)
    v, g, w = (np.array([c[i] for c in FAR])[kind] for i in range(3))
    bias = np.concatenate([v, g - w * rng.random(f)]).astype(np.float32)
    x = Mx(gpu, FP8, rows, n, np.zeros((rows, n), np.uint8), np.full((rows, n // 32), 127, np.uint8))
    wm = Mx(gpu, FP4, out, n, rng.integers(0, 16, (1, n)).astype(np.uint8).repeat(out, 0), np.full((out, n // 32), 127, np.uint8))
    y, need = Mx(gpu, to, rows, f), gpu.mx_matmul_workspace_bytes(wm.mx, x.mx, True)
    ws = gpu.DeviceBuffer(max(1, need))
    gpu.mx_matmul_swiglu_dev(wm.mx, x.mx, y.mx, ws, need, d_bias=buf(gpu, bias))
    gpu.synchronize()
    codes, s = y.read()
    assert (codes == codes[:1]).all() and (s == s[:1]).all()
    b = bias.astype(np.float64)
    act = (b[:f] * b[f:] / (1 + np.exp(-b[f:])))[None]
    off = np.abs(act) * 2.0 ** -20 + 2.0 ** -148
    low, high = quantize(np.sign(act) * (np.abs(act) - off).clip(0), to), quantize(np.sign(act) * (np.abs(act) + off), to)
    assert ((s[:1] >= low[1]) & (s[:1] <= high[1])).all()
    sure = np.repeat(low[1] == high[1], 32, 1)
    a, lo, hi = (np.abs(values(*c, to)) for c in ((codes[:1], s[:1]), low, high))
    assert ((a >= lo) & (a <= hi))[sure].all() and sure.mean() > 0.9
    assert codes[0].reshape(-1, 32).any(1)[kind[::32] < 4].all()


@pytest.mark.parametrize("to", [FP8, FP4])
@pytest.mark.parametrize("modulate", [False, True])
def test_norm_past_fp32(gpu, modulate, to):
    """Values that fp32 cannot hold (through a weight, or a modulation) make their block NaN, as infinities do, and no other."""
    rows, n = 3, 256
    x, w = np.ones((rows, n), np.float32), np.ones(n, np.float32)
    x[1], x[1, 40] = 0, 4                                     # 16 after the norm
    w[40] = 3e37
    scale, shift = np.zeros((rows, n), np.float32), np.zeros((rows, n), np.float32)
    if modulate:
        w[40], scale[1, 40], shift[2, 200], scale[2, 200] = 1, 3e37, -3e38, -3e38
    y, d = Mx(gpu, to, rows, n), [buf(gpu, a) for a in (x, w, shift, scale)]
    gpu.mx_norm_dev(F32, d[0], d[1], 0.0, y.mx, d_shift=d[2] if modulate else None, d_scale=d[3] if modulate else None)
    gpu.synchronize()
    codes, s = y.read()
    nan = np.zeros(s.shape, bool)
    nan[1, 1], nan[2, 6] = True, modulate
    assert np.array_equal(s == 255, nan) and not codes[np.repeat(nan, 32, 1)].any()
    e = x / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True)) * w.astype(np.float64)
    want = quantize(np.where(np.repeat(nan, 32, 1), 0, e * (1 + scale.astype(np.float64)) + shift), to)
    assert np.array_equal(s[~nan], want[1][~nan]) and np.array_equal(codes[~np.repeat(nan, 32, 1)], want[0][~np.repeat(nan, 32, 1)])


@pytest.mark.parametrize("rows,n,out", [(19, 5088, 40064), (40, 5088, 40064), (12, 13856, 20096), (30, 13856, 20096), (422, 16480, 5504)])
def test_swiglu_codes_of_random_rows(gpu, rows, n, out):
    """Streamed weights, whole and in parts, and large tiles in parts: the formula's codes but where fp32 sums leave two."""
    codes_of_exact_sums(gpu, rows, n, out)
