"""Microscaled (MX) rows and their products in 64 bits, from the formats' definitions, and device copies of them."""
import numpy as np

from seqs_ref import BF16, F16, F32, from_type, to_type

FP4, FP8 = 1, 2
TOP = {FP4: 6.0, FP8: 448.0}
# half a step of each type, relative (fp16 and bf16 rows of results)
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _code_values(fmt):
    if fmt == FP4:
        a = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    else:
        c = np.arange(128)
        e, f = c >> 3, c & 7
        a = np.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7.0), f * 2.0 ** -9)
        a[127] = np.nan
    return np.concatenate([a, -a])


VALUES = {FP4: _code_values(FP4), FP8: _code_values(FP8)}


def scale_bytes(amax, fmt):
    """The least s >= 0 with amax <= top * 2^(s - 127); 255 for NaN and infinity."""
    amax = np.asarray(amax, np.float64)
    m, e = np.frexp(np.where(np.isfinite(amax), amax, 1.0))
    tm, te = np.frexp(TOP[fmt])
    s = np.where(amax > 0, e - te + (m > tm) + 127, 0)
    return np.where(np.isfinite(amax), np.maximum(s, 0), 255).astype(np.uint8)


def unit(s):
    s = np.asarray(s, np.int64)
    return np.where(s == 255, np.nan, np.ldexp(1.0, np.minimum(s, 254) - 127))


def quantize(x, fmt):
    """Codes (one to a byte) and scale bytes of rows x, to the nearest code, ties to the even one."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[0], -1, 32)
    s = scale_bytes(np.abs(b).max(-1), fmt)
    with np.errstate(all="ignore"):
        y = np.where((s == 255)[..., None], 0.0, b / np.where(s == 255, 1.0, unit(s))[..., None]).reshape(x.shape)
    half = len(VALUES[fmt]) // 2
    grid = VALUES[fmt][:half] if fmt == FP4 else VALUES[fmt][:half - 1]
    mid = (grid[1:] + grid[:-1]) / 2
    a = np.abs(y)
    code = np.searchsorted(mid, a, side="left")                      # a tie stays at the lower code ...
    tie = (code < len(mid)) & (a == mid[np.minimum(code, len(mid) - 1)])
    code = np.where(tie & (code % 2 == 1), code + 1, code)           # ... unless that is odd
    return (code + half * np.signbit(y)).astype(np.uint8), s


def values(codes, s, fmt):
    v = VALUES[fmt][codes]
    with np.errstate(all="ignore"):
        return (v.reshape(v.shape[0], -1, 32) * unit(s)[..., None]).reshape(v.shape)


def pack(codes, fmt):
    return codes if fmt == FP8 else codes[:, ::2] | codes[:, 1::2] << 4


def unpack(raw, fmt):
    return raw if fmt == FP8 else np.stack([raw & 15, raw >> 4], -1).reshape(raw.shape[0], -1)


def strides(fmt, n):
    return (n // 2 if fmt == FP4 else n), (n // 32 + 3) // 4 * 4


class Mx:
    """MX rows on the device: gaps between rows hold `pad`."""

    def __init__(self, F, fmt, rows, n, codes=None, s=None, gap=0, gap_scales=0, pad=0xFF):
        self.F, self.fmt, self.rows, self.n = F, fmt, rows, n
        w, ws = strides(fmt, n)
        self.ld, self.lds = w + gap, ws + gap_scales
        raw, sc = np.full((rows, self.ld), pad, np.uint8), np.full((rows, self.lds), pad, np.uint8)
        if codes is not None:
            raw[:, :w], sc[:, :n // 32] = pack(codes, fmt), s
        self.dc, self.ds = F.DeviceBuffer.from_array(raw), F.DeviceBuffer.from_array(sc)
        self.pad = pad

    @property
    def mx(self):
        return self.F.mx(self.fmt, self.rows, self.n, self.dc, self.ds, self.ld, self.lds)

    def read(self):
        """Codes and scale bytes; what stands between rows must be as it was."""
        raw, sc = self.dc.download(np.uint8, (self.rows, self.ld)), self.ds.download(np.uint8, (self.rows, self.lds))
        w = strides(self.fmt, self.n)[0]
        assert (raw[:, w:] == self.pad).all() and (sc[:, self.n // 32:] == self.pad).all()
        return unpack(raw[:, :w], self.fmt), sc[:, :self.n // 32]


def random_rows(rng, rows, n, fmt, spread=2.0):
    """Codes, scales and values of rows whose blocks differ in size."""
    x = rng.standard_normal((rows, n)) * np.repeat(np.exp2(rng.uniform(-spread, spread, (rows, n // 32))), 32, 1)
    c, s = quantize(x, fmt)
    return c, s, values(c, s, fmt)


def buf(F, a):
    return F.DeviceBuffer.from_array(a)


__all__ = ["BF16", "F16", "F32", "from_type", "to_type", "FP4", "FP8", "HALF", "VALUES", "Mx", "buf", "quantize", "random_rows",
           "scale_bytes", "strides", "unit", "unpack", "values"]
