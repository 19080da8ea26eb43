"""64-bit plain forms of the packed-sequence and key/value-cache calls
(include/fh3/fh3_hip.h), and the bounds their results are held to."""
import math

import numpy as np

PAGE = 64
F32, F16, BF16 = 0, 1, 30          # FH3_QUANT_*
NAMES = {F32: "F32", F16: "F16", BF16: "BF16"}
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # half a step, relative


def to_type(x, t):
    """fp32 values -> the stored array of a type (BF16 as uint16), rounded to nearest even."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if t == F32:
        return x
    if t == F16:
        return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_type(a, t):
    """A stored array -> float64 values, exactly."""
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def head_outputs(q, k, v, pos, scale, cap, slope, see):
    """One head: (o, weighted |v|, largest sum |q_i k_i| * scale) for rows at
    positions pos; see [rows][keys] says which keys a row sees.  A key that is
    not seen counts for nothing, whatever it holds."""
    seen_k = see.any(0)
    kk = np.where(seen_k[:, None], k, 0.0)
    s = (q @ kk.T) * scale
    if cap:
        s = cap * np.tanh(s / cap)
    if slope is not None:
        s = s - slope * np.abs(pos[:, None] - np.arange(k.shape[0])[None, :])
    s = np.where(see, s, -np.inf)
    top = s.max(1, keepdims=True, initial=-np.inf)
    w = np.exp(s - np.where(np.isinf(top), 0.0, top))
    w = np.where(see, w, 0.0)
    total = w.sum(1, keepdims=True)
    w = w / np.where(total == 0, 1.0, total)
    vv = np.where(seen_k[:, None], v, 0.0)
    big = (np.abs(q) @ np.abs(kk).T * scale * see).max(initial=0.0)
    return w @ vv, w @ np.abs(vv), big


def attention(q, k, v, first, heads, kv, hd, causal=True, scale=None, cap=0.0, slopes=None, prefix=None):
    """Packed sequences: q [n][heads*hd], k, v [n][kv*hd] float64.  Returns o, the weighted |v| and the
    largest score's sum of |products|; rows of no sequence are zero."""
    o, a, big = np.zeros_like(q), np.zeros_like(q), 0.0
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    for s in range(len(first) - 1):
        r = slice(first[s], first[s + 1])
        n = max(0, first[s + 1] - first[s])
        i, j = np.arange(n)[:, None], np.arange(n)[None, :]
        see = (j <= i) if causal else np.ones((n, n), bool)
        if prefix is not None:
            see = see | (j < prefix[s])
        for h in range(heads):
            hc, kc = slice(h * hd, (h + 1) * hd), slice(h // (heads // kv) * hd, (h // (heads // kv) + 1) * hd)
            o[r, hc], a[r, hc], b = head_outputs(q[r, hc], k[r, kc], v[r, kc], np.arange(n), scale, cap,
                                                 None if slopes is None else float(slopes[h]), see)
            big = max(big, b)
    return o, a, big


def bound(t, o, a, big, hd, keys):
    """How far an output may be from the 64-bit one, elementwise.  With u half a
    step of the type: the weights are rounded once (u of the weighted |v|), their
    sum is taken of rounded or exact weights (u |o|), the output is rounded once
    (u |o|).  F32 operands are two 16-bit terms each: weights and values lose
    2^-16 each and the product of the two low terms (2^-16) is left out.  Scores
    are fp32 sums of hd products, at most hd 2^-24 of their sum of |products|
    (F32: and 3 * 2^-22 of it for the split), and exp2, tanh and the scale add a
    few 2^-24 of the score; a score that is off by d changes weights by a
    factor exp(2 d) at most.  The fp32 sum over the keys adds 2^-24 for every step
    of 16 keys and 16 within one."""
    u = UNIT[t]
    d = (hd + 16) * 2.0 ** -24 * (big + 1) + (3 * 2.0 ** -22 * big if t == F32 else 0)
    weights = 3 * 2.0 ** -16 if t == F32 else u
    return (weights + 2 * d + (keys / 16 + 16) * 2.0 ** -24) * a + 2 * u * np.abs(o) + 1e-30


#: relative Frobenius error: rounding errors are uniform, so each contributes at most u / sqrt(3); the weights',
#: the sum's and the output's together stay below 1.8 u / sqrt(3) ~ u (F32: three terms of 2^-16 / sqrt(3) at
#: worst, of which the low terms' own rounding is seldom near its limit).
FRO = {F32: 1e-5, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def check(got, t, o, a, big, hd, keys, what, floor=0.0):
    got = from_type(got, t)
    off = np.abs(got - o)
    lim = bound(t, o, a, big, hd, keys) + floor
    worst = float((off / lim).max(initial=0.0))
    norm = np.linalg.norm(o)
    fro = float(np.linalg.norm(got - o) / norm) if norm else float(off.max(initial=0.0))
    print("%s %s: worst %.3f of its bound, rel_fro %.2e" % (what, NAMES[t], worst, fro), flush=True)
    assert np.isfinite(got).all()
    assert worst <= 1.0, (what, worst)
    assert fro <= FRO[t], (what, fro)


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------
def k_index(hd):
    """[64][hd] -> byte of K."""
    t, d = np.arange(PAGE)[:, None], np.arange(hd)[None, :]
    return ((t // 16 * (hd // 64) + d // 64) * 4 + d % 64 // 16) * 256 + t % 16 * 16 + d % 16


def v_index(hd):
    t, d = np.arange(PAGE)[:, None], np.arange(hd)[None, :]
    return (d // 16 * 4 + t % 16 // 4) * 256 + d % 16 * 16 + t // 16 * 4 + t % 4


def scale_of(amax):
    """The least 2^e >= 2^-100 with amax <= 127 2^e."""
    e = -100
    if amax > 0:
        m, x = math.frexp(amax)
        e = max(-100, x - 7 if m <= 127 / 128 else x - 6)
    return 2.0 ** e


def quantise(x, scale):
    with np.errstate(over="ignore", invalid="ignore"):
        q = np.clip(np.rint(x / scale), -127, 127)
    return np.where(np.isnan(x), 0, q)


class Cache:
    """The cache's rules on host arrays: q [pages][kv][2][64][hd] and scales [pages][kv][2]."""

    def __init__(self, kv, hd, pages, table, rng):
        self.kv, self.hd, self.pages, self.table = kv, hd, pages, np.asarray(table)
        self.q = rng.integers(-127, 128, (pages, kv, 2, PAGE, hd)).astype(np.float64)
        self.scale = 2.0 ** rng.integers(-9, -4, (pages, kv, 2))

    def pool(self):
        """The device bytes."""
        raw = np.zeros((self.pages, self.kv, 2, PAGE * self.hd), np.uint8)
        for w, ix in ((0, k_index(self.hd)), (1, v_index(self.hd))):
            raw[:, :, w, ix.ravel()] = (self.q[:, :, w].reshape(self.pages, self.kv, -1) + 128).astype(np.uint8)
        return np.concatenate([raw.ravel(), self.scale.astype(np.float32).ravel().view(np.uint8)])

    def page(self, s, p):
        if not 0 <= p < self.table.shape[1]:
            return -1
        i = int(self.table[s, p])
        return i if 0 <= i < self.pages else -1

    def append(self, rows, first, lens):
        """rows: (k, v) float64 [n][kv * hd]."""
        for s in range(len(first) - 1):
            cnt = first[s + 1] - first[s]
            base = lens[s] - cnt
            for p in range(base // PAGE, (lens[s] - 1) // PAGE + 1 if cnt else base // PAGE):
                i = self.page(s, p)
                if i < 0:
                    continue
                lo, hi = max(base, p * PAGE), min(lens[s], (p + 1) * PAGE)
                for w, x in enumerate(rows):
                    part = x[first[s] + lo - base:first[s] + hi - base].reshape(hi - lo, self.kv, self.hd)
                    for h in range(self.kv):
                        y = part[:, h]
                        fine = np.abs(y[np.isfinite(y)])
                        now = scale_of(fine.max(initial=0.0))
                        held = lo - p * PAGE
                        if held:
                            before = self.scale[i, h, w]
                            now = max(now, before)
                            self.q[i, h, w, :held] = np.rint(self.q[i, h, w, :held] * (before / now))
                        self.scale[i, h, w] = now
                        self.q[i, h, w, held:held + hi - lo] = quantise(y, now)

    def values(self, s, lo, hi):
        """K and V of positions lo .. hi - 1, [hi-lo][kv][hd] each, and which are held."""
        out, there = np.zeros((2, hi - lo, self.kv, self.hd)), np.zeros(hi - lo, bool)
        for j in range(lo, hi):
            i = self.page(s, j // PAGE) if j >= 0 else -1
            if i >= 0:
                there[j - lo] = True
                out[:, j - lo] = (self.q[i, :, :, j % PAGE] * self.scale[i][..., None]).transpose(1, 0, 2)
        return out[0], out[1], there

    def read(self, first, lens):
        out = np.zeros((2, first[-1], self.kv * self.hd))
        for s in range(len(first) - 1):
            n = first[s + 1] - first[s]
            k, v, _ = self.values(s, lens[s] - n, lens[s])
            w = self.kv * self.hd
            out[0, first[s]:first[s + 1]], out[1, first[s]:first[s + 1]] = k.reshape(n, w), v.reshape(n, w)
        return out

    def attention(self, q, first, lens, heads, causal=True, scale=None, cap=0.0, slopes=None):
        o, a, big = np.zeros_like(q), np.zeros_like(q), 0.0
        kv, hd = self.kv, self.hd
        scale = 1.0 / math.sqrt(hd) if scale is None else scale
        for s in range(len(first) - 1):
            n = first[s + 1] - first[s]
            held = min(lens[s], self.table.shape[1] * PAGE)
            k, v, there = self.values(s, 0, held)
            pos = lens[s] - n + np.arange(n)
            see = np.broadcast_to(there[None, :], (n, held))
            if causal:
                see = see & (np.arange(held)[None, :] <= pos[:, None])
            for h in range(heads):
                hc, m = slice(h * hd, (h + 1) * hd), h // (heads // kv)
                r = slice(first[s], first[s + 1])
                o[r, hc], a[r, hc], b = head_outputs(q[r, hc], k[:, m], v[:, m], pos, scale, cap,
                                                     None if slopes is None else float(slopes[h]), see)
                big = max(big, b)
        return o, a, big
