"""The 8-bit key/value cache on the GPU (fh3_hip_kv_extend_dev, _append_dev,
_read_dev, _attention_dev) against its rules on the host, in 64 bits: the stored
integers and scales are equal, attention is held to a derived bound."""
import ctypes

import numpy as np
import pytest

import seqs_ref as R
from seqs_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu


def _offsets(lens):
    return [0] + list(np.cumsum(lens))


class Held:
    """A cache on the device beside its model on the host."""

    def __init__(self, F, kv, hd, lens, seed, spare=2, max_pages=None, pages=None, table=None):
        rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // R.PAGE) for n in lens]
        most = max(1, max(need)) if max_pages is None else max_pages
        pages = sum(need) + spare if pages is None else pages
        if table is None:
            order = iter(rng.permutation(pages))
            table = np.full((len(lens), most), -1, np.int64)
            for s, n in enumerate(need):
                for p in range(min(n, most)):
                    table[s, p] = next(order)
        self.F, self.lens = F, list(lens)
        self.model = R.Cache(kv, hd, pages, table, rng)
        pool = self.model.pool()
        assert pool.nbytes == F.kv_pool_bytes(kv, hd, pages)
        self.pool = F.DeviceBuffer.from_array(pool)
        self.table = F.DeviceBuffer.from_array(np.asarray(table, np.int32))
        self.len = F.DeviceBuffer.from_array(np.asarray(lens, np.int32))
        self.kv = F.kv_cache(kv, hd, pages, most, self.pool, self.table, self.len)

    def append(self, t, k, v, first, **kw):
        F, model = self.F, self.model
        dk, dv, df = (F.DeviceBuffer.from_array(x) for x in (k, v, np.asarray(first, np.int32)))
        F.kv_append_dev(self.kv, t, dk, dv, k.shape[0], len(first) - 1, df, **kw)
        F.synchronize()
        model.append((R.from_type(k, t), R.from_type(v, t)), first, self.lens)

    def same(self):
        """The held tokens' integers and scales are the model's."""
        m = self.model
        got = self.pool.download(np.uint8, (self.pool.nbytes,))
        n = m.pages * m.kv * 2 * R.PAGE * m.hd
        raw, sc = got[:n].reshape(m.pages, m.kv, 2, -1), got[n:].view(np.float32).reshape(m.pages, m.kv, 2)
        for s, length in enumerate(self.lens):
            for p in range(-(-length // R.PAGE)):
                i, tok = m.page(s, p), min(R.PAGE, length - p * R.PAGE)
                if i < 0:
                    continue
                assert np.array_equal(sc[i], m.scale[i].astype(np.float32)), (s, p)
                for w, ix in ((0, R.k_index(m.hd)), (1, R.v_index(m.hd))):
                    q = raw[i, :, w][:, ix[:tok].ravel()].astype(np.int64) - 128
                    assert np.array_equal(q, m.q[i, :, w, :tok].reshape(m.kv, -1)), (s, p, w)

    def read(self, t, first, n=None):
        F, m = self.F, self.model
        n = first[-1] if n is None else n
        out = [R.to_type(np.full((n, m.kv * m.hd), 5), t) for _ in "kv"]
        dk, dv, df = (F.DeviceBuffer.from_array(x) for x in (*out, np.asarray(first, np.int32)))
        F.kv_read_dev(self.kv, t, dk, dv, n, len(first) - 1, df)
        F.synchronize()
        return [b.download(out[0].dtype, out[0].shape) for b in (dk, dv)]

    def attend(self, t, q, first, heads, rows=None, slopes=None, ws=None, **cfg):
        F, m = self.F, self.model
        ds = None if slopes is None else F.DeviceBuffer.from_array(np.asarray(slopes, np.float32))
        c = F.attn_cfg(heads, m.kv, m.hd, t, d_slopes=ds, **cfg)
        rows = q.shape[0] if rows is None else rows
        need = F.kv_attention_workspace_bytes(c, self.kv, rows, len(first) - 1)
        if ws is None:
            ws = F.DeviceBuffer(max(1, need))
            ws.fill(0xFF)      # what an earlier use may have left: NaN
        dq, df = F.DeviceBuffer.from_array(q), F.DeviceBuffer.from_array(np.asarray(first, np.int32))
        do = F.DeviceBuffer.from_array(np.full_like(q, 7))
        F.kv_attention_dev(c, self.kv, dq, do, rows, len(first) - 1, ws, need, df)
        F.synchronize()
        return do.download(q.dtype, q.shape)

    def check_attend(self, t, q, first, heads, what, slopes=None, causal=True, softcap=0.0):
        got = self.attend(t, q, first, heads, slopes=slopes, causal=causal, softcap=softcap)
        o, a, big = self.model.attention(R.from_type(q, t), first, self.lens, heads, causal, None, softcap, slopes)
        n, m = first[-1], self.model
        # Weights enter as fp16 (F32: two terms), whose least step is 2^-24: each is off by up to 2^-25 more where it
        # is small, beside a largest of at least 2^6, so the output by 2^-31 of the sum of the |v| of all keys.  That
        # matters where the key that a row is about has a 0 in a channel.
        vs = [m.values(s, 0, n_k)[1] for s, n_k in enumerate(self.lens)]
        floor = np.zeros_like(o)
        for s, v in enumerate(vs):
            floor[first[s]:first[s + 1]] = np.repeat(np.abs(v).sum(0), heads // m.kv, 0).ravel() * 2.0 ** -31 if len(v) else 0
        R.check(got[:n], t, o[:n], a[:n], big, m.hd, max(self.lens), what, floor[:n])
        return got


def _rows(seed, t, n, width, scale=1.0):
    x = np.random.default_rng(seed).standard_normal((n, width)) * scale
    return R.to_type(x, t)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("kv,hd", [(1, 64), (8, 128), (3, 64)])
def test_append_to_empty_and_read(gpu, t, kv, hd):
    lens = [1, 63, 64, 65, 200, 0]
    h = Held(gpu, kv, hd, lens, 3)
    first = _offsets(lens)
    k, v = _rows(1, t, first[-1], kv * hd, 0.7), _rows(2, t, first[-1], kv * hd, 30.0)
    h.append(t, k, v, first)
    h.same()
    for got, want in zip(h.read(t, first), h.model.read(first, lens)):
        assert np.array_equal(R.from_type(got, t), want)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 300.0])
def test_append_behind_held_tokens(gpu, t, scale):
    """Small new values keep the pages' scales, large ones raise them and the held tokens are rounded again."""
    kv, hd, held, new = 2, 128, [0, 10, 63, 64, 100, 190, 5], [3, 1, 1, 1, 130, 2, 0]
    lens = [a + b for a, b in zip(held, new)]
    h = Held(gpu, kv, hd, lens, 4)
    first = _offsets(new)
    k, v = _rows(5, t, first[-1], kv * hd, scale), _rows(6, t, first[-1], kv * hd, scale)
    h.append(t, k, v, first)
    h.same()
    before = h.pool.download(np.uint8, (h.pool.nbytes,))
    h.append(t, k, v, first)            # again: nothing changes
    h.same()
    assert np.array_equal(before, h.pool.download(np.uint8, (h.pool.nbytes,)))


def test_values_not_finite_and_extremes(gpu):
    kv, hd = 1, 64
    x = _rows(7, F32, 8, hd)
    x[0, 3], x[1, 5], x[2, 7] = np.nan, np.inf, -np.inf
    x[3], x[4] = 0, np.float32(3.4e38)
    x[5], x[6, :] = np.float32(1e-42), -0.0
    for rows in ([0, 1, 2, 3], [3], [4], [5], [6], [4, 5], [0, 1, 2]):
        h = Held(gpu, kv, hd, [len(rows)], 8)
        h.append(F32, x[rows], x[rows][::-1].copy(), [0, len(rows)])
        h.same()
    bad = np.full((2, hd), np.nan, np.float32)    # nothing finite: the least scale
    h = Held(gpu, kv, hd, [2], 9)
    h.append(F32, bad, np.full((2, hd), np.inf, np.float32), [0, 2])
    h.same()
    k, v = h.read(F32, [0, 2])
    assert (k == 0).all() and (v == 127 * 2.0 ** -100).all()


def test_scale_border(gpu):
    """Largest values just below, at and above 127 times a power of two."""
    hd = 64
    for e in (-30, 0, 9):
        for off in (-1, 0, 1):
            top = np.float32(127 * 2.0 ** e)
            top = np.nextafter(top, np.float32(off) * np.float32(np.inf)) if off else top
            x = np.zeros((1, hd), np.float32)
            x[0, 9], x[0, 10], x[0, 11] = -top, top / 254, top * 3 / 254   # ties, to even
            h = Held(gpu, 1, hd, [1], 1)
            h.append(F32, x, -x, [0, 1])
            h.same()
            assert h.model.scale[h.model.table[0, 0], 0, 0] == 2.0 ** (e + (off > 0))


def test_pages_that_hold_nothing(gpu):
    """Table entries outside the pool, lengths past the table and negative ones: not written, read as zeros, not seen."""
    kv, hd, heads = 2, 64, 4
    table = np.asarray([[3, -1, 0], [99, 1, -2 ** 31], [2, 2 ** 31 - 1, 4], [5, 6, 7]])
    lens = [190, 150, 70, 250]
    h = Held(gpu, kv, hd, lens, 10, pages=9, table=table, max_pages=3)
    new = [130, 150, 3, 70]
    first = _offsets(new)
    k, v = _rows(11, F32, first[-1], kv * hd), _rows(12, F32, first[-1], kv * hd)
    page = kv * 2 * R.PAGE * hd
    before = h.pool.download(np.uint8, (h.pool.nbytes,))
    h.append(F32, k, v, first)
    h.same()
    after = h.pool.download(np.uint8, (h.pool.nbytes,))
    for i in (1, 8):    # page 1: its sequence's rows end before it; page 8: in no table
        assert np.array_equal(after[i * page:(i + 1) * page], before[i * page:(i + 1) * page]) == (i == 8)
    for got, want in zip(h.read(F32, first), h.model.read(first, lens)):
        assert np.array_equal(got, want)
    h.check_attend(F32, _rows(13, F32, first[-1], heads * hd), first, heads, "holes")
    few = [0, 1, 2, 3, 4]
    h.check_attend(BF16, _rows(13, BF16, 4, heads * hd), few, heads, "holes, one token")
    for lens in ([0, -5, 2, -2 ** 31], [1, 1, 1, 2 ** 31 - 1]):    # more new rows than tokens: the rest see nothing
        h.len.upload(np.asarray(lens, np.int32))
        h.lens = [max(n, 0) for n in lens]
        q = _rows(14, F32, 12, heads * hd)
        if max(lens) < 1000:
            h.check_attend(F32, q, [0, 3, 6, 9, 12], heads, "short")
        else:
            got = h.attend(F32, q, [0, 3, 6, 9, 12], heads)
            assert (got[[0, 1, 3, 4, 6, 7]] == 0).all() and np.isfinite(got).all()
        k, _ = h.read(F32, [0, 3, 6, 9, 12])
        assert (k[:2] == 0).all()


def test_rows_behind_the_last_sequence_stay(gpu):
    kv, hd, heads, lens = 2, 64, 4, [40, 100]
    h = Held(gpu, kv, hd, lens, 15)
    got = h.read(F32, [0, 5, 8], n=12)
    assert all((x[8:] == 5).all() and not (x[:8] == 5).all() for x in got)
    q = _rows(16, F32, 12, heads * hd)
    assert (h.attend(F32, q, [0, 5, 8], heads)[8:] == 7).all()


# heads, kv, hd, lens, new, causal, cap, alibi
ATTEND = [
    (1, 1, 64, [1], [1], True, 0.0, False),
    (64, 8, 128, [300], [1], True, 0.0, False),
    (8, 8, 128, [64, 65, 63, 1], [1, 1, 1, 1], True, 0.0, False),
    (16, 2, 64, [500, 0, 129, 700], [1, 0, 1, 1], True, 0.0, False),
    (10, 2, 128, [129, 1000], [1, 1], True, 50.0, False),
    (16, 2, 128, [700, 300, 64], [2, 4, 2], True, 0.0, True),
    (32, 1, 64, [333, 1500], [1, 1], True, 0.0, False),
    (4, 1, 128, [100, 260], [8, 5], False, 0.0, False),
    (12, 4, 64, [1111, 90], [5, 5], True, 30.0, True),
    (64, 8, 128, [520, 40], [130, 40], True, 0.0, False),
    (40, 8, 128, [600], [77], True, 50.0, False),
    (16, 16, 64, [190, 300], [64, 200], True, 0.0, True),
    (6, 2, 128, [400, 5, 290], [33, 5, 1], False, 20.0, False),
    (128, 1, 64, [150], [7], True, 0.0, False),
    (24, 1, 128, [800, 700, 3], [1, 2, 1], True, 0.0, False),
]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_attention_over_the_cache(gpu, t, i):
    heads, kv, hd, lens, new, causal, cap, alibi = ATTEND[i]
    print("case %d %s lens %s new %s" % (i, R.NAMES[t], lens, new), flush=True)
    h = Held(gpu, kv, hd, lens, 20 + i)
    first = _offsets(new)
    slopes = np.asarray([2.0 ** (-8 * (j + 1) / heads) for j in range(heads)], np.float32) if alibi else None
    q = _rows(21, t, first[-1], heads * hd, 0.4)
    a = h.check_attend(t, q, first, heads, "case %d" % i, slopes, causal, cap)
    b = h.attend(t, q, first, heads, slopes=slopes, causal=causal, softcap=cap)
    assert np.array_equal(a, b)    # the same bits again


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_long_and_ragged(gpu, t, new):
    """Lengths from 1 to some thousands in one call, so that parts of sequences meet in the same workgroup."""
    kv, hd, heads = 2, 64, 8
    lens = [new + x for x in (0, 4000, 3, 900, 64, 1, 2222, 128, 0, 700, 63)]
    h = Held(gpu, kv, hd, lens, 41)
    first = _offsets([new] * len(lens))
    h.check_attend(t, _rows(42, t, first[-1], heads * hd, 1.5), first, heads, "ragged, %d new" % new)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_chunk_of_peaked_scores(gpu, t, hd):
    """Scores that pass the running offset in either half of a page, pages of different value scales."""
    kv, heads, lens, new = 1, 2, [1500, 130], [100, 70]
    h = Held(gpu, kv, hd, lens, 61)
    first = _offsets(new)
    h.check_attend(t, _rows(62, t, first[-1], heads * hd, 8.0), first, heads, "peaked chunk")


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [0.5, 64.0, 65.0, 1e8, 1e30])
def test_caps_of_any_size(gpu, t, cap):
    kv, hd, heads, lens = 2, 64, 4, [150, 70]
    h = Held(gpu, kv, hd, lens, 71)
    for new in (1, 40):
        first = _offsets([new, new])
        h.check_attend(t, _rows(72, t, first[-1], heads * hd), first, heads, "cap %g, %d new" % (cap, new), softcap=cap)


@pytest.mark.parametrize("new", [1, 60])
def test_shared_pages(gpu, new):
    """Three sequences with the same first pages, one after the other and one behind what the table holds."""
    kv, hd, heads, lens = 2, 128, 8, [190, 150, 129]
    table = np.asarray([[5, 3, 1], [5, 3, 0], [5, 3, 2]], np.int64)
    h = Held(gpu, kv, hd, lens, 63, pages=6, table=table, max_pages=3)
    first = _offsets([new] * 3)
    h.check_attend(F16, _rows(64, F16, first[-1], heads * hd), first, heads, "shared pages, %d new" % new)


def test_lengths_lowered(gpu):
    """Tokens taken back and others put in their place: the page keeps at least its scale, the tokens before them theirs."""
    kv, hd, lens = 2, 64, [70]
    h = Held(gpu, kv, hd, lens, 65)
    h.append(F32, _rows(66, F32, 6, kv * hd, 50.0), _rows(67, F32, 6, kv * hd, 9.0), [0, 6])
    h.same()
    for length, new in ((67, 2), (66, 1), (65, 1), (65, 65)):   # (65, 65: all of it from the start)
        h.lens = [length]
        h.len = gpu.DeviceBuffer.from_array(np.asarray(h.lens, np.int32))
        h.kv = gpu.kv_cache(kv, hd, h.model.pages, h.model.table.shape[1], h.pool, h.table, h.len)
        h.append(F32, _rows(68, F32, new, kv * hd, 0.1), _rows(69, F32, new, kv * hd, 100.0), [0, new])
        h.same()


def test_many_sequences(gpu):
    kv, hd, heads, n = 2, 64, 4, 200
    lens = [int(x) for x in np.random.default_rng(3).integers(1, 130, n)]
    h = Held(gpu, kv, hd, lens, 43)
    h.check_attend(BF16, _rows(44, BF16, n, heads * hd), list(range(n + 1)), heads, "200 sequences")


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_queries_of_any_size(gpu, t):
    """Rows of q from tiny to large (a scale of their own each), one row not finite: only it is lost."""
    kv, hd, heads, lens = 1, 128, 4, [200, 70]
    h = Held(gpu, kv, hd, lens, 50)
    h.model.scale[:] = 2.0 ** -5
    h.pool.upload(h.model.pool())
    size = {F32: (1e-30, 1e-4, 1.0, 30.0), F16: (1e-6, 1e-3, 1.0, 30.0), BF16: (1e-30, 1e-4, 1.0, 30.0)}[t]
    x = np.random.default_rng(51).standard_normal((2, heads, hd)) * np.asarray(size)[None, :, None] * 0.1
    q = R.to_type(x.reshape(2, heads * hd), t)
    clean = h.check_attend(t, q, [0, 1, 2], heads, "sizes")
    for bad in (np.nan, np.inf):
        q2 = q.copy()
        q2[0, 2 * hd + 5] = R.to_type(np.full(1, bad), t)[0]
        got = h.attend(t, q2, [0, 1, 2], heads)
        lost = R.from_type(got[0, 2 * hd:3 * hd], t)
        assert not np.isfinite(lost).any()
        got[0, 2 * hd:3 * hd] = clean[0, 2 * hd:3 * hd]
        assert np.array_equal(got, clean)


def test_scales_far_apart(gpu):
    """Pages whose scales differ by many powers of two, K and V alike."""
    kv, hd, heads, lens = 1, 64, 2, [640]
    h = Held(gpu, kv, hd, lens, 52)
    h.model.scale[:, :, 0] = 2.0 ** np.random.default_rng(1).integers(-12, -4, (h.model.pages, 1))
    h.model.scale[:, :, 1] = 2.0 ** np.random.default_rng(2).integers(-60, 60, (h.model.pages, 1))
    h.pool.upload(h.model.pool())
    for t in (F32, BF16):
        h.check_attend(t, _rows(53, t, 1, heads * hd), [0, 1], heads, "scales")
        h.check_attend(t, _rows(53, t, 40, heads * hd), [0, 40], heads, "scales")


def test_offsets_past_32_bits(gpu):
    """Pages beyond the 4 GiB mark of the pool."""
    F, kv, hd, heads, t = gpu, 8, 128, 16, BF16
    per = F.kv_pool_bytes(kv, hd, 1)
    pages = (1 << 32) // per + 40
    lens = [130, 70]
    near = Held(F, kv, hd, lens, 60, pages=7)
    first = [0, 130, 200]
    k, v, q = _rows(61, t, 200, kv * hd), _rows(62, t, 200, kv * hd), _rows(63, t, 200, heads * hd)
    near.append(t, k, v, first)
    want, want1 = near.attend(t, q, first, heads), near.attend(t, q[[129, 199]], [0, 1, 2], heads)
    read = near.read(t, first)
    pool = F.DeviceBuffer(F.kv_pool_bytes(kv, hd, pages))
    table = F.DeviceBuffer.from_array(np.asarray([[pages - 1, 5, pages - 2], [pages - 30, pages - 3, -1]], np.int32))
    far = near
    far.pool, far.table = pool, table
    far.kv = F.kv_cache(kv, hd, pages, 3, pool, table, far.len)
    dk, dv, df = (F.DeviceBuffer.from_array(x) for x in (k, v, np.asarray(first, np.int32)))
    F.kv_append_dev(far.kv, t, dk, dv, 200, 2, df)
    for got, w in zip(far.read(t, first), read):
        assert np.array_equal(got, w)
    assert np.array_equal(far.attend(t, q, first, heads), want)
    assert np.array_equal(far.attend(t, q[[129, 199]], [0, 1, 2], heads), want1)
    pool.close()


def test_extend(gpu):
    F = gpu
    h = Held(F, 1, 64, [0, 5, -3, 2 ** 31 - 2, 9], 70, pages=4, max_pages=2, table=np.zeros((5, 2), int))
    df = F.DeviceBuffer.from_array(np.asarray([0, 2, 3, 7, 10, 10], np.int32))
    F.kv_extend_dev(h.kv, 10, 5, df)
    F.synchronize()
    assert list(h.len.download(np.int32, (5,))) == [2, 6, 4, 2 ** 31 - 1, 9]
    F.kv_extend_dev(h.kv, 5, 5)
    F.synchronize()
    assert list(h.len.download(np.int32, (5,))) == [3, 7, 5, 2 ** 31 - 1, 10]


def test_prompt_then_tokens_as_they_are_used(gpu):
    """A layer's whole use: two prompts attended to at full precision and written to the cache, then steps of
    one token each in a captured graph (lengths moved on, rows appended, attention), a chunk at the end; every
    output against 64 bits from the cache's own values."""
    F, t, heads, kv, hd = gpu, BF16, 16, 2, 128
    prompt, steps, chunk = [70, 33], 40, 50
    total = [p + steps + chunk for p in prompt]
    h = Held(F, kv, hd, total, 80)
    h.lens = [0, 0]
    h.len.upload(np.asarray(h.lens, np.int32))
    cfg = F.attn_cfg(heads, kv, hd, t)

    def rows(seed, n):
        return _rows(seed, t, n, heads * hd), _rows(seed + 1, t, n, kv * hd), _rows(seed + 2, t, n, kv * hd)

    first = _offsets(prompt)
    q, k, v = rows(81, first[-1])
    dq, dk, dv, df = (F.DeviceBuffer.from_array(x) for x in (q, k, v, np.asarray(first, np.int32)))
    do = F.DeviceBuffer(q.nbytes)
    F.kv_extend_dev(h.kv, first[-1], 2, df)
    F.kv_append_dev(h.kv, t, dk, dv, first[-1], 2, df)
    F.attention_seqs_dev(cfg, dq, dk, dv, do, first[-1], 2, df)
    F.synchronize()
    o, a, big = R.attention(*(R.from_type(x, t) for x in (q, k, v)), first, heads, kv, hd)
    R.check(do.download(q.dtype, q.shape), t, o, a, big, hd, 70, "prompt")
    h.lens = list(prompt)
    h.model.append((R.from_type(k, t), R.from_type(v, t)), first, h.lens)
    h.same()

    bufs = [F.DeviceBuffer.from_array(x) for x in rows(90, 2)]
    out = F.DeviceBuffer(2 * heads * hd * 2)
    need = F.kv_attention_workspace_bytes(cfg, h.kv, 2, 2)
    ws = F.DeviceBuffer(max(1, need))

    def step():
        F.kv_extend_dev(h.kv, 2, 2)
        F.kv_append_dev(h.kv, t, bufs[1], bufs[2], 2, 2)
        F.kv_attention_dev(cfg, h.kv, bufs[0], out, 2, 2, ws, need)

    g = F.capture(step)
    try:
        for i in range(steps):
            q, k, v = rows(100 + 3 * i, 2)
            for b, x in zip(bufs, (q, k, v)):
                b.upload(x)
            g.launch()
            F.synchronize()
            h.lens = [n + 1 for n in h.lens]
            h.model.append((R.from_type(k, t), R.from_type(v, t)), [0, 1, 2], h.lens)
            o, a, big = h.model.attention(R.from_type(q, t), [0, 1, 2], h.lens, heads)
            R.check(out.download(q.dtype, q.shape), t, o, a, big, hd, max(h.lens), "step %d" % i)
    finally:
        g.close()
    h.same()
    assert list(h.len.download(np.int32, (2,))) == h.lens

    first = [0, chunk, 2 * chunk]
    q, k, v = rows(400, 2 * chunk)
    df = F.DeviceBuffer.from_array(np.asarray(first, np.int32))
    F.kv_extend_dev(h.kv, 2 * chunk, 2, df)
    h.lens = [n + chunk for n in h.lens]
    h.append(t, k, v, first)
    h.same()
    h.check_attend(t, q, first, heads, "chunk")


def test_two_graphs_two_streams(gpu):
    """Two captured steps with a workspace each, replayed on two streams at once, several times."""
    F, t, heads, kv, hd = gpu, F32, 16, 2, 128
    sides = []
    for i, lens in enumerate(([1500, 900, 40], [2000, 3, 700])):
        h = Held(F, kv, hd, lens, 90 + i)
        q = _rows(95 + i, t, 3, heads * hd)
        want = h.attend(t, q, [0, 1, 2, 3], heads)
        cfg = F.attn_cfg(heads, kv, hd, t)
        need = F.kv_attention_workspace_bytes(cfg, h.kv, 3, 3)
        ws, dq, do = F.DeviceBuffer(max(1, need)), F.DeviceBuffer.from_array(q), F.DeviceBuffer(q.nbytes)
        g = F.capture(lambda: F.kv_attention_dev(cfg, h.kv, dq, do, 3, 3, ws, need))
        st = ctypes.c_void_p()
        assert F.lib().hipStreamCreateWithFlags(ctypes.byref(st), ctypes.c_uint(1)) == 0
        sides.append((h, g, do, want, st, (ws, dq)))
    for r in range(4):
        for h, g, do, want, st, _ in sides:
            do.fill(0)
        F.synchronize()
        for h, g, do, want, st, _ in sides:
            g.launch(st.value)
        F.synchronize()
        for h, g, do, want, st, _ in sides:
            assert np.array_equal(do.download(want.dtype, want.shape), want), r
    for side in sides:
        side[1].close()
        assert F.lib().hipStreamDestroy(side[4]) == 0
