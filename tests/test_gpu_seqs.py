"""fh3_hip_attention_seqs_dev on the GPU against a 64-bit plain form: value
types, shared key heads, ragged and empty sequences, prefixes, capped scores,
distance bias, strides, values that are not finite, replays and streams."""
import ctypes

import numpy as np
import pytest

import seqs_ref as R
from seqs_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu


def _buf(F, a):
    return F.DeviceBuffer.from_array(a)


def _case(seed, t, n, heads, kv, hd, qs=1.5):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((n, heads * hd)) * qs
    k = rng.standard_normal((n, kv * hd))
    k[:, ::32] *= 3
    v = rng.standard_normal((n, kv * hd))
    return [R.to_type(x, t) for x in (q, k, v)]


def _run(F, arrays, t, first, heads, kv, hd, prefix=None, slopes=None, rows=None, **cfg):
    q, k, v = arrays
    rows = q.shape[0] if rows is None else rows
    dq, dk, dv = (_buf(F, x) for x in (q, k, v))
    o = np.full_like(q, 7)
    do = _buf(F, o)
    df = _buf(F, np.asarray(first, np.int32))
    dp = None if prefix is None else _buf(F, np.asarray(prefix, np.int32))
    ds = None if slopes is None else _buf(F, np.asarray(slopes, np.float32))
    c = F.attn_cfg(heads, kv, hd, t, d_slopes=ds, **cfg)
    F.attention_seqs_dev(c, dq, dk, dv, do, rows, len(first) - 1, df, dp)
    F.synchronize()
    return do.download(o.dtype, o.shape)


def _offsets(lens):
    return [0] + list(np.cumsum(lens))


CASES = [
    # heads, kv, hd, lens, causal, cap, alibi, prefix
    (1, 1, 64, [1], True, 0.0, False, None),
    (8, 8, 128, [1, 2, 3], True, 0.0, False, None),
    (16, 2, 128, [63, 64, 65], True, 0.0, False, None),
    (8, 1, 64, [0, 5, 0, 0, 129, 0], True, 0.0, False, None),
    (10, 2, 128, [31, 300], True, 50.0, False, None),
    (14, 2, 64, [127, 33], False, 0.0, False, None),
    (6, 2, 128, [200, 77], True, 0.0, True, None),
    (4, 4, 64, [191, 1, 90], True, 20.0, True, [50, 1, 90]),
    (40, 8, 128, [257, 130], True, 0.0, False, [0, 400]),
    (3, 1, 128, [600], True, 0.0, False, [65]),
    (16, 16, 64, [1024, 17], True, 0.0, False, None),
    (56, 1, 128, [70], True, 30.0, True, [11]),
    (8, 2, 64, [333, 90], False, 15.0, True, None),
    (128, 1, 64, [9, 40], True, 0.0, False, None),
]


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_against_64_bits(gpu, t, i):
    heads, kv, hd, lens, causal, cap, alibi, prefix = CASES[i]
    first = _offsets(lens)
    print("case %d type %s lens %s" % (i, R.NAMES[t], lens), flush=True)
    arrays = _case(100 + i, t, first[-1], heads, kv, hd)
    slopes = np.asarray([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], np.float32) if alibi else None
    got = _run(gpu, arrays, t, first, heads, kv, hd, prefix, slopes, causal=causal, softcap=cap)
    o, a, big = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd, causal, None, cap, slopes, prefix)
    R.check(got, t, o, a, big, hd, max(lens), "case %d" % i)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_and_peaked(gpu, t, hd):
    """2300 tokens with scores of up to about a hundred: rows that one key wins, and offsets raised often."""
    heads, kv, n = 2, 1, 2300
    arrays = _case(31, t, n, heads, kv, hd, qs=9.0)
    got = _run(gpu, arrays, t, [0, n], heads, kv, hd)
    o, a, big = R.attention(*(R.from_type(x, t) for x in arrays), [0, n], heads, kv, hd)
    assert big > 50
    R.check(got, t, o, a, big, hd, n, "peaked")


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,hd", [(16, 16, 64), (16, 8, 128)])
def test_many_sequences(gpu, t, heads, kv, hd):
    """More than 64 sequences, some empty, one long: more workgroups than the card holds at once."""
    lens = [int(x) for x in np.random.default_rng(17).integers(0, 40, 150)]
    lens[97] = 500
    first = _offsets(lens)
    arrays = _case(18, t, first[-1], heads, kv, hd)
    got = _run(gpu, arrays, t, first, heads, kv, hd)
    o, a, big = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd)
    R.check(got, t, o, a, big, hd, 500, "many")


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_rows_behind_the_last_sequence(gpu, t):
    heads, kv, hd = 4, 2, 64
    arrays = _case(5, t, 90, heads, kv, hd)
    for x in arrays:  # nothing there is read either
        x[70:] = R.to_type(np.full(1, np.nan), t)
    got = _run(gpu, arrays, t, [0, 33, 70], heads, kv, hd)
    assert (got[70:] == 7).all()
    o, a, big = R.attention(*(R.from_type(x[:70], t) for x in arrays), [0, 33, 70], heads, kv, hd)
    R.check(got[:70], t, o, a, big, hd, 40, "tail")


def test_offsets_outside_the_rows_are_cut(gpu):
    """d_first may name rows that are not there: they are cut to the n_tok given, a falling pair is an empty sequence."""
    heads, kv, hd = 4, 2, 64
    arrays = _case(6, BF16, 50, heads, kv, hd)
    want = _run(gpu, arrays, BF16, [0, 10, 50], heads, kv, hd)
    got = _run(gpu, arrays, BF16, [-9, 10, 1000], heads, kv, hd)
    assert np.array_equal(got, want)
    got = _run(gpu, arrays, BF16, [0, 50, 10], heads, kv, hd)
    assert np.array_equal(got, _run(gpu, arrays, BF16, [0, 50], heads, kv, hd))
    wild = [-10 ** 9, 50]
    assert np.array_equal(_run(gpu, arrays, BF16, [0, 50], heads, kv, hd, prefix=[-7]), _run(gpu, arrays, BF16, wild, heads, kv, hd))
    assert np.array_equal(_run(gpu, arrays, BF16, [0, 50], heads, kv, hd, prefix=[2 ** 31 - 1]),
                          _run(gpu, arrays, BF16, [0, 50], heads, kv, hd, causal=False))


def test_equal_sequences_without_offsets(gpu):
    F, t, heads, kv, hd = gpu, F16, 8, 2, 128
    arrays = _case(8, t, 4 * 37, heads, kv, hd)
    want = _run(F, arrays, t, [0, 37, 74, 111, 148], heads, kv, hd)
    dq, dk, dv = (_buf(F, x) for x in arrays)
    do = F.DeviceBuffer(arrays[0].nbytes)
    F.attention_seqs_dev(F.attn_cfg(heads, kv, hd, t), dq, dk, dv, do, 148, 4)
    F.synchronize()
    assert np.array_equal(do.download(np.float16, want.shape), want)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_parts_of_one_buffer(gpu, t):
    """q, k, v inside one projection's output, o rows with a gap that stays as it is."""
    F, heads, kv, hd, lens = gpu, 6, 2, 128, [100, 31]
    first = _offsets(lens)
    q, k, v = _case(9, t, first[-1], heads, kv, hd)
    want = _run(F, (q, k, v), t, first, heads, kv, hd)
    qkv = np.concatenate([q, k, v], 1)
    buf, size, ld = _buf(F, qkv), qkv.itemsize, qkv.shape[1]
    wide = np.full((first[-1], heads * hd + 16), 3, q.dtype)
    do, df = _buf(F, wide), _buf(F, np.asarray(first, np.int32))
    F.attention_seqs_dev(F.attn_cfg(heads, kv, hd, t), buf, buf.ptr + heads * hd * size, buf.ptr + (heads + kv) * hd * size,
                         do, first[-1], 2, df, ldq=ld, ldk=ld, ldv=ld, ldo=wide.shape[1])
    F.synchronize()
    got = do.download(wide.dtype, wide.shape)
    assert np.array_equal(got[:, :heads * hd], want)
    assert (got[:, heads * hd:] == 3).all()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_not_finite_reaches_only_rows_that_see_it(gpu, t, where, bad):
    """A key or value that is not finite, in the middle of a tile: rows before it and the other sequence keep
    their bits; rows that see it are not finite (V: in its channel, and only there)."""
    heads, kv, hd, first, at, ch = 4, 2, 64, [0, 150, 230], 101, 37
    arrays = _case(12, t, 230, heads, kv, hd)
    clean = R.from_type(_run(gpu, arrays, t, first, heads, kv, hd), t)
    arrays[1 if where == "k" else 2][at, hd + ch] = R.to_type(np.full(1, bad), t)[0]
    got = R.from_type(_run(gpu, arrays, t, first, heads, kv, hd), t).reshape(230, heads, hd)
    clean = clean.reshape(230, heads, hd)
    rest = [r for r in range(230) if not at <= r < 150]
    assert np.array_equal(got[rest], clean[rest])
    assert np.array_equal(got[at:150, :2], clean[at:150, :2])   # the other key head's rows
    hit = got[at:150, 2:]
    if where == "v":
        assert not np.isfinite(hit[..., ch]).any()
        others = np.delete(np.arange(hd), ch)
        assert np.array_equal(hit[..., others], clean[at:150, 2:][..., others])
    elif np.isnan(bad):
        assert np.isnan(hit).all()
    else:  # an infinite score: rows whose product is +inf are NaN, -inf leaves the key out
        assert (np.isnan(hit).all(-1) | np.isfinite(hit).all(-1)).all()


def test_closed_forms(gpu):
    """Equal keys: the mean of what is seen; one key seen: its value."""
    heads, kv, hd, n = 2, 1, 64, 130
    rng = np.random.default_rng(1)
    q, v = rng.standard_normal((n, heads * hd)).astype(np.float32), rng.standard_normal((n, hd)).astype(np.float32)
    k = np.repeat(rng.standard_normal((1, hd)), n, 0).astype(np.float32)
    got = _run(gpu, (q, k, v), F32, [0, n], heads, kv, hd).reshape(n, heads, hd)
    mean = np.cumsum(v.astype(np.float64), 0) / np.arange(1, n + 1)[:, None]
    assert np.abs(got - mean[:, None]).max() < 4 * 2.0 ** -16 * np.abs(v).max()
    assert np.abs(got[0] - v[0]).max() <= 2.0 ** -16 * np.abs(v).max()


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [0.5, 64.0, 65.0, 1e4, 1e8, 1e30])
def test_caps_of_any_size(gpu, t, cap):
    """A cap far above the scores leaves them as they are, one far below makes them +-cap."""
    heads, kv, hd, lens = 4, 2, 64, [130, 20]
    first = _offsets(lens)
    arrays = _case(23, t, first[-1], heads, kv, hd)
    got = _run(gpu, arrays, t, first, heads, kv, hd, softcap=cap)
    o, a, big = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd, True, None, cap)
    R.check(got, t, o, a, big, hd, max(lens), "cap %g" % cap)


def test_values_far_from_one(gpu):
    """fp32 operands of any size: keys and values near the ends of fp32 and of fp16's range."""
    heads, kv, hd, n = 2, 1, 128, 90
    rng = np.random.default_rng(2)
    for qs, ks, vs in ((1e-20, 1e20, 1e30), (1e15, 1e-15, 1e-25), (3e5, 1e-6, 7e4)):
        arrays = [(rng.standard_normal((n, w * hd)) * s).astype(np.float32) for w, s in ((heads, qs), (kv, ks), (kv, vs))]
        got = _run(gpu, arrays, F32, [0, n], heads, kv, hd)
        o, a, big = R.attention(*(x.astype(np.float64) for x in arrays), [0, n], heads, kv, hd)
        R.check(got, F32, o, a, big, hd, n, "q %g k %g v %g" % (qs, ks, vs))


@pytest.mark.parametrize("hd,lens", [(128, [230]), (64, [230]), (128, [40, 230] + [20] * 130)])
@pytest.mark.parametrize("sizes", [(1.0, 1e-9), (1e-9, 1.0), (1.0, 1e5), (1e5, 1.0), (0.0, 1e-12), (1e-12, 0.0), (1e-20, 1e20),
                                   (30.0, 500.0, 1e-3), (1.0, 1e30, 1e-30), (1e-30, 1e30, 1.0)])
def test_rows_of_v_of_different_sizes(gpu, hd, lens, sizes):
    """fp32 V whose rows change size from run to run of keys, zeros among them, with rows that see one size only.

    V and the weights enter as two fp16 terms, whose least step is 2^-24.  A row of V is off by 2^-25 in units in
    which its largest is 2^3 at least (2^4 at 2^-5 times 512), so by 2^-28 of its largest.  A weight is off by 2^-25
    beside a largest of 2^6 at least, in units of the largest factor seen: times a row whose largest is 2^15 at most
    where that of the factor's is 2^14 at least (large rows) or 2^4 where it is 2^3 (small ones and those left alone: 2^4),
    so by 2^-30 of the largest row for every key."""
    heads, kv = 16, 8
    first = _offsets(lens)
    q, k, v = _case(19, F32, first[-1], heads, kv, hd)
    for s, n in enumerate(lens):
        for j in range(n):
            v[first[s] + j] *= sizes[min(j // 50, len(sizes) - 1)] if n > 50 else sizes[s % len(sizes)]
    got = _run(gpu, (q, k, v), F32, first, heads, kv, hd)
    o, a, big = R.attention(*(x.astype(np.float64) for x in (q, k, v)), first, heads, kv, hd)
    floor = np.zeros_like(o)
    top = np.repeat(np.abs(v.reshape(-1, kv, hd)).max(2).astype(np.float64), heads // kv, 1)
    for s, n in enumerate(lens):
        for j in range(n):
            m = top[first[s]:first[s] + j + 1].max(0)
            floor[first[s] + j] = np.repeat(m * (2.0 ** -28 + (j + 1) * 2.0 ** -30), hd)
    R.check(got, F32, o, a, big, hd, max(lens), "sizes %s" % (sizes,), floor)


def test_replays_and_streams(gpu):
    """Captured and replayed, with other eager work between, and on a stream of its own: the eager bits."""
    F, t, heads, kv, hd = gpu, BF16, 16, 2, 128
    first = _offsets([200, 3, 61])
    arrays = _case(14, t, first[-1], heads, kv, hd)
    want = _run(F, arrays, t, first, heads, kv, hd)
    dq, dk, dv = (_buf(F, x) for x in arrays)
    do, df = F.DeviceBuffer(arrays[0].nbytes), _buf(F, np.asarray(first, np.int32))
    cfg = F.attn_cfg(heads, kv, hd, t)
    g = F.capture(lambda: F.attention_seqs_dev(cfg, dq, dk, dv, do, first[-1], 3, df))
    try:
        for r in range(3):
            do.fill(0)
            F.synchronize()
            g.launch()
            F.synchronize()
            assert np.array_equal(do.download(want.dtype, want.shape), want), r
            _run(F, arrays, t, [0, first[-1]], heads, kv, hd)
        df.upload(np.asarray([0, 100, 100, 264], np.int32))   # read anew at each replay
        g.launch()
        F.synchronize()
        assert np.array_equal(do.download(want.dtype, want.shape), _run(F, arrays, t, [0, 100, 100, 264], heads, kv, hd))
    finally:
        g.close()
    df.upload(np.asarray(first, np.int32))
    st = ctypes.c_void_p()
    assert F.lib().hipStreamCreateWithFlags(ctypes.byref(st), ctypes.c_uint(1)) == 0
    do.fill(0)
    F.synchronize()
    F.attention_seqs_dev(cfg, dq, dk, dv, do, first[-1], 3, df, stream_ptr=st.value)
    F.synchronize()
    assert F.lib().hipStreamDestroy(st) == 0
    assert np.array_equal(do.download(want.dtype, want.shape), want)
