"""Attention over the 8-bit cache at the ends of the ranges, and its less used
paths: scores and cached values of any size, pages of zeros, runs of hundreds of
pages, many long sequences, a chunk beside single tokens."""
import numpy as np
import pytest

import seqs_ref as R
from seqs_ref import BF16, F16, F32
from test_gpu_kv import Held, _offsets, _rows
from test_gpu_seqs_range import _near

pytestmark = pytest.mark.gpu

# rows to a sequence below with two heads to a key head: 2, 6, 20, 80
NEW = [1, 3, 10, 40]


def _put(h):
    """The model's pages to the device."""
    h.pool.upload(h.model.pool())


def _against(h, t, q, first, heads, what, **kw):
    got = h.attend(t, q, first, heads, **kw)
    o, _, _ = h.model.attention(R.from_type(q, t), first, h.lens, heads, kw.get("causal", True), kw.get("scale"),
                                kw.get("softcap", 0.0), kw.get("slopes"))
    _near(got, o, t, what)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** e for e in (-14, -7, -5, -4, -3, 0, 20, 40, 69, 90)])
def test_scores_of_any_size(gpu, t, hd, scale):
    """Products of +-2^30 + 128 n, exact; the longer sequence's tiles are divided."""
    heads, kv, lens = 4, 2, [3000, 70]
    h = Held(gpu, kv, hd, lens, 31)
    h.model.scale[:, :, 0] = 2.0 ** 9
    k = h.model.q[:, :, 0]
    k[:] = 0
    k[..., 0] = 64
    k[..., hd - 1] = np.random.default_rng(32).integers(0, 21, k.shape[:-1])
    _put(h)
    for new in NEW:
        first = _offsets([new, new])
        q = np.zeros((2 * new, heads, hd))
        q[:, :, 0] = np.where(np.arange(heads) % 2, -2.0 ** 15, 2.0 ** 15)
        q[:, :, hd - 1] = 0.25
        _against(h, t, R.to_type(q.reshape(2 * new, -1), t), first, heads, "scale %g, %d new" % (scale, new), scale=scale)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("kind", ["large", "mixed", "small"])
def test_values_near_the_ends(gpu, t, kind):
    """V of up to 127 2^121, of 2^-100 at the least, and pages of either kind beside each other."""
    heads, kv, hd, lens = 4, 2, 64, [3000, 70]
    h = Held(gpu, kv, hd, lens, 33)
    rng = np.random.default_rng(34)
    e = {"large": np.full((h.model.pages, kv), 121), "small": np.full((h.model.pages, kv), -100),
         "mixed": rng.choice([121, 119, 0, -100], (h.model.pages, kv))}[kind]
    h.model.scale[:, :, 0] = 2.0 ** -6
    h.model.scale[:, :, 1] = 2.0 ** e
    h.model.q[:, :, 1] = rng.integers(40, 128, h.model.q[:, :, 1].shape)
    _put(h)
    for new in NEW:
        first = _offsets([new, new])
        _against(h, t, _rows(35, t, 2 * new, heads * hd, 0.5), first, heads, "%s, %d new" % (kind, new))


@pytest.mark.parametrize("new", NEW)
def test_pages_of_zeros_and_small_queries(gpu, new):
    """Pages whose K is 0 have the least scale, 2^-100; times that of a small q it is below fp32's least number.  All
    scores are 0: the mean of what is seen."""
    heads, kv, hd, lens = 4, 2, 128, [200, 70]
    h = Held(gpu, kv, hd, lens, 36)
    h.model.q[:, :, 0] = 0
    h.model.scale[:, :, 0] = 2.0 ** -100
    _put(h)
    for size in (1.0, 1e-8, 1e-13, 1e-25):
        first = _offsets([new, new])
        _against(h, F32, _rows(37, F32, 2 * new, heads * hd, size), first, heads, "q %g, %d new" % (size, new))


@pytest.mark.parametrize("t", [F16, BF16])
def test_equal_values_come_back_exactly(gpu, t):
    """V the same in every token, whole numbers of seven bits: the weights as they enter the product are what is summed,
    so the output is V.  The last token's key is the only one that is not 0, by 0 to 10 in scores above the others
    that came before it, so that a weight which is no power of two decides the sum."""
    heads, kv, hd = 64, 2, 64
    lens = [300, 261, 40, 3, 2]
    h = Held(gpu, kv, hd, lens, 38)
    h.model.scale[:, :, 1] = 2.0 ** -4
    h.model.q[:, :, 1] = np.random.default_rng(39).integers(96, 128, (1, kv, 1, hd))
    h.model.q[:, :, 0] = 0
    h.model.scale[:, :, 0] = 2.0 ** -6
    for s, n in enumerate(lens):
        h.model.q[h.model.page(s, (n - 1) // R.PAGE), :, 0, (n - 1) % R.PAGE, 0] = 64
    _put(h)
    want = np.repeat(h.model.q[0, :, 1, 0] / 16, heads // kv, 0).ravel()
    for new in (1, 2):
        first = _offsets([new] * len(lens))
        q = np.zeros((first[-1], heads, hd))
        q[:, :, 0] = np.random.default_rng(40).uniform(0, 80, q.shape[:2])
        got = R.from_type(h.attend(t, R.to_type(q.reshape(first[-1], -1), t), first, heads), t)
        assert np.array_equal(got, np.broadcast_to(want, got.shape)), new


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("new", [1, 40])
def test_runs_of_hundreds_of_pages(gpu, t, new):
    """256 key heads: two workgroups to a head, runs of 310 pages each, so that page numbers and scales are fetched
    64 at a time more than once.  The table repeats seven pages in no order."""
    F, kv, hd, pages, n_pages = gpu, 256, 64, 7, 620
    rng = np.random.default_rng(41)
    table = rng.integers(0, pages, (1, n_pages))
    length = n_pages * R.PAGE - 5
    h = Held(F, kv, hd, [length], 42, pages=pages, table=table, max_pages=n_pages)
    first = [0, new]
    q = _rows(43, t, new, kv * hd, 0.5)
    got = R.from_type(h.attend(t, q, first, kv), t).reshape(new, kv, hd)
    m, qv = h.model, R.from_type(q, t).reshape(new, kv, hd)
    pos = length - new + np.arange(new)
    see = np.arange(length)[None, :] <= pos[:, None]
    for head in (0, 1, 100, 255):
        k, v = ((m.q[table[0], head, w] * m.scale[table[0], head, w][:, None, None]).reshape(-1, hd)[:length] for w in (0, 1))
        o, _, _ = R.head_outputs(qv[:, head], k, v, pos, 1 / np.sqrt(hd), 0.0, None, see)
        _near(R.to_type(got[:, head], t), o, t, "head %d, %d new" % (head, new))


@pytest.mark.parametrize("t", [F32, BF16])
def test_many_long_sequences(gpu, t):
    """100 sequences of 1 to 1500 tokens, one new token each: divided tiles behind the first 64 sequences."""
    kv, hd, heads, n = 2, 64, 4, 100
    lens = [int(x) for x in np.random.default_rng(44).integers(1, 1500, n)]
    lens[70], lens[99] = 1500, 1400
    h = Held(gpu, kv, hd, lens, 45)
    _against(h, t, _rows(46, t, n, heads * hd), list(range(n + 1)), heads, "100 sequences")


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("singles", [30, 150])
def test_a_chunk_beside_single_tokens(gpu, t, singles):
    """One sequence's chunk in a call with single tokens of others: 128-row tiles for all, or 32-row ones."""
    kv, hd, heads = 2, 64, 16
    rng = np.random.default_rng(47)
    new = [1] * (singles // 2) + [300] + [1] * (singles - singles // 2)
    lens = [int(x) for x in rng.integers(1, 700, len(new))]
    lens[singles // 2] = 900
    h = Held(gpu, kv, hd, lens, 48)
    first = _offsets(new)
    _against(h, t, _rows(49, t, first[-1], heads * hd), first, heads, "chunk and %d tokens" % singles)


def test_read_back_between_each_other(gpu):
    """K and V read to the two halves of one buffer's rows."""
    F, kv, hd, lens = gpu, 2, 64, [70, 3]
    h = Held(F, kv, hd, lens, 50)
    first = _offsets(lens)
    want = h.model.read(first, lens)
    w = kv * hd
    out, df = F.DeviceBuffer(first[-1] * 2 * w * 4), F.DeviceBuffer.from_array(np.asarray(first, np.int32))
    F.kv_read_dev(h.kv, F32, out.ptr, out.ptr + w * 4, first[-1], 2, df, ldk=2 * w, ldv=2 * w)
    F.synchronize()
    got = out.download(np.float32, (first[-1], 2, w))
    assert np.array_equal(got[:, 0], want[0]) and np.array_equal(got[:, 1], want[1])
