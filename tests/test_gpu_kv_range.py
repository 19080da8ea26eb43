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
