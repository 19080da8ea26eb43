"""fp32 attention over sequences and over the cache, held to what two fp16 terms of
each operand give.

An operand is hi + lo, each rounded to 11 bits: off by 2^-23 of itself at most and
2^-24 r.m.s., as long as lo is above fp16's least step, which the powers of two see to
(2^-29 of a row's largest and below).  Scores that spread by sigma are sums of
products that spread as much, so the operands' terms, the fp32 sums and log2(e) put
them off by less than 2^-22 sigma; a score's error moves an output by as much of
itself, r.m.s.  Weights (exp2, two terms), their sum and V's terms give 2^-23 to
2^-22 each, independent of sigma: 2^-21 together.  A cap's tanh and a distance bias
put scores off by a few last bits more, 2^-22 and 2^-20.  One term of 16 bits in
place of two, or bf16 terms (8 bits each, 2^-17), are far outside."""
import numpy as np
import pytest

import seqs_ref as R
from seqs_ref import F32
from test_gpu_kv import Held
from test_gpu_seqs import _offsets, _run
from test_gpu_seqs_range import _near

pytestmark = pytest.mark.gpu


def _tol(sigma, cap=0.0, bias=False):
    return 2.0 ** -22 * (2 + sigma) + (2.0 ** -22 if cap else 0) + (2.0 ** -20 if bias else 0)


def _arrays(seed, n, heads, kv, hd, sigma, k_rms, v_rms=1.0):
    rng = np.random.default_rng(seed)
    return [(rng.standard_normal((n, w * hd)) * s).astype(np.float32)
            for w, s in ((heads, sigma / k_rms), (kv, k_rms), (kv, v_rms))]


@pytest.mark.parametrize("sigma", [1.5, 6.0])
@pytest.mark.parametrize("k_rms", [1e-3, 0.013, 0.05, 1.0, 20.0, 60.0, 180.0, 5e3, 1e5])
@pytest.mark.parametrize("hd", [64, 128])
def test_keys_of_any_size(gpu, hd, k_rms, sigma):
    """Rows of K just above, at and below the sizes at which their power of two changes."""
    heads, kv, lens = 4, 2, [600, 40]
    first = _offsets(lens)
    arrays = _arrays(71, first[-1], heads, kv, hd, sigma, k_rms)
    got = _run(gpu, arrays, F32, first, heads, kv, hd)
    o, _, _ = R.attention(*(x.astype(np.float64) for x in arrays), first, heads, kv, hd)
    _near(got, o, F32, "k %g sigma %g" % (k_rms, sigma), _tol(sigma))


@pytest.mark.parametrize("v_rms", [1e-3, 0.013, 1.0, 30.0, 1e4])
def test_values_of_any_size(gpu, v_rms):
    heads, kv, hd, n = 4, 2, 128, 500
    arrays = _arrays(72, n, heads, kv, hd, 1.5, 1.0, v_rms)
    got = _run(gpu, arrays, F32, [0, n], heads, kv, hd)
    o, _, _ = R.attention(*(x.astype(np.float64) for x in arrays), [0, n], heads, kv, hd)
    _near(got, o, F32, "v %g" % v_rms, _tol(1.5))


@pytest.mark.parametrize("heads,kv,hd,lens,causal,cap,bias,prefix", [
    (64, 8, 128, [600], True, 0.0, False, None),
    (64, 8, 128, [37], True, 0.0, False, None),
    (16, 16, 64, [900, 17, 300], True, 0.0, False, [100, 17, 0]),
    (10, 2, 128, [300, 31], False, 0.0, False, None),
    (8, 4, 128, [400, 90], True, 30.0, False, None),
    (8, 4, 64, [400, 90], True, 0.0, True, None),
])
def test_sequences(gpu, heads, kv, hd, lens, causal, cap, bias, prefix):
    first = _offsets(lens)
    arrays = _arrays(73, first[-1], heads, kv, hd, 1.5, 1.0)
    slopes = np.asarray([2.0 ** (-8 * (h + 1) / heads) for h in range(heads)], np.float32) if bias else None
    got = _run(gpu, arrays, F32, first, heads, kv, hd, prefix, slopes, causal=causal, softcap=cap)
    o, _, _ = R.attention(*(x.astype(np.float64) for x in arrays), first, heads, kv, hd, causal, None, cap, slopes, prefix)
    _near(got, o, F32, "lens %s" % lens, _tol(1.5, cap, bias))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 10, 40])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (30.0, False), (0.0, True)])
def test_cache(gpu, hd, new, cap, bias):
    """K and V are whole numbers times powers of two, exact: q's terms, the weights' and the sums are left."""
    heads, kv, lens = 4, 2, [1500, 90]
    h = Held(gpu, kv, hd, lens, 74)
    h.model.scale[:, :, 0] = 2.0 ** -6    # r.m.s. 73 / 64
    h.pool.upload(h.model.pool())
    first = _offsets([new, new])
    q = (np.random.default_rng(75).standard_normal((first[-1], heads * hd)) * 1.5).astype(np.float32)
    slopes = np.asarray([2.0 ** (-2 * (j + 1)) for j in range(heads)], np.float32) if bias else None
    got = h.attend(F32, q, first, heads, slopes=slopes, softcap=cap)
    o, _, _ = h.model.attention(q.astype(np.float64), first, lens, heads, True, None, cap, slopes)
    _near(got, o, F32, "%d new, cap %g bias %s" % (new, cap, bias), _tol(1.5 * 73 / 64, cap, bias))
