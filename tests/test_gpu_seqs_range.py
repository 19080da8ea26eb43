"""fh3_hip_attention_seqs_dev at the ends of the operands' ranges: scores of any
size, values near the type's largest and least, scales near fp32's least, keys
that are infinite.  The oracle is the 64-bit plain form; scores are built so that
both compute them exactly, or so that one key wins by far."""
import numpy as np
import pytest

import seqs_ref as R
from seqs_ref import BF16, F16, F32
from test_gpu_seqs import _case, _offsets, _run

pytestmark = pytest.mark.gpu


def _near(got, want, t, what, tol=None):
    """Relative Frobenius error within the type's (seqs_ref.FRO), nothing that is not finite."""
    got = R.from_type(got, t)
    big = np.abs(want).max()
    got, want = got / big, want / big      # (squares of the largest values would overflow)
    fro = float(np.linalg.norm(got - want) / np.linalg.norm(want))
    print("%s %s: rel_fro %.2e" % (what, R.NAMES[t], fro), flush=True)
    assert np.isfinite(got).all(), what
    assert fro <= (R.FRO[t] if tol is None else tol), (what, fro)


def exact_scores(seed, t, n, heads, kv, hd):
    """q, k, v whose products are +-2^30 + 128 n_j, exact in every type and in fp32 sums, n_j from 0 to 20."""
    rng = np.random.default_rng(seed)
    q, k = np.zeros((n, heads, hd)), np.zeros((n, kv, hd))
    q[:, :, 0] = np.where(np.arange(heads) % 2, -2.0 ** 15, 2.0 ** 15)
    q[:, :, hd - 1] = 128
    k[:, :, 0] = 2.0 ** 15
    k[:, :, hd - 1] = rng.integers(0, 21, (n, kv))
    v = rng.standard_normal((n, kv * hd))
    return [R.to_type(x.reshape(n, -1), t) for x in (q, k, v)]


# at 2^-7 neighbouring scores differ by 1 at 8 10^6; at 2^90 all are beyond 10^36
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** e for e in (-14, -7, -5, -4, -3, 0, 20, 40, 69, 90)])
def test_scores_of_any_size(gpu, t, hd, scale):
    heads, kv, lens = 4, 2, [300, 37]
    first = _offsets(lens)
    arrays = exact_scores(3, t, first[-1], heads, kv, hd)
    for causal in (True, False):
        got = _run(gpu, arrays, t, first, heads, kv, hd, scale=scale, causal=causal)
        o, _, _ = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd, causal, scale)
        _near(got, o, t, "scale %g causal %s" % (scale, causal))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("size", [5e3, 1e4, 1.5e4, 3e4])
def test_large_operands(gpu, t, size):
    """Scores of 10^8 to 10^10, whose fp32 sums are off by more than 1: only that each row is a mean of what it sees can be said."""
    heads, kv, hd, n = 4, 1, 128, 200
    rng = np.random.default_rng(4)
    q, k = (np.clip(rng.standard_normal((n, w * hd)) * size, -6e4, 6e4) for w in (heads, kv))
    arrays = [R.to_type(x, t) for x in (q, k, np.ones((n, kv * hd)))]
    got = R.from_type(_run(gpu, arrays, t, [0, n], heads, kv, hd), t)
    assert np.isfinite(got).all()
    # weights and their sum: half a step each (F32: two terms of the weights, 2^-21; sums of up to 200)
    assert np.abs(got - 1).max() <= (2.0 ** -20 if t == F32 else 2 * R.UNIT[t])
    arrays[2] = R.to_type(rng.standard_normal((n, kv * hd)), t)
    got = R.from_type(_run(gpu, arrays, t, [0, n], heads, kv, hd), t)
    v = R.from_type(arrays[2], t)
    assert np.isfinite(got).all() and np.abs(got[0].reshape(heads, hd) - v[0]).max() <= 2 * R.UNIT[t] * np.abs(v[0]).max() + 2.0 ** -20


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("slope", [1e8, -1e8, 1e30, -1e30])
def test_distance_bias_of_any_size(gpu, t, slope):
    """The nearest token wins, or the farthest, by far."""
    heads, kv, hd, lens = 2, 1, 64, [150, 40]
    first = _offsets(lens)
    arrays = _case(6, t, first[-1], heads, kv, hd)
    slopes = np.asarray([slope, slope / 3], np.float32)
    got = _run(gpu, arrays, t, first, heads, kv, hd, None, slopes)
    o, _, _ = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd, True, None, 0.0, slopes)
    _near(got, o, t, "slope %g" % slope)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_capped_scores_far_below_zero(gpu, t):
    """Every score is -10^30, the cap: the mean of what is seen."""
    heads, kv, hd, n = 2, 1, 64, 100
    arrays = exact_scores(7, t, n, heads, kv, hd)
    got = _run(gpu, arrays, t, [0, n], heads, kv, hd, scale=2.0 ** 75, softcap=1e30)
    o, _, _ = R.attention(*(R.from_type(x, t) for x in arrays), [0, n], heads, kv, hd, True, 2.0 ** 75, 1e30)
    _near(got, o, t, "cap")


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("scale,cap", [(1e-5, 1e30), (1e30, 1e-3), (1e-36, 1e-3), (1e25, 1e-8)])
def test_caps_far_from_the_scale(gpu, t, scale, cap):
    """Scores that are 0 beside the cap, or at the cap by far."""
    heads, kv, hd, lens = 4, 2, 64, [100, 30]
    first = _offsets(lens)
    arrays = _case(13, t, first[-1], heads, kv, hd)
    got = _run(gpu, arrays, t, first, heads, kv, hd, scale=scale, softcap=cap)
    o, _, _ = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd, True, scale, cap)
    _near(got, o, t, "scale %g cap %g" % (scale, cap))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1e-30, 1e-40, 1e-44])
def test_scales_near_the_least(gpu, t, scale):
    """All scores are 0 to within fp32: the mean of what is seen."""
    heads, kv, hd, lens = 4, 2, 128, [100, 9]
    first = _offsets(lens)
    arrays = _case(8, t, first[-1], heads, kv, hd)
    got = _run(gpu, arrays, t, first, heads, kv, hd, scale=scale)
    o, _, _ = R.attention(*(R.from_type(x, t) for x in arrays), first, heads, kv, hd, True, scale)
    _near(got, o, t, "scale %g" % scale)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size,n", [(3.3e38, 1000), (1e36, 3000), (1e-30, 300), (1e-34, 3000)])
def test_values_near_the_ends(gpu, t, hd, size, n):
    """V next to the type's largest and least normal values; the outputs are its means."""
    heads, kv = 4, 2
    q, k, _ = _case(9, t, n, heads, kv, hd)
    rng = np.random.default_rng(10)
    v = R.to_type(rng.uniform(0.5, 1.0, (n, kv * hd)) * np.where(rng.random((n, kv * hd)) < 0.25, -1, 1) * size, t)
    assert np.isfinite(R.from_type(v, t)).all()
    got = _run(gpu, (q, k, v), t, [0, n], heads, kv, hd)
    o, _, _ = R.attention(*(R.from_type(x, t) for x in (q, k, v)), [0, n], heads, kv, hd)
    _near(got, o, t, "v %g" % size)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("qs,ks", [(1e-32, 1e32), (1e-33, 2e34), (1e36, 1e-36), (1e-20, 1e34)])
def test_keys_near_the_ends(gpu, hd, qs, ks):
    """fp32 q and k at the two ends of the range, products of ordinary size (the last: of 10^14, one key wins)."""
    heads, kv, n = 4, 2, 300
    rng = np.random.default_rng(11)
    arrays = [(rng.standard_normal((n, w * hd)) * s).astype(np.float32) for w, s in ((heads, qs), (kv, ks), (kv, 1.0))]
    got = _run(gpu, arrays, F32, [0, n], heads, kv, hd)
    o, _, _ = R.attention(*(x.astype(np.float64) for x in arrays), [0, n], heads, kv, hd)
    _near(got, o, F32, "q %g k %g" % (qs, ks))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [0.0, 30.0, 1e4])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_infinite_keys(gpu, t, cap, bad):
    """A key with an infinite channel.  F16 and BF16: its score is infinite as the sign of q says: +inf makes the row
    NaN, -inf leaves the key out, and a cap takes either to +-cap.  F32: the row is NaN."""
    heads, kv, hd, n, at, ch = 4, 2, 64, 150, 70, 21
    arrays = _case(12, t, n, heads, kv, hd)
    arrays[1][at, hd + ch] = R.to_type(np.full(1, bad), t)[0]
    got = R.from_type(_run(gpu, arrays, t, [0, n], heads, kv, hd, softcap=cap), t).reshape(n, heads, hd)
    q, k, v = (R.from_type(x, t) for x in arrays)
    k0 = k.copy()
    k0[at, hd + ch] = 0
    o, _, _ = R.attention(q, k0, v, [0, n], heads, kv, hd, True, None, cap)
    o = o.reshape(n, heads, hd)
    _near(R.to_type(got[:at], t), o[:at], t, "before")
    _near(R.to_type(got[:, :2], t), o[:, :2], t, "the other key head")
    lost = 0
    for h in (2, 3):
        sign = np.sign(q[:, h * hd + ch]) * np.sign(bad)
        for r in range(at, n):
            if t == F32 or (not cap and sign[r] > 0):
                assert np.isnan(got[r, h]).all(), (r, h)
                lost += 1
                continue
            s = (k0[:r + 1, hd:] @ q[r, h * hd:(h + 1) * hd]) / np.sqrt(hd)
            s = cap * np.tanh(s / cap) if cap else s
            s[at] = sign[r] * cap if cap else -np.inf
            w = np.exp(s - s.max())
            want = w @ v[:r + 1, hd:] / w.sum()
            # half a step of the weights and one of the output, of the weighted |v|
            lim = 3 * R.UNIT[t] * (w @ np.abs(v[:r + 1, hd:]) / w.sum()) + 1e-5
            assert (np.abs(got[r, h] - want) <= lim).all(), (r, h)
    assert lost == (2 * (n - at) if t == F32 else 0 if cap else lost) and (cap or 0 < lost)
