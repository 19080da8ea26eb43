"""Ways of calling the sequence and cache entry points that the parity tests leave out: strides everywhere, rows
behind the last sequence, many empty sequences, several streams at once, replays of the fp32 forms, a thread of
its own."""
import ctypes
import threading

import numpy as np
import pytest

import seqs_ref as R
from seqs_ref import BF16, F16, F32
from test_gpu_kv import Held, _rows
from test_gpu_seqs import _buf, _case, _offsets, _run

pytestmark = pytest.mark.gpu


def _streams(F, n):
    out = []
    for _ in range(n):
        st = ctypes.c_void_p()
        assert F.lib().hipStreamCreateWithFlags(ctypes.byref(st), ctypes.c_uint(1)) == 0
        out.append(st)
    return out


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_cache_rows_at_strides(gpu, t):
    """k and v as parts of a projection's output, q and o with gaps: the same bits as dense rows, the gaps stay."""
    F, kv, hd, heads, lens, new = gpu, 2, 64, 8, [90, 70, 200], [20, 0, 130]
    first = _offsets(new)
    n, w, wq = first[-1], kv * hd, heads * hd
    q, k, v = _rows(1, t, n, wq), _rows(2, t, n, w), _rows(3, t, n, w)
    dense, wide = Held(F, kv, hd, lens, 4), Held(F, kv, hd, lens, 4)
    dense.append(t, k, v, first)
    gap = R.to_type(np.full((n, 8), 3), t)
    qkv = np.concatenate([q, gap, k, gap, v], 1)
    buf, size, ld = _buf(F, qkv), qkv.itemsize, qkv.shape[1]
    df = _buf(F, np.asarray(first, np.int32))
    at = [buf.ptr + x * size for x in (0, wq + 8, wq + w + 16)]
    F.kv_append_dev(wide.kv, t, at[1], at[2], n, 3, df, ldk=ld, ldv=ld)
    F.synchronize()
    assert np.array_equal(wide.pool.download(np.uint8, (wide.pool.nbytes,)), dense.pool.download(np.uint8, (dense.pool.nbytes,)))
    for rows in (n, 3):       # chunks, and one token each
        f = first if rows == n else [0, 1, 2, 3]
        want = dense.attend(t, q[:rows], f, heads)
        cfg = F.attn_cfg(heads, kv, hd, t)
        need = F.kv_attention_workspace_bytes(cfg, wide.kv, rows, 3)
        ws, df2 = F.DeviceBuffer(max(1, need)), _buf(F, np.asarray(f, np.int32))
        o = np.full((rows, wq + 24), 5, q.dtype)
        do = _buf(F, o)
        F.kv_attention_dev(cfg, wide.kv, buf, do, rows, 3, ws, need, df2, ldq=ld, ldo=wq + 24)
        F.synchronize()
        got = do.download(o.dtype, o.shape)
        assert np.array_equal(got[:, :wq], want) and (got[:, wq:] == 5).all()


def test_append_rows_behind_the_last_sequence(gpu):
    """Rows behind the last sequence are not written to the cache, whatever they hold."""
    F, kv, hd, lens, new = gpu, 2, 128, [70, 130], [3, 66]
    first = _offsets(new)
    a, b = Held(F, kv, hd, lens, 5), Held(F, kv, hd, lens, 5)
    k, v = _rows(6, F32, first[-1], kv * hd), _rows(7, F32, first[-1], kv * hd)
    a.append(F32, k, v, first)
    tail = np.full((40, kv * hd), 1e9, np.float32)
    dk, dv, df = (_buf(F, x) for x in (np.concatenate([k, tail]), np.concatenate([v, tail]), np.asarray(first, np.int32)))
    F.kv_append_dev(b.kv, F32, dk, dv, first[-1] + 40, 2, df)
    F.synchronize()
    assert np.array_equal(a.pool.download(np.uint8, (a.pool.nbytes,)), b.pool.download(np.uint8, (b.pool.nbytes,)))


@pytest.mark.parametrize("t", [F32, BF16])
def test_many_empty_sequences(gpu, t):
    """More sequences than rows, nearly all empty: over packed rows, appended, attended."""
    F, kv, hd, heads, n_seq = gpu, 2, 64, 4, 700
    new = [0] * n_seq
    for s, c in ((3, 5), (64, 1), (65, 70), (699, 2)):
        new[s] = c
    first = _offsets(new)
    arrays = _case(8, t, first[-1], heads, kv, hd)
    got = _run(F, arrays, t, first, heads, kv, hd)
    assert np.array_equal(got, _run(F, arrays, t, [0, 5, 6, 76, 78], heads, kv, hd))
    lens = [(c + 60) if c else 0 for c in new]
    h = Held(F, kv, hd, lens, 9)
    h.append(t, arrays[1], arrays[2], first)
    h.same()
    o, a, big = h.model.attention(R.from_type(arrays[0], t), first, lens, heads)
    # (bound: the cache's weights are fp16's, whose least step is 2^-31 of the sum of the |v| seen)
    got = h.attend(t, arrays[0], first, heads)
    R.check(got, t, o, a, big, hd, max(lens), "empty sequences", 2.0 ** -31 * 130 * np.abs(R.from_type(arrays[2], t)).max() * 4)


@pytest.mark.parametrize("heads,kv,hd,lens", [(64, 8, 128, [600]), (64, 8, 128, [37]), (16, 16, 64, [300, 1, 250]), (16, 2, 128, [200, 90, 400])])
def test_fp32_replays_and_streams_at_once(gpu, heads, kv, hd, lens):
    """The fp32 forms captured, and four calls of different inputs on four streams at once: the eager bits."""
    F, first = gpu, _offsets(lens)
    n = first[-1]
    sides, cfg, df = [], F.attn_cfg(heads, kv, hd, F32), _buf(F, np.asarray(first, np.int32))
    for i, st in enumerate(_streams(F, 4)):
        arrays = _case(20 + i, F32, n, heads, kv, hd)
        want = _run(F, arrays, F32, first, heads, kv, hd)
        bufs = [_buf(F, x) for x in arrays] + [F.DeviceBuffer(arrays[0].nbytes)]
        g = F.capture(lambda: F.attention_seqs_dev(cfg, *bufs, n, len(lens), df))
        sides.append((st, bufs, want, g))
    for r in range(3):
        for st, bufs, want, g in sides:
            bufs[3].fill(0)
        F.synchronize()
        for st, bufs, want, g in sides:
            if r == 1:
                g.launch(st.value)
            else:
                F.attention_seqs_dev(cfg, *bufs, n, len(lens), df, stream_ptr=st.value)
        F.synchronize()
        for st, bufs, want, g in sides:
            assert np.array_equal(bufs[3].download(want.dtype, want.shape), want), r
    for st, bufs, want, g in sides:
        g.close()
        assert F.lib().hipStreamDestroy(st) == 0


def test_append_and_read_replayed(gpu):
    """Append and read-back captured together and replayed with other rows and lengths."""
    F, t, kv, hd, n = gpu, F16, 2, 64, 4
    h = Held(F, kv, hd, [200, 70, 130, 64], 30)
    kb, vb = F.DeviceBuffer(n * kv * hd * 2), F.DeviceBuffer(n * kv * hd * 2)
    ko, vo = F.DeviceBuffer(kb.nbytes), F.DeviceBuffer(vb.nbytes)

    def step():
        F.kv_append_dev(h.kv, t, kb, vb, n, n)
        F.kv_read_dev(h.kv, t, ko, vo, n, n)

    g = F.capture(step)
    try:
        for r, lens in enumerate(([100, 70, 66, 1], [101, 65, 67, 64], [102, 64, 128, 2])):
            k, v = _rows(31 + r, t, n, kv * hd, 3.0 ** r), _rows(41 + r, t, n, kv * hd, 0.3)
            kb.upload(k)
            vb.upload(v)
            h.len.upload(np.asarray(lens, np.int32))
            g.launch()
            F.synchronize()
            h.lens = lens
            h.model.append((R.from_type(k, t), R.from_type(v, t)), [0, 1, 2, 3, 4], lens)
            h.same()
            for got, want in zip((ko, vo), h.model.read([0, 1, 2, 3, 4], lens)):
                assert np.array_equal(got.download(np.float16, (n, kv * hd)).astype(np.float64), want)
    finally:
        g.close()


def test_threads_of_their_own(gpu):
    """Four host threads, each with its own arrays, workspace and stream, over packed rows and over one cache."""
    F, t, heads, kv, hd, lens = gpu, BF16, 16, 2, 128, [1500, 90, 700]
    h = Held(F, kv, hd, lens, 50)
    cfg, first = F.attn_cfg(heads, kv, hd, t), [0, 1, 2, 3]
    need = F.kv_attention_workspace_bytes(cfg, h.kv, 3, 3)
    df = _buf(F, np.asarray(first, np.int32))
    jobs, wrong = [], []
    for i, st in enumerate(_streams(F, 4)):
        q = _rows(51 + i, t, 3, heads * hd)
        jobs.append((st, h.attend(t, q, first, heads), _buf(F, q), F.DeviceBuffer(q.nbytes), F.DeviceBuffer(max(1, need))))
    F.synchronize()

    def work(st, want, dq, do, ws):
        try:
            for _ in range(10):
                F.kv_attention_dev(cfg, h.kv, dq, do, 3, 3, ws, need, df, stream_ptr=st.value)
            assert F.lib().hipStreamSynchronize(st) == 0
            if not np.array_equal(do.download(want.dtype, want.shape), want):
                wrong.append("other bits")
        except Exception as e:  # noqa: BLE001  (told to the main thread)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong
    for j in jobs:
        assert F.lib().hipStreamDestroy(j[0]) == 0
