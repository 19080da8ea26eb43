"""Ways of calling the microscaled entry points that the parity tests leave out: a block's calls one after the other,
several streams and threads at once, replays, arrays past 4 GiB, what stands behind the last row."""
import threading

import numpy as np
import pytest

from mx_ref import BF16, F16, F32, FP4, FP8, HALF, Mx, buf, from_type, quantize, random_rows, scale_bytes, strides, to_type, unit, unpack, values
from test_gpu_mx import Case, _check_quantized, _norm_exact, _product_bound, NORM_REL
from test_gpu_seqs_calls import _streams

pytestmark = pytest.mark.gpu


def _empty(F, fmt, rows, n):
    return Mx(F, fmt, rows, n, pad=0)


class Layer:
    """The calls of a transformer block around its attention, at sizes of its own: norm, projection, attention's output
    back to codes, gated residual, norm, SwiGLU, gated residual; x and h in fp32."""

    def __init__(self, F, seed, rows, hidden=256, heads=2, hd=128, ff=384, fmt=FP8):
        rng = np.random.default_rng(seed)
        inner = heads * hd
        self.F, self.rows, self.hidden, self.heads, self.hd, self.ff, self.inner = F, rows, hidden, heads, hd, ff, inner
        self.w = {}
        for name, out, n in (("qkv", 3 * inner, hidden), ("out", hidden, inner), ("fc1", 2 * ff, hidden), ("fc2", hidden, ff)):
            c, s, v = random_rows(rng, out, n, FP4, 0.5)
            s = (s - 4).astype(np.uint8)      # weights of about 1 / 16
            self.w[name] = (Mx(F, FP4, out, n, c, s), values(c, s, FP4))
        self.norm = [1 + 0.1 * rng.standard_normal(hidden).astype(np.float32) for _ in range(2)]
        self.mod = [0.2 * rng.standard_normal((rows, hidden)).astype(np.float32) for _ in range(6)]   # shift, scale, gate twice
        self.x, self.add = (rng.standard_normal((rows, hidden)).astype(np.float32) for _ in range(2))
        self.d = {"x": buf(F, self.x), "add": buf(F, self.add), "h": F.DeviceBuffer(self.x.nbytes), "qkv": F.DeviceBuffer(rows * 3 * inner * 4),
                  "att": F.DeviceBuffer(rows * inner * 4), "h1": F.DeviceBuffer(self.x.nbytes), "h2": F.DeviceBuffer(self.x.nbytes)}
        self.d["norm"], self.d["mod"] = [buf(F, a) for a in self.norm], [buf(F, a) for a in self.mod]
        self.n1, self.n2 = _empty(F, fmt, rows, hidden), _empty(F, fmt, rows, hidden)
        self.a, self.act = _empty(F, fmt, rows, inner), _empty(F, fmt, rows, ff)
        pairs = (("qkv", self.n1, False), ("out", self.a, False), ("fc1", self.n2, True), ("fc2", self.act, False))
        self.need = max(F.mx_matmul_workspace_bytes(self.w[k][0].mx, m.mx, s) for k, m, s in pairs)
        self.ws = F.DeviceBuffer(max(1, self.need))

    def run(self, stream=None):
        F, d, st = self.F, self.d, dict(stream_ptr=stream)
        mod, w = d["mod"], {k: v[0].mx for k, v in self.w.items()}
        F.mx_norm_dev(F32, d["x"], d["norm"][0], 1e-6, self.n1.mx, d_add=d["add"], d_sum=d["h"], d_shift=mod[0], d_scale=mod[1], **st)
        F.mx_matmul_dev(w["qkv"], self.n1.mx, F32, d["qkv"], self.ws, self.need, **st)
        cfg = F.attn_cfg(self.heads, self.heads, self.hd, F32, causal=True)
        ld = 3 * self.inner
        F.attention_seqs_dev(cfg, d["qkv"].ptr, d["qkv"].ptr + 4 * self.inner, d["qkv"].ptr + 8 * self.inner, d["att"], self.rows, ldq=ld, ldk=ld,
                             ldv=ld, **st)
        F.mx_quantize_dev(F32, d["att"], self.a.mx, **st)
        F.mx_matmul_dev(w["out"], self.a.mx, F32, d["h1"], self.ws, self.need, d_gate=mod[2], d_res=d["h"], **st)
        F.mx_norm_dev(F32, d["h1"], d["norm"][1], 1e-6, self.n2.mx, d_shift=mod[3], d_scale=mod[4], **st)
        F.mx_matmul_swiglu_dev(w["fc1"], self.n2.mx, self.act.mx, self.ws, self.need, **st)
        F.mx_matmul_dev(w["fc2"], self.act.mx, F32, d["h2"], self.ws, self.need, d_gate=mod[5], d_res=d["h1"], **st)

    def got(self, name, n):
        return self.d[name].download(np.float32, (self.rows, n))

    def outputs(self):
        return [self.got("h2", self.hidden), self.got("h1", self.hidden), *self.act.read(), *self.n2.read(), *self.a.read()]


def _held(y, want, xv, wv, gate, res):
    b, _ = _product_bound(xv, wv, F32, True, want)
    f = 1.0 if gate is None else np.abs(gate)
    assert (np.abs(y - want) <= b * f + 2.0 ** -22 * (np.abs(want) + (0 if res is None else np.abs(res)))).all()


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("rows", [1, 19, 150, 700])
def test_a_blocks_calls(gpu, rows, fmt):
    """Each call's output against the formula of what it was given by the one before."""
    b = Layer(gpu, rows, rows, fmt=fmt)
    b.run()
    gpu.synchronize()
    h = b.got("h", b.hidden)
    assert np.array_equal(h, b.x + b.add)
    size = lambda x, i: np.abs(_norm_exact(x.astype(np.float64), b.norm[i // 3], 1e-6)) * (1 + np.abs(b.mod[i + 1])) + np.abs(b.mod[i])  # noqa: E731
    for mx, x, i in ((b.n1, h, 0), (b.n2, b.got("h1", b.hidden), 3)):
        exact = _norm_exact(x.astype(np.float64), b.norm[i // 3].astype(np.float64), 1e-6, b.mod[i], b.mod[i + 1])
        codes, s = mx.read()
        half = np.maximum(np.abs(exact) * 2.0 ** (-2 if fmt == FP4 else -4),
                          (0.25 if fmt == FP4 else 2.0 ** -10) * np.repeat(np.exp2(s.astype(np.float64) - 127), 32, 1))
        assert (np.abs(values(codes, s, fmt) - exact) <= half + NORM_REL * size(x, i)).all()
    xv = values(*b.n1.read(), fmt)
    qkv = b.got("qkv", 3 * b.inner)
    _held(qkv, xv @ b.w["qkv"][1].T, xv, b.w["qkv"][1], None, None)
    assert np.array_equal(np.concatenate(b.a.read(), 1), np.concatenate(quantize(b.got("att", b.inner), fmt), 1))
    for mx, wname, gate, res, out in ((b.a, "out", b.mod[2], h, "h1"), (b.act, "fc2", b.mod[5], b.got("h1", b.hidden), "h2")):
        xv, wv = values(*mx.read(), fmt), b.w[wname][1]
        want = res.astype(np.float64) + gate * (xv @ wv.T)
        _held(b.got(out, b.hidden), want, xv, wv, gate, res)
    y = values(*b.n2.read(), fmt) @ b.w["fc1"][1].T
    act = y[:, :b.ff] * y[:, b.ff:] / (1 + np.exp(-y[:, b.ff:]))
    got = values(*b.act.read(), fmt)
    # half a step of codes, at the least of the block's largest; the products' own error is far below it
    step = np.repeat(np.abs(act).reshape(rows, -1, 32).max(-1), 32, 1)
    assert (np.abs(got - act) <= np.abs(act) * 2.0 ** (-2 if fmt == FP4 else -4) + step * 2.0 ** (-3 if fmt == FP4 else -14) + 1e-3 * step).all()


def test_streams_and_threads_at_once(gpu):
    """Blocks of different sizes on streams of their own, from threads of their own: the same bits as one after the other."""
    rows = (1, 30, 130, 600)
    layers = [Layer(gpu, 50 + r, r) for r in rows]
    for b in layers:
        b.run()
    gpu.synchronize()
    want = [b.outputs() for b in layers]
    streams = _streams(gpu, len(rows))
    for _ in range(3):
        for b, st in zip(layers, streams):
            b.run(st)
    gpu.synchronize()
    for st in streams:
        assert gpu.lib().hipStreamSynchronize(st) == 0
    assert all(np.array_equal(x, y) for b, w in zip(layers, want) for x, y in zip(b.outputs(), w))
    errors = []

    def work(b, st):
        try:
            for _ in range(20):
                b.run(st)
            assert gpu.lib().hipStreamSynchronize(st) == 0
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(layers, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(np.array_equal(x, y) for b, w in zip(layers, want) for x, y in zip(b.outputs(), w))


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_replays(gpu, rows):
    """A captured block, replayed with other inputs, eager calls and synchronisations between: as eager each time."""
    b, other = Layer(gpu, 7, rows), Layer(gpu, 8, rows)
    b.run()
    other.run()
    gpu.synchronize()
    graph = gpu.capture(b.run)
    for i in range(5):
        x = np.random.default_rng(i).standard_normal(b.x.shape).astype(np.float32) * np.float32(1 + i)
        b.d["x"].upload(x)
        b.run()
        gpu.synchronize()
        want = b.outputs()
        for k in ("h2", "h1"):
            b.d[k].fill(0xFF)
        for m in (b.act, b.n2, b.a):
            m.dc.fill(0)
            m.ds.fill(0)
        other.run()
        graph.launch()
        if i % 2:
            other.run()
        gpu.synchronize()
        assert all(np.array_equal(p, q) for p, q in zip(b.outputs(), want)), i


@pytest.mark.parametrize("rows,out,n", [(1, 40, 512), (20, 100, 288), (150, 130, 640), (150, 200, 4096), (600, 520, 256)])
@pytest.mark.parametrize("t", [F32, BF16])
def test_behind_the_last_row(gpu, rows, out, n, t):
    """Nothing behind the last row of y, of codes and scales, or of the workspace is written."""
    F = gpu
    c = Case(rows + out, rows, n, out, FP8)
    x, w = Mx(F, FP8, rows, n, *c.x[:2]), Mx(F, FP4, out, n, *c.w[:2])
    kind = to_type(np.zeros(1, np.float32), t).dtype
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx)
    full = np.full(rows * out + 5000, 9, kind)
    dy, ws = buf(F, full), F.DeviceBuffer(need + 4096)
    ws.fill(0x5A)
    F.mx_matmul_dev(w.mx, x.mx, t, dy, ws, need)
    F.synchronize()
    got = dy.download(kind, full.shape)
    assert (got[rows * out:] == 9).all()
    c.check(got[:rows * out].reshape(rows, out), t)
    assert (ws.download(np.uint8, (need + 4096,))[need:] == 0x5A).all()
    if out % 128 == 0 or out == 520:
        return
    f = 128
    w2 = Mx(F, FP4, 2 * f, n, *random_rows(np.random.default_rng(1), 2 * f, n, FP4)[:2])
    lc, ls = strides(FP8, f)
    dc, ds = buf(F, np.full(rows * lc + 512, 3, np.uint8)), buf(F, np.full(rows * ls + 64, 3, np.uint8))
    need = F.mx_matmul_workspace_bytes(w2.mx, x.mx, True)
    ws = F.DeviceBuffer(max(1, need))
    F.mx_matmul_swiglu_dev(w2.mx, x.mx, F.mx(FP8, rows, f, dc, ds), ws, need)
    F.mx_quantize_dev(F32, buf(F, np.ones((rows, f), np.float32)), F.mx(FP8, rows, f, dc, ds))
    F.synchronize()
    assert (dc.download(np.uint8, (rows * lc + 512,))[rows * lc:] == 3).all() and (ds.download(np.uint8, (rows * ls + 64,))[rows * ls:] == 3).all()


def _tail(F, b, at, a):
    a = np.ascontiguousarray(a)
    assert F.lib().fh3_hip_memcpy_htod(b.ptr + at, a.ctypes.data, a.nbytes) == 0


@pytest.mark.parametrize("rows,fmt", [(1, FP8), (3, FP4), (100, FP8), (300, FP4)])
def test_weights_past_4_gib(gpu, rows, fmt):
    """Weight rows and outputs whose offsets pass 32 bits: the last rows come out as in a matrix of their own."""
    F, n, out, last = gpu, 8192, 1_100_000, 300
    rng = np.random.default_rng(rows)
    c, s, _ = random_rows(rng, last, n, FP4)
    xc, xs, _ = random_rows(rng, rows, n, fmt)
    wc, wsc = F.DeviceBuffer(out * n // 2), F.DeviceBuffer(out * n // 32)
    wc.fill(0)
    wsc.fill(127)
    _tail(F, wc, (out - last) * (n // 2), c[:, ::2] | c[:, 1::2] << 4)
    _tail(F, wsc, (out - last) * (n // 32), s)
    x, w, few = Mx(F, fmt, rows, n, xc, xs), F.mx(FP4, out, n, wc, wsc), Mx(F, FP4, last, n, c, s)
    y, small = F.DeviceBuffer(rows * out * 4), F.DeviceBuffer(rows * last * 4)
    need = F.mx_matmul_workspace_bytes(w, x.mx)
    ws = F.DeviceBuffer(max(1, need, F.mx_matmul_workspace_bytes(few.mx, x.mx)))
    F.mx_matmul_dev(w, x.mx, F32, y, ws, ws.nbytes)
    F.mx_matmul_dev(few.mx, x.mx, F32, small, ws, ws.nbytes)
    F.synchronize()
    want = small.download(np.float32, (rows, last))
    xv, wv = values(xc, xs, fmt), values(c, s, FP4)
    bound, _ = _product_bound(xv, wv, F32, fmt == FP8, want)
    for r in {0, rows // 2, rows - 1}:
        row = np.empty(out, np.float32)
        assert F.lib().fh3_hip_memcpy_dtoh(row.ctypes.data, y.ptr + r * out * 4, row.nbytes) == 0
        assert (row[:out - last] == 0).all()
        assert (np.abs(row[out - last:] - want[r]) <= 2 * bound[r]).all()


@pytest.mark.parametrize("fmt", [FP4, FP8])
def test_rows_past_4_gib(gpu, fmt):
    """Quantisation, read-back and norm of rows whose offsets pass 32 bits."""
    F, n, rows, last = gpu, 32768, 270_000, 5
    x = np.random.default_rng(4).standard_normal((last, n)).astype(np.float32)
    big = F.DeviceBuffer(rows * n * 2)
    big.fill(0)
    xb = to_type(x, BF16)
    _tail(F, big, (rows - last) * n * 2, xb)
    lc, ls = strides(fmt, n)
    dc, ds, back = F.DeviceBuffer(rows * lc), F.DeviceBuffer(rows * ls), F.DeviceBuffer(rows * n * 2)
    m = F.mx(fmt, rows, n, dc, ds)
    want = quantize(from_type(xb, BF16), fmt)

    def read(b, at, shape, dtype):
        a = np.empty(shape, dtype)
        assert F.lib().fh3_hip_memcpy_dtoh(a.ctypes.data, b.ptr + at, a.nbytes) == 0
        return a

    F.mx_quantize_dev(BF16, big, m)
    F.mx_dequant_dev(m, BF16, back)
    F.synchronize()
    assert np.array_equal(unpack(read(dc, (rows - last) * lc, (last, lc), np.uint8), fmt), want[0])
    assert np.array_equal(read(ds, (rows - last) * ls, (last, ls), np.uint8), want[1])
    assert np.array_equal(read(back, (rows - last) * n * 2, (last, n), np.uint16), to_type(values(*want, fmt).astype(np.float32), BF16))
    F.mx_norm_dev(BF16, big, buf(F, np.ones(n, np.float32)), 1e-6, m)
    F.synchronize()
    got = unpack(read(dc, (rows - last) * lc, (last, lc), np.uint8), fmt), read(ds, (rows - last) * ls, (last, ls), np.uint8)
    _check_quantized(got, _norm_exact(from_type(xb, BF16), np.ones(n), 1e-6), fmt, NORM_REL)


@pytest.mark.parametrize("rows", [1, 50, 200, 520])
def test_the_same_bits_each_time(gpu, rows):
    c = Case(rows, rows, 2080, 390, FP8, bias=True, gate=True)
    for t in (F32, F16, BF16):
        y = c.run(gpu, t)
        assert all(np.array_equal(c.run(gpu, t), y) for _ in range(3))


@pytest.mark.parametrize("call", ["quantize", "norm"])
def test_more_rows_than_a_launch_dimension_has_lanes_for(gpu, call):
    """Rows of bf16 values (64 GiB) with 1024 lanes to each row of the norm, 256 of the quantisation: 2^32 lanes and more."""
    F, n, rows, last = gpu, 8192, (1 << 22) + 3, 5
    if call == "quantize":
        n, rows = 2048, (1 << 24)
    x = to_type(np.random.default_rng(6).standard_normal((last, n)).astype(np.float32), BF16)
    big = F.DeviceBuffer(rows * n * 2)
    big.fill(0)
    _tail(F, big, (rows - last) * n * 2, x)
    lc, ls = strides(FP4, n)
    dc, ds = F.DeviceBuffer(rows * lc), F.DeviceBuffer(rows * ls)
    dc.fill(0xEE)
    m = F.mx(FP4, rows, n, dc, ds)
    if call == "norm":
        F.mx_norm_dev(BF16, big, buf(F, np.ones(n, np.float32)), 1e-6, m)
    else:
        F.mx_quantize_dev(BF16, big, m)
    F.synchronize()

    def read(b, at, shape):
        a = np.empty(shape, np.uint8)
        assert F.lib().fh3_hip_memcpy_dtoh(a.ctypes.data, b.ptr + at, a.nbytes) == 0
        return a

    for r in (0, rows // 2, 1 << 21, rows - last - 1):
        assert not read(dc, r * lc, (1, lc)).any()
    got = unpack(read(dc, (rows - last) * lc, (last, lc)), FP4), read(ds, (rows - last) * ls, (last, ls))
    if call == "norm":
        _check_quantized(got, _norm_exact(from_type(x, BF16), np.ones(n), 1e-6), FP4, NORM_REL)
    else:
        want = quantize(from_type(x, BF16), FP4)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        big.fill(0x77)
        F.mx_dequant_dev(m, BF16, big)
        F.synchronize()
        a = np.empty((last, n), np.uint16)
        assert F.lib().fh3_hip_memcpy_dtoh(a.ctypes.data, big.ptr + (rows - last) * n * 2, a.nbytes) == 0
        assert np.array_equal(a, to_type(values(*want, FP4).astype(np.float32), BF16))


class Repeated:
    """Many rows made of few: copy k of the base rows has 2^(k % 5) times their scales (weights: % 7), so that the
    outputs of all follow from the products of the base rows."""

    def __init__(self, seed, rows, n, out, fmt, base_x=90, base_w=130):
        rng = np.random.default_rng(seed)
        self.rows, self.n, self.out, self.fmt = rows, n, out, fmt
        self.x, self.w = random_rows(rng, base_x, n, fmt, 0.3), random_rows(rng, base_w, n, FP4, 0.3)
        self.ix, self.iw = np.arange(rows) % base_x, np.arange(out) % base_w
        self.px, self.pw = np.arange(rows) // base_x % 5, np.arange(out) // base_w % 7

    def arrays(self, F):
        def of(part, i, p, fmt):
            return Mx(F, fmt, len(i), self.n, part[0][i], (part[1][i] - 6 + p[:, None]).astype(np.uint8))
        return of(self.x, self.ix, self.px, self.fmt), of(self.w, self.iw, self.pw, FP4)

    def exact(self, t):
        """The products and the bound on their sums."""
        y = self.x[2] @ self.w[2].T * 2.0 ** -12
        b, _ = _product_bound(self.x[2], self.w[2], t, self.fmt == FP8, y)
        k = np.exp2(self.px[:, None] + self.pw[None])
        at = np.ix_(self.ix, self.iw)
        return y[at] * k, b[at] * k * 2.0 ** -12


def _scaled_back(c, rows):
    """Case-like rows of c for the bias, gate and residual of tests."""
    rng = np.random.default_rng(rows)
    return rng.standard_normal(c.out).astype(np.float32), rng.standard_normal((rows, c.out)).astype(np.float32), rng.standard_normal((rows, c.out))


# few rows against many weights, whole and in parts of the rows' length, ragged in both directions
MANY_WEIGHTS = [(5088, 15361), (25632, 5130), (2080, 40003)]


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("t,extra", [(F32, False), (F32, True), (BF16, True)])
@pytest.mark.parametrize("n,out", MANY_WEIGHTS)
@pytest.mark.parametrize("rows", [1, 15, 17, 33, 64])
def test_few_rows_many_weights(gpu, rows, n, out, t, extra, fmt):
    F, c = gpu, Repeated(rows + n, rows, n, out, fmt, base_x=rows)
    x, w = c.arrays(F)
    want, b = c.exact(t)
    kind, ld = to_type(np.zeros(1, np.float32), t).dtype, out + 5
    full = np.full(3 + rows * ld, 77, kind)
    kw, size, at = {}, np.abs(want), 3 * kind.itemsize
    y = F.DeviceBuffer.from_array(full)
    if extra:
        bias, gate, res = _scaled_back(c, rows)
        res = to_type(4 * res, t)
        r = from_type(res, t).astype(np.float64)
        want, b, size = r + gate * (want + bias), b * np.abs(gate), np.abs(r) + np.abs(gate) * (size + np.abs(bias))
        full[3:].reshape(rows, ld)[:, :out] = res
        y = buf(F, full)
        kw = dict(d_bias=buf(F, bias), d_gate=buf(F, gate), d_res=y.ptr + at, ldres=ld)
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx)
    ws = F.DeviceBuffer(need + 1024)
    ws.fill(0xFF)
    F.mx_matmul_dev(w.mx, x.mx, t, y.ptr + at, ws, need, ldy=ld, **kw)
    F.synchronize()
    got = y.download(kind, full.shape)
    rest = got[3:].reshape(rows, ld)
    assert (got[:3] == 77).all() and (rest[:, out:] == 77).all() and (ws.download(np.uint8, (need + 1024,))[need:] == 0xFF).all()
    bad = np.abs(from_type(rest[:, :out], t).astype(np.float64) - want) - (b + 2.0 ** -22 * size + HALF[t] * np.abs(want))
    assert (bad <= 0).all(), (float(bad.max()), np.argwhere(~(bad <= 0))[:3])


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("n,out", MANY_WEIGHTS)
@pytest.mark.parametrize("rows", [2, 30, 50])
def test_few_rows_many_weights_nan_rows(gpu, rows, n, out, fmt):
    F, c = gpu, Repeated(rows + n, rows, n, out, fmt, base_x=rows)
    x, w = c.arrays(F)
    y, need = F.DeviceBuffer(rows * out * 4), F.mx_matmul_workspace_bytes(w.mx, x.mx)
    ws = F.DeviceBuffer(max(1, need))

    def run():
        y.fill(0)
        F.mx_matmul_dev(w.mx, x.mx, F32, y, ws, need)
        F.synchronize()
        return y.download(np.float32, (rows, out))

    clean = run()
    _tail(F, x.ds, (rows - 1) * strides(fmt, n)[1] + n // 32 - 1, np.array([255], np.uint8))
    _tail(F, w.ds, (out - 1) * strides(FP4, n)[1], np.array([255], np.uint8))
    _tail(F, w.ds, 700 * strides(FP4, n)[1] + 33, np.array([255], np.uint8))
    bad = run()
    nan = np.zeros(clean.shape, bool)
    nan[rows - 1], nan[:, out - 1], nan[:, 700] = True, True, True
    assert np.array_equal(np.isnan(bad), nan) and np.array_equal(bad[~nan], clean[~nan])


# many tiles, whole, in parts of the rows' length, and with a last round of smaller ones: the larger tiles
LARGE = [(1930, 1824, 4401), (422, 16480, 5532), (2100, 1824, 8101)]


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("t,off,more,extra", [(F32, 0, 7, False), (BF16, 0, 7, True), (F16, 1, 4, True), (F32, 0, 3, True)])
@pytest.mark.parametrize("rows,n,out", LARGE)
def test_large_products(gpu, rows, n, out, t, off, more, extra, fmt):
    F, c = gpu, Repeated(rows, rows, n, out, fmt)
    x, w = c.arrays(F)
    want, b = c.exact(t)
    rng = np.random.default_rng(1)
    kind, ld = to_type(np.zeros(1, np.float32), t).dtype, out + more
    full = np.full(off + rows * ld, 77, kind)
    kw = {}
    size = np.abs(want)
    if extra:
        bias, gate = rng.standard_normal(out).astype(np.float32), rng.standard_normal((rows, out)).astype(np.float32)
        res = to_type(4 * rng.standard_normal((rows, out)).astype(np.float32), t)
        r = from_type(res, t).astype(np.float64)
        want, b, size = r + gate * (want + bias), b * np.abs(gate), np.abs(r) + np.abs(gate) * (size + np.abs(bias))
        kw = dict(d_bias=buf(F, bias), d_gate=buf(F, gate), d_res=buf(F, res))
    y = buf(F, full)
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx)
    assert (need > 0) == (rows == 422)
    ws = F.DeviceBuffer(max(1, need))
    ws.fill(0xFF)
    F.mx_matmul_dev(w.mx, x.mx, t, y.ptr + off * kind.itemsize, ws, need, ldy=ld, **kw)
    F.synchronize()
    got = y.download(kind, full.shape)
    rest = got[off:].reshape(rows, ld)
    assert (got[:off] == 77).all() and (rest[:, out:] == 77).all()
    bad = np.abs(from_type(rest[:, :out], t).astype(np.float64) - want) - (b + 2.0 ** -22 * size + HALF[t] * np.abs(want))
    assert (bad <= 0).all(), (float(bad.max()), np.argwhere(~(bad <= 0))[:3])


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("to", [FP8, FP4])
@pytest.mark.parametrize("rows,n,out", [(1930, 1824, 4480), (422, 16480, 5504), (2100, 1824, 8192), (1, 5088, 40064), (19, 5088, 40064), (40, 5088, 40064), (64, 2080, 40064),
                                        (12, 13856, 20096), (30, 13856, 20096), (60, 13856, 20096)])
def test_large_swiglu(gpu, rows, n, out, to, fmt):
    F, c, f = gpu, Repeated(rows + 1, rows, n, out, fmt), out // 2
    x, w = c.arrays(F)
    y, b = c.exact(BF16)
    o = Mx(F, to, rows, f)
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx, True)
    assert rows not in (422, 1930) or (need > 0) == (rows == 422)
    ws = F.DeviceBuffer(max(1, need))
    ws.fill(0xFF)
    F.mx_matmul_swiglu_dev(w.mx, x.mx, o.mx, ws, need)
    F.synchronize()
    codes, s = o.read()
    val, gate = y[:, :f], y[:, f:]
    with np.errstate(over="ignore"):
        act = val * gate / (1 + np.exp(-gate))
    # as in the small cases: through silu (slope at most 1.1) and val, and six roundings
    b = b + 2.0 ** -23 * np.abs(y)
    tol = np.abs(gate) * b[:, :f] + 1.1 * np.abs(val) * b[:, f:] + 1.1 * b[:, :f] * b[:, f:] + np.abs(act) * (8 + np.abs(gate)) * 2.0 ** -23
    amax, blocks = np.abs(act).reshape(rows, -1, 32), tol.reshape(rows, -1, 32)
    lo, hi = scale_bytes(np.maximum(amax - blocks, 0).max(-1), to), scale_bytes((amax + blocks).max(-1), to)
    assert ((s >= lo) & (s <= hi)).all()
    half = np.maximum(np.abs(act) * (2.0 ** -2 if to == FP4 else 2.0 ** -4), (0.25 if to == FP4 else 2.0 ** -10) * np.repeat(unit(s), 32, 1))
    off = np.abs(values(codes, s, to) - act)
    assert (off <= half + 1.25 * tol).all(), float((off - half - 1.25 * tol).max())


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("rows,out", [(1930, 4401), (2100, 8101)])
def test_large_products_nan_rows(gpu, rows, out, fmt):
    F, c = gpu, Repeated(3, rows, 1824, out, fmt)
    x, w = c.arrays(F)
    y = F.DeviceBuffer(rows * out * 4)

    def run():
        y.fill(0)
        F.mx_matmul_dev(w.mx, x.mx, F32, y, None, 0)
        F.synchronize()
        return y.download(np.float32, (rows, out))

    clean = run()
    _tail(F, x.ds, 1000 * strides(fmt, 1824)[1] + 56, np.array([255], np.uint8))
    _tail(F, w.ds, (out - 1) * strides(FP4, 1824)[1], np.array([255], np.uint8))
    bad = run()
    nan = np.zeros(clean.shape, bool)
    nan[1000], nan[:, out - 1] = True, True
    assert np.array_equal(np.isnan(bad), nan) and np.array_equal(bad[~nan], clean[~nan])


@pytest.mark.parametrize("fmt", [FP8, FP4])
@pytest.mark.parametrize("rows,out", [(1, 20), (20, 33), (40, 300), (70, 20), (300, 130)])
def test_the_longest_rows(gpu, rows, out, fmt):
    F, n = gpu, 1 << 20
    c = Repeated(rows, rows, n, out, fmt, base_x=3, base_w=5)
    x, w = c.arrays(F)
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx)
    ws, y = F.DeviceBuffer(max(1, need)), F.DeviceBuffer(rows * out * 4)
    ws.fill(0xFF)
    for t in (F32, BF16):
        want, b = c.exact(t)
        F.mx_matmul_dev(w.mx, x.mx, t, y, ws, need)
        F.synchronize()
        got = from_type(y.download(to_type(np.zeros(1, np.float32), t).dtype, (rows, out)), t)
        assert (np.abs(got - want) <= b + 2.0 ** -22 * np.abs(want) + HALF[t] * np.abs(want)).all()


def test_many_threads_query_and_call(gpu):
    """Plans, workspaces and launches from many threads: nothing is kept between calls."""
    F, errors = gpu, []
    cases = [Case(r, r, n, o, FP8) for r, n, o in ((1, 5120, 130), (20, 1024, 300), (70, 4096, 200), (300, 512, 260))]
    want = [c.run(F, F32) for c in cases]
    streams = _streams(F, len(cases))

    def work(c, y, st):
        try:
            for _ in range(10):
                x, w = Mx(F, FP8, c.rows, c.n, *c.x[:2]), Mx(F, FP4, c.out, c.n, *c.w[:2])
                need, out = F.mx_matmul_workspace_bytes(w.mx, x.mx), F.DeviceBuffer(y.nbytes)
                ws = F.DeviceBuffer(max(1, need))
                F.mx_matmul_dev(w.mx, x.mx, F32, out, ws, need, stream_ptr=st)
                assert F.lib().hipStreamSynchronize(st) == 0
                assert np.array_equal(out.download(np.float32, y.shape), y)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("rows,n,out", [(1, 5120, 640), (20, 1024, 640), (50, 2080, 512), (130, 1056, 640), (300, 4096, 1280), (2100, 1824, 8192)])
def test_swiglu_codes_are_those_of_exact_sums(gpu, rows, n, out):
    """FP8 rows: but for values within fp32 sums' error of a border between two codes, the formula's codes and scales."""
    F, c, f = gpu, Repeated(rows + 5, rows, n, out, FP8), out // 2
    x, w = c.arrays(F)
    y, b = c.exact(F32)
    o = Mx(F, FP8, rows, f)
    need = F.mx_matmul_workspace_bytes(w.mx, x.mx, True)
    ws = F.DeviceBuffer(max(1, need))
    F.mx_matmul_swiglu_dev(w.mx, x.mx, o.mx, ws, need)
    F.synchronize()
    codes, s = o.read()
    val, gate = y[:, :f], y[:, f:]
    with np.errstate(over="ignore"):
        act = val * gate / (1 + np.exp(-gate))
    tol = np.abs(gate) * b[:, :f] + 1.1 * np.abs(val) * b[:, f:] + 1.1 * b[:, :f] * b[:, f:] + np.abs(act) * (8 + np.abs(gate)) * 2.0 ** -23
    lo, hi = quantize(act - tol, FP8), quantize(act + tol, FP8)
    amax, blocks = np.abs(act).reshape(rows, -1, 32), tol.reshape(rows, -1, 32)
    s_lo, s_hi = scale_bytes(np.maximum(amax - blocks, 0).max(-1), FP8), scale_bytes((amax + blocks).max(-1), FP8)
    assert ((s >= s_lo) & (s <= s_hi)).all()
    sure = np.repeat((s_lo == s_hi) & (lo[1] == s) & (hi[1] == s), 32, 1)
    got, least, most = (values(a, b, FP8) for a, b in ((codes, s), lo, hi))
    assert ((got >= least) & (got <= most))[sure].all()


@pytest.mark.parametrize("to", [FP8, FP4])
@pytest.mark.parametrize("rows", [1, 20, 50, 300])
def test_swiglu_of_fp8_rows_is_exact(gpu, rows, to):
    """Eight products of very different sizes: large ones that cancel beside small ones that are the value; what a single
    block-scaled instruction cuts off would change the codes.  The gates are 512 and more, where silu(g) is g."""
    F, n, f = gpu, 256, 128
    x = np.zeros((rows, n), np.uint8)
    x[:, ::8], x[:, 1::8], x[:, 2::8], x[:, 3::8] = 0x7E, 0x01, 0x09, 0x58     # 448, 2^-9, 1.125 * 2^-6, 16
    w = np.zeros((2 * f, n), np.uint8)
    w[:f, ::16], w[:f, 8::16] = 2, 10                                          # 1 and -1: the large ones cancel
    w[:f, 1::8], w[:f, 2::8] = 1, (np.arange(f) % 7 + 1)[:, None]
    w[f:, 3::8] = 2
    one = np.full((rows, n // 32), 127, np.uint8)
    xm, wm, o = Mx(F, FP8, rows, n, x, one), Mx(F, FP4, 2 * f, n, w, one[:1].repeat(2 * f, 0)), Mx(F, to, rows, f)
    need = F.mx_matmul_workspace_bytes(wm.mx, xm.mx, True)
    ws = F.DeviceBuffer(max(1, need))
    F.mx_matmul_swiglu_dev(wm.mx, xm.mx, o.mx, ws, need)
    F.synchronize()
    y = values(x, one, FP8) @ values(w, one[:1].repeat(2 * f, 0), FP4).T
    assert (y[:, f:] == 512).all() and (y[:, :f] < 4).all()
    got, want = o.read(), quantize(y[:, :f] * y[:, f:], to)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
