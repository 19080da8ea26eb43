"""What the microscaled calls refuse, before anything reaches a GPU: every refusal is FH3_E_INVALID with a message."""
import ctypes

import pytest

from test_seqs_args import STEP, _refused, at

FP4, FP8 = 1, 2


@pytest.fixture
def F(fh3):
    return fh3


def mx(F, i, **kw):
    """An operand at places of its own: FP8 rows of 160 values, or what is said."""
    return F.mx(**{**dict(mx_type=FP8, rows=5, n=160, d_codes=at(i), d_scales=at(i, STEP // 2)), **kw})


BAD = [dict(mx_type=0), dict(mx_type=3), dict(rows=0), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(n=0), dict(n=-32), dict(n=100),
       dict(n=16), dict(n=(1 << 20) + 32), dict(d_codes=None), dict(d_codes=at(1, 8)), dict(d_scales=None), dict(d_scales=at(1, STEP // 2 + 2)),
       dict(ld=64), dict(ld=168), dict(ld=-160), dict(ld=(1 << 23) + 16), dict(ld_scales=4), dict(ld_scales=6), dict(ld_scales=-8),
       dict(ld_scales=(1 << 23) + 4)]


@pytest.mark.parametrize("change", BAD)
def test_operands_refused(F, change):
    bad, good = mx(F, 1, **change), mx(F, 2)
    w = mx(F, 3, mx_type=FP4, rows=128)
    _refused(F, F.mx_quantize_dev, 0, at(0), bad)
    _refused(F, F.mx_dequant_dev, bad, 0, at(0))
    _refused(F, F.mx_norm_dev, 0, at(0), at(4), 1e-6, bad)
    _refused(F, F.mx_matmul_dev, w, bad, 0, at(0), at(5), STEP)
    _refused(F, F.mx_matmul_swiglu_dev, w, bad, mx(F, 4, n=64), at(5), STEP)
    _refused(F, F.mx_matmul_dev, mx(F, 1, **{**dict(mx_type=FP4, rows=128), **change}), good, 0, at(0), at(5), STEP)
    if not any(k.startswith("d_") for k in change):
        assert F.mx_matmul_workspace_bytes(w, bad) == 0


def test_operands_missing(F):
    lib, none = F.lib(), ctypes.POINTER(F.Fh3Mx)()
    m, w = mx(F, 1), mx(F, 2, mx_type=FP4)
    assert lib.fh3_hip_mx_quantize_dev(0, at(0), 0, none, None) == F.FH3_E_INVALID
    assert lib.fh3_hip_mx_dequant_dev(none, 0, at(0), 0, None) == F.FH3_E_INVALID
    assert lib.fh3_hip_mx_norm_dev(0, at(0), 0, None, 0, None, 0, at(4), 1e-6, None, None, none, None) == F.FH3_E_INVALID
    assert lib.fh3_hip_mx_matmul_dev(none, m, None, None, None, 0, 0, at(0), 0, at(5), STEP, None) == F.FH3_E_INVALID
    assert lib.fh3_hip_mx_matmul_dev(w, none, None, None, None, 0, 0, at(0), 0, at(5), STEP, None) == F.FH3_E_INVALID
    assert lib.fh3_hip_mx_matmul_swiglu_dev(w, m, None, none, at(5), STEP, None) == F.FH3_E_INVALID
    assert lib.fh3_hip_mx_matmul_workspace_bytes(none, m, 0) == 0 and lib.fh3_hip_mx_matmul_workspace_bytes(w, none, 0) == 0


@pytest.mark.parametrize("change", [
    dict(qtype=12), dict(qtype=-1), dict(d_x=None), dict(d_x=at(0, 8)), dict(ldx=128), dict(ldx=161), dict(ldx=1 << 24),
    dict(d_x=at(1)), dict(d_x=at(1, 16)), dict(d_x=at(1, STEP // 2)), dict(d_x=at(1, STEP // 2 - 16))])
def test_quantize_refused(F, change):
    a = {**dict(qtype=0, d_x=at(0), y=mx(F, 1), ldx=0), **change}
    _refused(F, F.mx_quantize_dev, a)
    _refused(F, F.mx_dequant_dev, dict(x=a["y"], qtype=a["qtype"], d_y=a["d_x"], ldy=a["ldx"]))


def test_quantize_codes_over_scales_refused(F):
    _refused(F, F.mx_quantize_dev, 0, at(0), mx(F, 1, d_scales=at(1, 64)))
    _refused(F, F.mx_norm_dev, 0, at(0), at(4), 1e-6, mx(F, 1, d_scales=at(1, 64)))


NORM = dict(qtype=0, d_x=at(0), d_norm_w=at(1), eps=1e-6, d_add=at(2), d_sum=at(3), d_shift=at(4), d_scale=at(5))


@pytest.mark.parametrize("change", [
    dict(qtype=8), dict(d_x=None), dict(d_norm_w=None), dict(d_sum=None), dict(d_shift=None), dict(d_scale=None), dict(eps=-1e-6),
    dict(eps=float("nan")), dict(eps=float("inf")), dict(d_x=at(0, 4)), dict(d_norm_w=at(1, 4)), dict(d_add=at(2, 8)), dict(d_sum=at(3, 2)),
    dict(d_shift=at(4, 4)), dict(d_scale=at(5, 8)), dict(ldx=96), dict(ldadd=159), dict(ldsum=162),
    dict(d_sum=at(0, 640)), dict(d_sum=at(2, -640)), dict(d_sum=at(0), ldsum=320), dict(d_sum=at(2), ldadd=320), dict(d_sum=at(1)),
    dict(d_sum=at(4, 16)), dict(d_sum=at(5)), dict(d_x=at(6)), dict(d_add=at(6, 640)), dict(d_sum=at(6)), dict(d_norm_w=at(6)),
    dict(d_shift=at(6)), dict(d_scale=at(6, STEP // 2))])
def test_norm_refused(F, change):
    _refused(F, F.mx_norm_dev, {**NORM, **change, "y": mx(F, 6)})


def test_norm_long_rows_refused(F):
    _refused(F, F.mx_norm_dev, {**NORM, "y": mx(F, 6, n=32800)})


PRODUCT = dict(qtype=0, d_y=at(0), d_ws=at(1), ws_bytes=STEP, d_bias=at(2), d_gate=at(3), d_res=at(4), ldres=0, ldy=0)


@pytest.mark.parametrize("change", [
    dict(qtype=12), dict(d_y=None), dict(d_y=at(0, 2)), dict(d_bias=at(2, 2)), dict(d_gate=at(3, 1)), dict(d_res=at(4, 2)),
    dict(d_res=None), dict(ldy=127), dict(ldy=-128), dict(ldres=100), dict(ldy=(1 << 25) + 1), dict(ldres=(1 << 25) + 1),
    dict(d_y=at(5)), dict(d_y=at(6, STEP // 2)), dict(d_y=at(2)), dict(d_y=at(3, 16)), dict(d_y=at(4, 4)), dict(d_y=at(4), ldy=256)])
def test_product_refused(F, change):
    _refused(F, F.mx_matmul_dev, mx(F, 5, mx_type=FP4, rows=128), mx(F, 6), {**PRODUCT, **change})


def test_product_shapes_refused(F):
    w, x = mx(F, 5, mx_type=FP4, rows=128), mx(F, 6)
    for a, b in ((mx(F, 5, rows=128), x), (w, mx(F, 6, n=192)), (mx(F, 5, mx_type=FP4, rows=1 << 24), mx(F, 6, rows=1 << 24))):
        assert F.mx_matmul_workspace_bytes(a, b) == 0
        _refused(F, F.mx_matmul_dev, a, b, PRODUCT)
    for rows in (64, 96, 130):
        bad = mx(F, 5, mx_type=FP4, rows=rows)
        assert F.mx_matmul_workspace_bytes(bad, x, True) == 0
        _refused(F, F.mx_matmul_swiglu_dev, bad, x, mx(F, 7, n=32), at(1), STEP)
    for y in (mx(F, 7, n=128), mx(F, 7, n=64, rows=4), mx(F, 5, n=64), mx(F, 6, n=64), mx(F, 7, n=64, d_scales=at(7, 32)),
              mx(F, 2, n=64), mx(F, 7, n=64, d_scales=at(6))):
        _refused(F, F.mx_matmul_swiglu_dev, w, x, y, at(1), STEP, at(2))


def _with_workspace(F):
    """A product that needs one, its operands, its size."""
    for rows in (100, 300, 1000):
        w, x = mx(F, 5, mx_type=FP4, rows=256, n=8192), mx(F, 6, rows=rows, n=8192)
        need = F.mx_matmul_workspace_bytes(w, x)
        if need:
            return w, x, need
    raise AssertionError("none of the sizes needs a workspace")


@pytest.mark.parametrize("change", [dict(d_ws=None), dict(d_ws=at(1, 8)), dict(ws_bytes=0), dict(ws_bytes=-1), dict(d_ws=at(0, -16)),
                                    dict(d_ws=at(2, -64)), dict(d_ws=at(3)), dict(d_ws=at(4, -16)), dict(d_ws=at(5)),
                                    dict(d_ws=at(5, STEP // 2)), dict(d_ws=at(6)), dict(d_ws=at(6, STEP // 2 - 16))])
def test_workspaces_refused(F, change):
    w, x, need = _with_workspace(F)
    if change.get("ws_bytes") == -1:
        change = dict(ws_bytes=need - 1)
    _refused(F, F.mx_matmul_dev, w, x, {**PRODUCT, "ws_bytes": need, **change})
