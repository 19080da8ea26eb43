"""What the packed-sequence and key/value-cache calls refuse, before anything
reaches a GPU: every refusal is FH3_E_INVALID with a message."""
import ctypes

import numpy as np
import pytest

BASE = 0x7F0000000000    # an address that is never read: the checks come first
STEP = 1 << 34


def at(i, off=0):
    return BASE + i * STEP + off


def _refused(F, fn, *args):
    with pytest.raises(F.Fh3Error) as e:
        fn(*args[:-1], **args[-1]) if args and isinstance(args[-1], dict) else fn(*args)
    assert e.value.code == F.FH3_E_INVALID, str(e.value)
    assert len(str(e.value)) > 20
    return str(e.value)


@pytest.fixture
def F(fh3):
    return fh3


SEQS = dict(d_q=at(0), d_k=at(1), d_v=at(2), d_o=at(3), n_tok=12, n_seq=3, d_first=at(4), d_prefix=None, ldq=0, ldk=0,
            ldv=0, ldo=0)


@pytest.mark.parametrize("change", [
    dict(d_q=None), dict(d_k=None), dict(d_v=None), dict(d_o=None), dict(n_tok=0), dict(n_tok=-1), dict(n_seq=0),
    dict(n_tok=(1 << 24) + 1), dict(n_seq=(1 << 20) + 1), dict(d_first=None, n_seq=5), dict(d_first=at(4, 2)),
    dict(d_prefix=at(5, 1)), dict(d_q=at(0, 8)), dict(d_k=at(1, 4)), dict(d_v=at(2, 2)), dict(d_o=at(3, 8)),
    dict(ldq=511), dict(ldk=127), dict(ldv=-1), dict(ldo=513), dict(ldk=129), dict(ldq=1 << 40),
    dict(d_o=at(0)), dict(d_o=at(1, 256)), dict(d_o=at(2, -16)),
])
def test_attention_seqs_refusals(F, change):
    cfg = F.attn_cfg(8, 2, 64)
    _refused(F, F.attention_seqs_dev, cfg, {**SEQS, **change})


CFGS = [dict(heads=0), dict(heads=-8), dict(kv_heads=0), dict(kv_heads=3), dict(heads=258, kv_heads=2), dict(hd=96),
        dict(hd=0), dict(qtype=12), dict(qtype=8), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
        dict(softcap=-0.5), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(d_slopes=at(9, 2))]


@pytest.mark.parametrize("change", CFGS)
def test_settings_refused(F, change):
    cfg = F.attn_cfg(**{**dict(heads=8, kv_heads=2, hd=64), **change})
    _refused(F, F.attention_seqs_dev, cfg, SEQS)
    kv = F.kv_cache(cfg.kv_heads, cfg.head_dim, 4, 3, at(5), at(6), at(7))
    assert F.kv_attention_workspace_bytes(cfg, kv, 12, 3) == 0
    _refused(F, F.kv_attention_dev, cfg, kv, dict(d_q=at(0), d_o=at(1), n_tok=12, n_seq=3, d_ws=at(2), ws_bytes=STEP))


def test_settings_missing(F):
    l = F.lib()
    assert l.fh3_hip_attention_seqs_dev(None, at(0), 0, at(1), 0, at(2), 0, at(3), 0, 12, 3, None, None, None) == F.FH3_E_INVALID
    assert l.fh3_hip_kv_extend_dev(None, 1, 1, None, None) == F.FH3_E_INVALID
    assert l.fh3_hip_kv_append_dev(None, 0, at(0), 0, at(1), 0, 1, 1, None, None) == F.FH3_E_INVALID
    assert l.fh3_hip_kv_read_dev(None, 0, at(0), 0, at(1), 0, 1, 1, None, None) == F.FH3_E_INVALID
    cfg = F.attn_cfg(8, 2, 64)
    assert l.fh3_hip_kv_attention_dev(ctypes.byref(cfg), None, at(0), 0, at(1), 0, 1, 1, None, at(2), STEP, None) == F.FH3_E_INVALID
    kv = F.kv_cache(2, 64, 4, 3, at(5), at(6), at(7))
    assert l.fh3_hip_kv_attention_dev(None, ctypes.byref(kv), at(0), 0, at(1), 0, 1, 1, None, at(2), STEP, None) == F.FH3_E_INVALID
    assert l.fh3_hip_kv_attention_workspace_bytes(None, ctypes.byref(kv), 1, 1) == 0
    assert l.fh3_hip_kv_attention_workspace_bytes(ctypes.byref(cfg), None, 1, 1) == 0


CACHES = [dict(kv_heads=0), dict(kv_heads=5000), dict(hd=32), dict(pages=0), dict(pages=-1), dict(max_pages=0),
          dict(max_pages=(1 << 24) + 1), dict(d_pool=None), dict(d_pool=at(5, 8)), dict(d_table=None),
          dict(d_table=at(6, 2)), dict(d_len=None), dict(d_len=at(7, 1))]


@pytest.mark.parametrize("change", CACHES)
def test_caches_refused(F, change):
    kv = F.kv_cache(**{**dict(kv_heads=2, hd=64, pages=4, max_pages=3, d_pool=at(5), d_table=at(6), d_len=at(7)), **change})
    _refused(F, F.kv_extend_dev, kv, 3, 3)
    _refused(F, F.kv_append_dev, kv, 0, at(0), at(1), 3, 3)
    _refused(F, F.kv_read_dev, kv, 0, at(0), at(1), 3, 3)
    _refused(F, F.kv_attention_dev, F.attn_cfg(8, 2, 64), kv, at(0), at(1), 3, 3, at(2), STEP)


@pytest.mark.parametrize("change", [
    dict(qtype=12), dict(d_k=at(0, 4)), dict(d_v=at(1, 8)), dict(n_tok=0), dict(n_seq=0), dict(n_seq=2), dict(ldk=127),
    dict(ldv=130), dict(d_first=at(4, 1), n_seq=2), dict(n_tok=(1 << 24) + 3)])
def test_rows_refused(F, change):
    kv = F.kv_cache(2, 64, 4, 3, at(5), at(6), at(7))
    args = {**dict(qtype=0, d_k=at(0), d_v=at(1), n_tok=3, n_seq=3), **change}
    _refused(F, F.kv_append_dev, kv, args)
    _refused(F, F.kv_read_dev, kv, args)


def test_rows_in_the_pool_refused(F):
    kv, pool = F.kv_cache(2, 64, 4, 3, at(5), at(6), at(7)), F.kv_pool_bytes(2, 64, 4)
    for d_k, d_v in ((at(5), at(1)), (at(0), at(5)), (at(0), at(5, pool - 16)), (at(5, 16 - 3 * 128 * 4), at(1))):
        _refused(F, F.kv_append_dev, kv, 0, d_k, d_v, 3, 3)
        _refused(F, F.kv_read_dev, kv, 0, d_k, d_v, 3, 3)


def test_missing_rows_refused(F):
    kv = F.kv_cache(2, 64, 4, 3, at(5), at(6), at(7))
    _refused(F, F.kv_append_dev, kv, 0, None, at(1), 3, 3)
    _refused(F, F.kv_append_dev, kv, 0, at(0), None, 3, 3)
    _refused(F, F.kv_read_dev, kv, 0, None, None, 3, 3)


def test_attention_over_the_cache_refusals(F):
    cfg, kv = F.attn_cfg(8, 2, 64), F.kv_cache(2, 64, 4, 3, at(5), at(6), at(7))
    good = dict(d_q=at(0), d_o=at(1), n_tok=3, n_seq=3, d_ws=at(2), ws_bytes=1 << 30)
    pool = F.kv_pool_bytes(2, 64, 4)
    for change in (dict(d_q=None), dict(d_o=None), dict(d_q=at(0, 8)), dict(d_o=at(1, 4)), dict(ldq=500), dict(ldo=513),
                   dict(n_tok=4), dict(d_o=at(0)), dict(d_o=at(5)), dict(d_o=at(5, pool - 16)), dict(n_seq=-1)):
        _refused(F, F.kv_attention_dev, cfg, kv, {**good, **change})
    _refused(F, F.kv_attention_dev, cfg, F.kv_cache(1, 64, 4, 3, at(5), at(6), at(7)), good)
    _refused(F, F.kv_attention_dev, cfg, F.kv_cache(2, 128, 4, 3, at(5), at(6), at(7)), good)
    need = F.kv_attention_workspace_bytes(cfg, kv, 3, 3)
    if need:
        _refused(F, F.kv_attention_dev, cfg, kv, {**good, "ws_bytes": need - 1})
        _refused(F, F.kv_attention_dev, cfg, kv, {**good, "d_ws": None})
        _refused(F, F.kv_attention_dev, cfg, kv, {**good, "d_ws": at(2, 4)})
        _refused(F, F.kv_attention_dev, cfg, kv, {**good, "d_ws": at(1)})
        _refused(F, F.kv_attention_dev, cfg, kv, {**good, "d_ws": at(5)})


def test_pool_bytes(F):
    assert F.kv_pool_bytes(8, 128, 10) == 10 * 8 * 2 * (64 * 128 + 4)
    assert F.kv_pool_bytes(1, 64, 1) == 2 * (64 * 64 + 4)
    for bad in ((0, 64, 1), (1, 96, 1), (1, 64, 0), (-1, 64, 1), (1, 64, -5)):
        assert F.kv_pool_bytes(*bad) == 0
    assert F.kv_pool_bytes(4096, 128, 2 ** 31 - 1) == (2 ** 31 - 1) * 4096 * 2 * (64 * 128 + 4)


def test_host_model_of_the_layout():
    """The byte orders are permutations, and K's and V's 16-byte pieces are what the header says."""
    import seqs_ref as R
    for hd in (64, 128):
        for ix in (R.k_index(hd), R.v_index(hd)):
            assert np.array_equal(np.sort(ix.ravel()), np.arange(64 * hd))
        k, v = R.k_index(hd), R.v_index(hd)
        assert np.array_equal(np.diff(k[5, 16:32]), np.ones(15)) and k[0, 0] == 0
        assert [int(v[16 * t + r, 3] - v[0, 3]) for t in range(4) for r in range(4)] == list(range(16))
