"""What the packed-sequence and key/value-cache calls refuse beyond single wrong
arguments: sizes past what a launch numbers, workspaces that do not fit, outputs
that overlap, settings whose product leaves fp32's range.  All before a GPU is
looked for, all FH3_E_INVALID with a message."""
import pytest

from test_seqs_args import F, STEP, _refused, at  # noqa: F401  (F: the fixture)

SEQS = dict(d_q=at(0), d_k=at(1), d_v=at(2), d_o=at(3), n_tok=12, n_seq=3, d_first=at(4))


@pytest.mark.parametrize("heads,kv,n_tok,n_seq", [
    (8, 8, 1 << 21, 1 << 20),        # a tile to each sequence and key head, and those of full rows
    (128, 1, 1 << 23, 1),            # 2^23 tiles of full rows
    (16, 16, 1 << 24, 1 << 20),
])
def test_more_tiles_than_a_launch_numbers(F, heads, kv, n_tok, n_seq):
    cfg = F.attn_cfg(heads, kv, 64, F.FH3_QUANT_BF16)
    for first in (at(4), None):
        tiles = n_tok * (heads // kv) // 128 + n_seq if first else n_seq * -(-(n_tok // n_seq * (heads // kv)) // 128)
        if tiles * kv >= 1 << 23:
            _refused(F, F.attention_seqs_dev, cfg, {**SEQS, "n_tok": n_tok, "n_seq": n_seq, "d_first": first, "d_q": at(0), "d_k": at(200),
                                                    "d_v": at(400), "d_o": at(600)})


@pytest.mark.parametrize("n_tok,n_seq,max_pages", [(1024, 1024, 1 << 24), (1 << 20, 1, 1 << 20), (1 << 16, 1 << 16, 1 << 15)])
def test_more_pages_than_a_cache_call_counts(F, n_tok, n_seq, max_pages):
    cfg, kv = F.attn_cfg(8, 2, 64), F.kv_cache(2, 64, 4, max_pages, at(5), at(6), at(7))
    assert F.kv_attention_workspace_bytes(cfg, kv, n_tok, n_seq) == 0
    _refused(F, F.kv_attention_dev, cfg, kv, dict(d_q=at(0), d_o=at(1), n_tok=n_tok, n_seq=n_seq, d_ws=at(2), ws_bytes=STEP))


def test_workspaces_refused(F):
    """A cache long enough that tiles are divided: the workspace is needed, and looked at."""
    cfg, kv = F.attn_cfg(8, 2, 64), F.kv_cache(2, 64, 40, 30, at(5), at(6), at(7))
    need = F.kv_attention_workspace_bytes(cfg, kv, 3, 3)
    assert need > 0 and need % 16 == 0
    good = dict(d_q=at(0), d_o=at(1), n_tok=3, n_seq=3, d_ws=at(2), ws_bytes=need)
    pool, rows = F.kv_pool_bytes(2, 64, 40), 3 * 8 * 64 * 4
    for change in (dict(ws_bytes=need - 1), dict(ws_bytes=0), dict(d_ws=None), dict(d_ws=at(2, 4)), dict(d_ws=at(2, 8)),
                   dict(d_ws=at(1)), dict(d_ws=at(1, rows - 16)), dict(d_ws=at(1, 16 - need)),       # o
                   dict(d_ws=at(0)), dict(d_ws=at(0, rows - 16)), dict(d_ws=at(0, -16)),             # q
                   dict(d_ws=at(5)), dict(d_ws=at(5, pool - 16)), dict(d_ws=at(5, 16 - need))):      # the pool
        assert "workspace" in _refused(F, F.kv_attention_dev, cfg, kv, {**good, **change}), change
    for hd, heads, n in ((64, 8, 40), (128, 32, 7), (128, 2, 300)):   # few and many rows
        cfg, kv = F.attn_cfg(heads, 2, hd), F.kv_cache(2, hd, 400, 200, at(5), at(6), at(7))
        need = F.kv_attention_workspace_bytes(cfg, kv, n, 1)
        assert need > 0
        _refused(F, F.kv_attention_dev, cfg, kv, dict(d_q=at(0), d_o=at(1), n_tok=n, n_seq=1, d_ws=at(2), ws_bytes=need - 1))


def test_read_back_onto_itself(F):
    """K and V read back to rows that overlap: whichever came last would stand there."""
    kv, w = F.kv_cache(2, 64, 4, 3, at(5), at(6), at(7)), 2 * 64
    for d_v, ld in ((at(0), 0), (at(0, 16), 0), (at(0, 2 * w * 4), 0), (at(0, w * 4 - 16), 2 * w), (at(0, w * 4 + 16), 2 * w)):
        _refused(F, F.kv_read_dev, kv, 0, at(0), d_v, dict(n_tok=3, n_seq=3, ldk=ld, ldv=ld))
    _refused(F, F.kv_read_dev, kv, 0, at(0), at(0, w * 4), dict(n_tok=3, n_seq=3, ldk=2 * w, ldv=3 * w))


def test_outputs_over_what_the_call_reads(F):
    """Outputs that lie over offsets, prefixes, slopes, the page table or the lengths."""
    cfg = F.attn_cfg(8, 2, 64, d_slopes=at(8))
    rows, w = 12 * 8 * 64 * 4, 2 * 64 * 4
    for d_o in (at(4), at(4, 16 - rows), at(9), at(9, 16 - rows), at(8), at(8, 16 - rows)):
        assert "overlaps" in _refused(F, F.attention_seqs_dev, cfg, {**SEQS, "d_prefix": at(9), "d_o": d_o})
    pool = F.kv_pool_bytes(2, 64, 40)
    kv = F.kv_cache(2, 64, 40, 30, at(5), at(6), at(7))
    need = F.kv_attention_workspace_bytes(cfg, kv, 3, 3)
    good = dict(d_q=at(0), d_o=at(1), n_tok=3, n_seq=3, d_ws=at(2), ws_bytes=need, d_first=at(4))
    for i, n in ((4, 16), (6, 3 * 30 * 4), (7, 12), (8, 32)):
        end = (n - 1) // 16 * 16
        for change in (dict(d_o=at(i)), dict(d_o=at(i, end)), dict(d_ws=at(i)), dict(d_ws=at(i, end)), dict(d_ws=at(i, 16 - need))):
            assert "overlaps" in _refused(F, F.kv_attention_dev, cfg, kv, {**good, **change})
        if i == 8:
            continue
        for d_k, d_v in ((at(i), at(1)), (at(0), at(i, end)), (None, at(i)), (at(i, 16 - 3 * w), None)):
            _refused(F, F.kv_read_dev, kv, 0, d_k, d_v, dict(n_tok=3, n_seq=3, d_first=at(4)))
    for table, length, first in ((at(5), at(7), None), (at(6), at(5, pool - 16), None), (at(6), at(7), at(5, 16))):
        _refused(F, F.kv_append_dev, F.kv_cache(2, 64, 40, 30, at(5), table, length), 0, at(0), at(1), dict(n_tok=3, n_seq=3, d_first=first))
    _refused(F, F.kv_extend_dev, kv, 3, 3, at(7, 4))


@pytest.mark.parametrize("scale,softcap", [(1e-20, 1e30), (1e-44, 1e-3), (1e30, 1e-7), (1.0, 1e-44), (0.0, 1e-38)])
def test_caps_too_far_from_the_scale(F, scale, softcap):
    """scale / softcap is one fp32 factor of the product: past its range every score would be 0, or the cap."""
    cfg = F.attn_cfg(8, 2, 64, scale=scale, softcap=softcap)
    _refused(F, F.attention_seqs_dev, cfg, SEQS)
