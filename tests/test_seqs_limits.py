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
