"""Calls of the paged-cache operators whose results would race with what other CTAs read, or whose sizes do not fit:
refused by the C entries before they touch CUDA (made-up addresses are never read)."""
import pytest

from mojo_llm_lab_b200 import _lib

EINVAL = _lib.MLLB_EINVAL


def cache(**kw):
    return _lib.PagedCache(**{**dict(k=1 << 40, v=2 << 40, pages=4, kv_heads=2, page_size=16, head_dim=128, page_stride=4096,
                                     head_stride=2048, row_stride=128, layers=1, layer_stride=0, type=_lib.TYPE_F16), **kw})


def attend(workspace_bytes=1 << 40, **kw):
    """3 tokens of 4 heads of 128: rows of 256 bytes."""
    args = _lib.PagedAttn(**{**dict(q=1 << 20, out=1 << 30, tokens=3, q_heads=4, q_token_stride=512, q_head_stride=128,
                                    out_token_stride=512, out_head_stride=128, page_table=4096, seq_lens=8192, seqs=3,
                                    table_width=2, scale=0.1), **kw})
    return _lib.lib().mllb_paged_attention(args, cache(), 1 << 41, workspace_bytes, 0, None)


@pytest.mark.parametrize("token,head", [(128, 128), (256, 128), (128, 256), (384, 128), (320, 192), (512, 160), (136, 128)])
def test_rows_of_out_over_one_another(token, head):
    assert attend(out_token_stride=token, out_head_stride=head) == EINVAL
    assert b"overlap" in _lib.lib().mllb_last_error()


@pytest.mark.parametrize("kw", [
    dict(out=(1 << 20) + 1024),                         # a token further on
    dict(out=(1 << 20) - 256),                          # a head before
    dict(out=(1 << 20) + 128),                          # half a row further on
    dict(out_token_stride=1024), dict(out_head_stride=256, out_token_stride=1024),  # its first row, then others
    dict(out_token_stride=128, out_head_stride=512),    # tokens and heads exchanged
    dict(q_token_stride=0),                             # one query for all tokens, its rows over the first result's
    dict(q_token_stride=1024, out_token_stride=1024, out=(1 << 20) + 512),  # the heads after the first two
])
def test_out_partly_over_q(kw):
    assert attend(**{**dict(out=1 << 20), **kw}) == EINVAL
    assert b"overlap" in _lib.lib().mllb_last_error()


@pytest.mark.parametrize("over", ["parents", "page_table", "seq_lens", "fresh"])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("where", ["same", "first", "last"])
def test_reorder_into_what_it_reads(over, which, where):
    """2 x 4 rows of 3 pages: lists of 32 bytes, tables of 96."""
    places = dict(parents=1 << 20, page_table=2 << 20, seq_lens=3 << 20, fresh=4 << 20)
    out, sizes = [5 << 20, 6 << 20, 7 << 20], [96, 32, 32]
    read = 96 if over == "page_table" else 32
    out[which] = places[over] + {"same": 0, "first": read - 4, "last": 4 - sizes[which]}[where]
    args = _lib.BeamRows(**places, batch=2, beams=4, table_width=3)
    assert _lib.lib().mllb_beam_reorder(args, cache(), *out, 0, None) == EINVAL
    assert b"overlap" in _lib.lib().mllb_last_error()


@pytest.mark.parametrize("which,by", [((0, 1), 0), ((0, 2), 92), ((1, 2), 28)])
def test_reorder_results_over_one_another(which, by):
    out = [5 << 20, 6 << 20, 7 << 20]
    out[which[1]] = out[which[0]] + by
    args = _lib.BeamRows(1 << 20, 2 << 20, 3 << 20, 4 << 20, 2, 4, 3)
    assert _lib.lib().mllb_beam_reorder(args, cache(), *out, 0, None) == EINVAL
    assert b"overlap" in _lib.lib().mllb_last_error()


def select(n=4, batch=3, out=(5 << 20, 6 << 20, 7 << 20), workspace=8 << 20, **kw):
    """batch entries of 4 beams: scores of 48 bytes, results of 12 n."""
    args = _lib.BeamScores(**{**dict(logits=1 << 20, batch=batch, beams=4, vocab=1000, n=n, batch_stride=4000, beam_stride=1000,
                                     scores=2 << 20, done=3 << 20, end_token=1), **kw})
    return _lib.lib().mllb_beam_select(args, *out, workspace, 1 << 20, 0, None)


@pytest.mark.parametrize("n,which,place", [
    (5, 0, 2 << 20), (3, 0, 2 << 20), (4, 0, (2 << 20) + 16), (4, 0, (2 << 20) - 44),  # one entry's results, another's scores
    (4, 1, 2 << 20), (4, 2, (2 << 20) + 44),                        # tokens and parents over scores
    (4, 0, 3 << 20), (4, 1, (3 << 20) + 8), (4, 2, (3 << 20) - 44),  # over done
    (4, 0, 8 << 20), (4, 1, (8 << 20) + 64),                        # over the workspace
    (4, 1, 5 << 20), (4, 2, (6 << 20) + 44)])                       # over one another
def test_select_into_what_it_reads(n, which, place):
    out = [5 << 20, 6 << 20, 7 << 20]
    out[which] = place
    assert select(n, out=out) == EINVAL
    assert b"overlap" in _lib.lib().mllb_last_error()


def test_sizes_whose_products_pass_64_bits():
    L = _lib.lib()
    assert L.mllb_beam_select_workspace(1 << 62, 4, 1000, 4) < 0
    assert select(batch=1 << 62, done=None) == EINVAL
    assert select(beam_stride=1 << 61) == EINVAL and select(batch_stride=1 << 61) == EINVAL
    for batch, beams in ((1 << 62, 4), (4, 1 << 62), (1 << 32, 1 << 32)):
        args = _lib.BeamRows(1 << 20, 2 << 20, 3 << 20, 4 << 20, batch, beams, 3)
        assert L.mllb_beam_reorder(args, cache(), 5 << 20, 6 << 20, 7 << 20, 0, None) == EINVAL
    assert L.mllb_paged_attention_workspace(2, 4, 2, 128, 1 << 62, 1 << 62) == _lib.MLLB_EUNSUPPORTED
    assert attend(table_width=1 << 60) == EINVAL
    assert attend(groups=1, prefix_table=4096, prefix_lens=4096, prefix_width=1 << 60) == EINVAL
    assert attend(q_token_stride=1 << 62) == EINVAL
    append = dict(qkv=1 << 20, tokens=3, positions=4096, rows=4096, page_table=4096, seqs=3, table_width=2, freqs=4096,
                  rot_dim=128, q_heads=4, eps=1e-6, magnitude=1.0, q_out=1 << 30, qkv_stride=1 << 61)
    assert L.mllb_paged_qkv_append(_lib.PagedAppend(**append), cache(), 0, None) == EINVAL


def test_call_workspace_refuses_what_the_call_refuses():
    need = _lib.lib().mllb_paged_attention_call_workspace
    assert need(None, cache()) == EINVAL and need(_lib.PagedAttn(), None) == EINVAL
    sizes = dict(tokens=3, q_heads=4, seqs=3, table_width=2)
    assert need(_lib.PagedAttn(**{**sizes, "tokens": 0}), cache()) == EINVAL
    assert need(_lib.PagedAttn(**{**sizes, "table_width": 1 << 60}), cache()) == EINVAL
    assert need(_lib.PagedAttn(**sizes), cache(head_dim=96)) == _lib.MLLB_EUNSUPPORTED


@pytest.mark.parametrize("name", ["page_table", "seq_lens", "prefix_table", "prefix_lens", "group_start", "q_start"])
def test_attention_indices_off_their_alignment(name):
    """A misaligned 4-byte load would end the context."""
    more = dict(groups=1, prefix_table=4096, prefix_lens=4096, prefix_width=2, group_start=4096, q_start=4096)
    assert attend(**{**more, name: 4098}) == _lib.MLLB_EALIGN
