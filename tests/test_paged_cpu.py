"""Refusals of the paged-cache operators and host formulas, without a GPU."""
import ctypes as C
import math

import pytest
import torch

from mojo_llm_lab_b200 import _lib, ops

F16, I32 = torch.float16, torch.int32


def caches(pages=6, heads=2, page=16, dim=128, dtype=F16):
    return torch.zeros(pages, heads, page, dim, dtype=dtype), torch.zeros(pages, heads, page, dim, dtype=dtype)


def append_args(**kw):
    k, v = caches()
    a = dict(qkv=torch.zeros(3, 8 * 128), positions=torch.zeros(3, dtype=I32), rows=torch.zeros(3, dtype=I32),
             page_table=torch.zeros(3, 2, dtype=I32), k_cache=k, v_cache=v, q_heads=4,
             freqs=torch.zeros(64, dtype=torch.float64))
    return {**a, **kw}


@pytest.mark.parametrize("kw,match", [
    ({}, "CUDA"),
    (dict(q_heads=5), "q_heads"),
    (dict(qkv=torch.zeros(3, 8 * 128, dtype=torch.float64)), "qkv"),
    (dict(qkv=torch.zeros(0, 8 * 128)), "empty"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions"),
    (dict(rows=torch.zeros(2, dtype=I32)), "rows"),
    (dict(page_table=torch.zeros(2, 2, dtype=I32)), "more tokens"),
    (dict(page_table=torch.zeros(6, dtype=I32)), "page_table"),
    (dict(page_table=torch.zeros(3, 4, dtype=I32)[:, ::2]), "page_table"),
    (dict(freqs=torch.zeros(65, dtype=torch.float64)), "freqs"),
    (dict(freqs=torch.zeros(64)), "freqs"),
    (dict(q_gamma=torch.zeros(64)), "q_gamma"),
    (dict(seq=torch.zeros(4, dtype=I32)), "seq"),
    (dict(v_cache=torch.zeros(6, 2, 16, 128, dtype=torch.bfloat16)), "v_cache"),
    (dict(v_cache=torch.zeros(6, 16, 2, 128, dtype=F16).transpose(1, 2)), "strides"),
    (dict(k_cache=torch.zeros(6, 2, 16, 128)), "k_cache"),
    (dict(q_out=torch.zeros(3, 4, 128)), "q_out"),
])
def test_append_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        ops.paged_qkv_append(**append_args(**kw))


def attention_args(**kw):
    k, v = caches()
    a = dict(q=torch.zeros(3, 4, 128, dtype=F16), k_cache=k, v_cache=v, page_table=torch.zeros(3, 2, dtype=I32),
             seq_lens=torch.zeros(3, dtype=I32))
    return {**a, **kw}


PREFIX = dict(prefix_table=torch.zeros(2, 2, dtype=I32), prefix_lens=torch.zeros(2, dtype=I32))


@pytest.mark.parametrize("kw,match", [
    ({}, "CUDA"),
    (dict(q=torch.zeros(3, 4, 64, dtype=F16)), "heads of 64"),
    (dict(q=torch.zeros(3, 5, 128, dtype=F16)), "multiple of kv_heads"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(4, 4, 128, dtype=F16)), "one token"),
    (dict(q=torch.zeros(3, 128, 4, dtype=F16).transpose(1, 2)), "contiguous"),
    (dict(seq_lens=torch.zeros(4, dtype=I32)), "seq_lens"),
    (dict(q_start=torch.zeros(3, dtype=I32)), "q_start"),
    (dict(prefix_table=torch.zeros(1, 2, dtype=I32)), "prefix_lens"),
    (dict(prefix_lens=torch.zeros(1, dtype=I32)), "prefix_table"),
    (dict(**PREFIX), "group_start"),
    (dict(**PREFIX, group_start=torch.zeros(2, dtype=I32)), "group_start"),
    (dict(out=torch.zeros(3, 4, 128)), "out"),
    (dict(out=torch.zeros(2, 4, 128, dtype=F16)), "shape"),
])
def test_attention_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        ops.paged_attention(**attention_args(**kw))


@pytest.mark.parametrize("kw,match", [
    ({}, "CUDA"),
    (dict(logits=torch.zeros(2, 3, 100, dtype=torch.float64)), "logits"),
    (dict(logits=torch.zeros(2, 300)), "dimensions"),
    (dict(scores=torch.zeros(3, 2)), "scores"),
    (dict(n=0), "positive"),
    (dict(n=301), "at most 64"),
    (dict(logits=torch.zeros(2, 3, 4), n=13), "out of range"),
    (dict(done=torch.zeros(2, 3), end_token=1), "done"),
    (dict(done=torch.zeros(2, 3, dtype=torch.bool)), "end_token"),
    (dict(done=torch.zeros(2, 3, dtype=torch.bool), end_token=100), "end_token"),
])
def test_select_refusals(kw, match):
    with pytest.raises((ValueError, _lib.MllbError), match=match):
        ops.beam_select(**{**dict(logits=torch.zeros(2, 3, 100), scores=torch.zeros(2, 3)), **kw})


@pytest.mark.parametrize("kw,match", [
    ({}, "CUDA"),
    (dict(parents=torch.zeros(6, dtype=I32)), "parents"),
    (dict(parents=torch.zeros(2, 4, dtype=I32)), "parents"),
    (dict(fresh=torch.zeros(5, dtype=I32)), "fresh"),
    (dict(seq_lens=torch.zeros(6)), "seq_lens"),
])
def test_reorder_refusals(kw, match):
    k, v = caches()
    a = dict(parents=torch.zeros(2, 3, dtype=I32), page_table=torch.zeros(6, 2, dtype=I32),
             seq_lens=torch.zeros(6, dtype=I32), fresh=torch.zeros(6, dtype=I32), k_cache=k, v_cache=v)
    with pytest.raises(ValueError, match=match):
        ops.beam_reorder(**{**a, **kw})


# The C entries refuse before they touch CUDA (made-up addresses are never read).

def c_cache(**kw):
    return _lib.PagedCache(**{**dict(k=4096, v=8192, pages=4, kv_heads=2, page_size=16, head_dim=128, page_stride=4096,
                                     head_stride=2048, row_stride=128, layers=1, layer_stride=0, type=_lib.TYPE_F16), **kw})


def c_append(**kw):
    return _lib.PagedAppend(**{**dict(qkv=4096, tokens=2, qkv_stride=1024, positions=4096, rows=4096, page_table=4096,
                                      seqs=2, table_width=2, freqs=4096, rot_dim=128, q_heads=4, eps=1e-6, magnitude=1.0,
                                      q_out=4096), **kw})


def c_attn(**kw):
    return _lib.PagedAttn(**{**dict(q=4096, out=4096, tokens=2, q_heads=4, q_token_stride=512, q_head_stride=128,
                                    out_token_stride=512, out_head_stride=128, page_table=4096, seq_lens=4096, seqs=2,
                                    table_width=2, scale=0.1), **kw})


BAD_CACHES = [(dict(k=None), _lib.MLLB_EINVAL), (dict(type=_lib.TYPE_F32), _lib.MLLB_EINVAL),
              (dict(head_dim=96), _lib.MLLB_EUNSUPPORTED), (dict(page_size=24), _lib.MLLB_EINVAL),
              (dict(page_size=8), _lib.MLLB_EINVAL), (dict(page_size=2048), _lib.MLLB_EINVAL),
              (dict(pages=0), _lib.MLLB_EINVAL), (dict(kv_heads=0), _lib.MLLB_EINVAL), (dict(k=4100), _lib.MLLB_EALIGN),
              (dict(row_stride=132), _lib.MLLB_EALIGN), (dict(row_stride=64), _lib.MLLB_EINVAL),
              (dict(page_stride=0), _lib.MLLB_EINVAL), (dict(layers=0), _lib.MLLB_EINVAL)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches(kw, code):
    L = _lib.lib()
    assert L.mllb_paged_qkv_append(c_append(), c_cache(**kw), 0, None) == code
    assert L.mllb_paged_attention(c_attn(), c_cache(**kw), 4096, 1 << 40, 0, None) == code
    rows = _lib.BeamRows(4096, 8192, 12288, 16384, 1, 4, 2)
    assert L.mllb_beam_reorder(rows, c_cache(**kw), 20480, 24576, 28672, 0, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(qkv=None), _lib.MLLB_EINVAL), (dict(rows=None), _lib.MLLB_EINVAL), (dict(tokens=0), _lib.MLLB_EINVAL),
    (dict(tokens=3), _lib.MLLB_EINVAL), (dict(rot_dim=0), _lib.MLLB_EINVAL), (dict(rot_dim=127), _lib.MLLB_EINVAL),
    (dict(rot_dim=130), _lib.MLLB_EINVAL), (dict(qkv_stride=1000), _lib.MLLB_EINVAL), (dict(qkv_stride=1026), _lib.MLLB_EALIGN),
    (dict(qkv=4104), _lib.MLLB_EALIGN), (dict(qkv_type=3), _lib.MLLB_EINVAL), (dict(eps=-1.0), _lib.MLLB_EINVAL),
    (dict(eps=math.nan), _lib.MLLB_EINVAL), (dict(q_heads=0), _lib.MLLB_EINVAL),
    (dict(q_out=4096 + 1024 * 4 + 1024 * 4 - 8), _lib.MLLB_EINVAL)])  # q_out over the end of qkv
def test_bad_appends(kw, code):
    assert _lib.lib().mllb_paged_qkv_append(c_append(**kw), c_cache(), 0, None) == code


def test_more_entries_refuse():
    L = _lib.lib()
    assert L.mllb_paged_qkv_append(c_append(), c_cache(), 8, None) == _lib.MLLB_EINVAL  # flags
    assert L.mllb_paged_qkv_append(c_append(), c_cache(layers=2, layer_stride=1 << 20), 0, None) == _lib.MLLB_EINVAL
    for kw, code in [(dict(q=None), _lib.MLLB_EINVAL), (dict(tokens=3), _lib.MLLB_EINVAL), (dict(q_heads=3), _lib.MLLB_EINVAL),
                     (dict(groups=1), _lib.MLLB_EINVAL), (dict(groups=3, prefix_table=4096, prefix_lens=4096), _lib.MLLB_EINVAL),
                     (dict(groups=2, prefix_table=4096, prefix_lens=4096, prefix_width=2), _lib.MLLB_EINVAL),
                     (dict(q_head_stride=130), _lib.MLLB_EALIGN), (dict(out_token_stride=0), _lib.MLLB_EINVAL),
                     (dict(out_head_stride=0), _lib.MLLB_EINVAL), (dict(out_head_stride=64), _lib.MLLB_EINVAL), (dict(out=4104), _lib.MLLB_EALIGN),
                     (dict(scale=math.inf), _lib.MLLB_EINVAL), (dict(scale=math.nan), _lib.MLLB_EINVAL),
                     (dict(table_width=0), _lib.MLLB_EINVAL), (dict(table_width=1 << 27), _lib.MLLB_EINVAL),
                     (dict(tokens=3000, seqs=3000), _lib.MLLB_EUNSUPPORTED)]:
        assert L.mllb_paged_attention(c_attn(**kw), c_cache(), 4096, 1 << 40, 0, None) == code, kw
    assert L.mllb_paged_attention_workspace(2, 4, 3, 128, 2, 0) == _lib.MLLB_EINVAL
    assert L.mllb_paged_attention_workspace(2, 4, 2, 80, 2, 0) == _lib.MLLB_EUNSUPPORTED
    scores = dict(logits=4096, batch=1, beams=4, vocab=1000, n=4, beam_stride=1000, scores=4096)
    for kw, code in [(dict(logits=None), _lib.MLLB_EINVAL), (dict(beams=65), _lib.MLLB_EUNSUPPORTED),
                     (dict(n=65), _lib.MLLB_EUNSUPPORTED), (dict(vocab=1 << 31), _lib.MLLB_EINVAL),
                     (dict(type=5), _lib.MLLB_EINVAL), (dict(done=4096, end_token=1000), _lib.MLLB_EINVAL),
                     (dict(logits=4098), _lib.MLLB_EALIGN), (dict(beam_stride=-1), _lib.MLLB_EINVAL),
                     (dict(batch=20000), _lib.MLLB_EINVAL)]:
        args = _lib.BeamScores(**{**scores, **kw})
        assert L.mllb_beam_select(args, 4096, 4096, 4096, 4096, 1 << 30, 0, None) == code, kw
    assert L.mllb_beam_select(_lib.BeamScores(**scores), 4096, 4096, 4096, 4096, 8, 0, None) == _lib.MLLB_EINVAL
    rows = _lib.BeamRows(4096, 8192, 12288, 16384, 1, 4, 2)
    assert L.mllb_beam_reorder(rows, c_cache(), 8192 + 28, 24576, 28672, 0, None) == _lib.MLLB_EINVAL  # over its input
    assert L.mllb_beam_reorder(rows, c_cache(), 20480, 12288, 28672, 0, None) == _lib.MLLB_EINVAL


@pytest.mark.parametrize("call", [
    lambda L: L.mllb_paged_qkv_append(None, None, 0, None),
    lambda L: L.mllb_paged_attention(None, None, None, 0, 0, None),
    lambda L: L.mllb_beam_select(None, None, None, None, None, 0, 0, None),
    lambda L: L.mllb_beam_reorder(None, None, None, None, None, 0, None),
])
def test_null_pointers(call):
    assert call(_lib.lib()) == _lib.MLLB_EINVAL
    assert b"null" in _lib.lib().mllb_last_error()


def test_rope_frequencies():
    freqs, m = ops.rope_frequencies(128, device="cpu")
    assert freqs.dtype == torch.float64 and freqs.shape == (64,) and m == 1.0
    want = torch.tensor([5e6 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64)
    assert torch.allclose(freqs, want, rtol=1e-14, atol=0)
    linear, _ = ops.rope_frequencies(128, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(linear, want / 4, rtol=1e-14, atol=0)
    # ntk: the fastest pair stays, the slowest is stretched by the factor.
    ntk, _ = ops.rope_frequencies(128, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(want[-1]) / 4, rel_tol=1e-12)
    # yarn: above 32 turns over the original context unchanged, below one turn stretched, monotone between.
    yarn, m = ops.rope_frequencies(128, scaling="yarn", factor=4.0, original_context=32768, device="cpu")
    turns = want * 32768 / (2 * math.pi)
    ratio = yarn / freqs  # of the same power function, whose last bit is not pow()'s
    assert math.isclose(m, 0.1 * math.log(4.0) + 1.0)
    assert torch.all(ratio[turns > 36] == 1.0) and torch.allclose(ratio[turns < 0.9], torch.tensor(0.25).double())
    assert torch.all(ratio[1:] <= ratio[:-1] + 1e-15)
    for kw in (dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=8, scaling="cubic"), dict(rot_dim=8, factor=0.5),
               dict(rot_dim=8, base=1.0), dict(rot_dim=2, scaling="ntk"),
               dict(rot_dim=8, scaling="yarn", fast_turns=1.0, slow_turns=2.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(device="cpu", **kw)
