"""Paged-cache operators at the edges: weights far below the largest, pages reserved ahead, nonsensical starts, memory."""
import math

import pytest
import torch

import paged_util as P
from mojo_llm_lab_b200 import _lib, ops

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
BAD_PAGE = 1 << 8


@pytest.fixture(autouse=True)
def no_device_error():
    ops.device_error()
    yield
    torch.cuda.synchronize()
    assert ops.device_error() == 0


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


# ------------------------------------------------------------------ weights far below the largest

@pytest.mark.parametrize("hq,tokens", [(1, 1), (32, 1), (64, 1), (128, 1), (4, 64)])
@pytest.mark.parametrize("at", [0, 1000, 3999])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_key_outweighs_a_long_tail(hq, tokens, at, dtype):
    """One key 17.5 nats above 3999 others, whose values alone are not zero: each weighs less than half of fp16's
    smallest number, all of them 1e-4.  300 sequences read the same pages, so that a CTA has whole items."""
    n, page, d, seqs = 4000 + tokens - 1, 16, 64, 300
    lines = -(-n // page)
    kc, vc = torch.zeros(lines, 1, page, d, dtype=dtype), torch.ones(lines, 1, page, d, dtype=dtype)
    kc[at // page, 0, at % page, 0] = 17.5
    vc[at // page, 0, at % page] = 0.0
    q = torch.zeros(seqs * tokens, hq, d, dtype=dtype)
    q[..., 0] = 1.0
    table = torch.arange(lines, dtype=torch.int32).repeat(seqs, 1).cuda()
    more = dict(q_start=ints([tokens * i for i in range(seqs + 1)])) if tokens > 1 else {}
    out = ops.paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table, ints([n] * seqs), scale=1.0, **more)
    seen = n - tokens + 1 + torch.arange(tokens, dtype=torch.float64).repeat(seqs)
    tail = (seen - 1) * math.exp(-17.5)
    want = (tail / (1 + tail))[:, None, None]
    # Weights and result rounded once each; the scores' 25 powers of two and 2^x in fp32 (25.3 x 2^-23 + 2^-22); sums.
    # fp16: a weight's steps are 2^-24 where the largest is 2^7 or more, so each is off by 2^-32 of the largest.
    h = P.HALF[dtype]
    bound = want * (2 * h + h * h + 26.3 * 2.0 ** -23 + (n / 8 + 64) * 2.0 ** -23)
    if dtype == F16:
        bound = bound + n * 2.0 ** -32 + 2.0 ** -25
    assert ((out.double().cpu() - want).abs() <= bound).all()


# ------------------------------------------------------------------ sequences side by side

@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_sequence_does_not_depend_on_its_neighbours_queries(dtype):
    """The rows behind a sequence's last in its row tile are the next sequence's: they decide nothing.  The prefix's keys
    grow, so that scores of large queries outgrow the running maximum again and again, those of small ones hardly."""
    g = torch.Generator().manual_seed(3)
    seqs, prefix, page, hq, hk, d = 40, 1500, 16, 32, 8, 128
    news = [20, 100] * (seqs // 2)
    table, pages, _ = P.tables(news + [prefix], page, 4)
    kc, vc = P.cache(pages, hk, page, d, dtype, 4)
    for i in range(prefix):
        kc[int(table[seqs, i // page]), :, i % page] *= 0.1 + 0.9 * i / prefix
    q = (torch.randn(sum(news), hq, d, generator=g) * 2).to(dtype).cuda()
    short = torch.tensor([n == 20 for n in news]).repeat_interleave(torch.tensor(news)).cuda()
    starts = ints([0] + torch.tensor(news).cumsum(0).tolist())
    more = dict(prefix_table=table[seqs:].contiguous().cuda(), prefix_lens=ints([prefix]), q_start=starts)
    own, kc, vc = table[:seqs, :-(-100 // page)].contiguous().cuda(), kc.cuda(), vc.cuda()
    outs = []
    for factor in (1.0, 4.0, 0.0):
        other = torch.where(short[:, None, None], q, q * factor)
        outs.append(ops.paged_attention(other, kc, vc, own, ints(news), **more)[short])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ------------------------------------------------------------------ pages reserved ahead

def test_reorder_keeps_pages_reserved_ahead():
    """Columns behind the parent's rows stay the row's own, unless the row's own rows were there."""
    page, width = 16, 5
    lens = [16, 33, 64, 0]
    table = torch.arange(4 * width, dtype=torch.int32).view(4, width)
    kc, vc = P.cache(30, 1, page, 64, F16, 3)
    spare = torch.arange(20, 24, dtype=torch.int32)
    #  children of a full page, of a part-full one twice, of a longer one, of an empty one
    for parents in ([0, 0, 0, 0], [1, 1, 1, 1], [2, 2, 2, 2], [3, 3, 3, 3], [0, 1, 2, 3], [3, 2, 1, 1], [1, 0, -1, 2]):
        out, out_lens, used = (x.cpu() for x in ops.beam_reorder(ints([parents]), table.cuda(), ints(lens), spare.cuda(),
                                                                 kc.cuda(), vc.cuda()))
        for r, p in enumerate(parents):
            if p < 0:
                assert (out[r] == -1).all()
                continue
            held, mine = -(-lens[p] // page), -(-lens[r] // page)
            want = table[p, :held].tolist() + [-1] * (mine - held) + table[r, max(held, mine):].tolist()
            copied = p in parents[:r] and lens[p] % page > 0
            if copied:
                want[held - 1] = int(spare[r])
            assert out[r].tolist() == want and int(out_lens[r]) == lens[p] and int(used[r]) == copied
        live = out[[p >= 0 for p in parents]]
        behind = [int(x) for line, n in zip(live, out_lens[[p >= 0 for p in parents]]) for x in line[-(-int(n) // page):] if x >= 0]
        assert len(behind) == len(set(behind))


def test_beams_with_reserved_pages_write_apart():
    """Three beams with 16-row pages reserved ahead go on from one of them, in the middle of a page and at its end: what
    each appends afterwards is its own."""
    page, d, beams, steps = 16, 64, 3, 40
    width = -(-steps // page)
    pages = beams * width + beams * steps
    kc, vc = torch.zeros(pages, 1, page, d, dtype=F16).cuda(), torch.zeros(pages, 1, page, d, dtype=F16).cuda()
    table, lens = torch.arange(beams * width, dtype=torch.int32).view(beams, width).cuda(), ints([0] * beams)
    fresh = torch.arange(beams * width, pages, dtype=torch.int32).view(steps, beams).cuda()
    freqs = torch.zeros(1, dtype=torch.float64).cuda()  # no rotation
    history = [[] for _ in range(beams)]
    for step in range(steps):
        qkv = torch.zeros(beams, 3 * d)
        qkv[:, 2 * d:] = (step * beams + torch.arange(beams, dtype=torch.float32))[:, None] / 8
        ops.paged_qkv_append(qkv.cuda(), lens, lens, table, kc, vc, 1, freqs)
        lens = lens + 1
        history = [h + [(step * beams + i) / 8] for i, h in enumerate(history)]
        parents = {7: [1, 1, 1], 15: [1, 1, 1], 20: [2, 0, 2], 31: [2, 2, 0]}.get(step, [0, 1, 2])
        table, lens, _ = ops.beam_reorder(ints([parents]), table, lens, fresh[step], kc, vc)
        history = [history[p] for p in parents]
        for i in range(beams):
            got = vc[table[i, :-(-(step + 1) // page)].long(), 0, :, 0].flatten()[:step + 1]
            assert got.tolist() == history[i], (step, i)


# ------------------------------------------------------------------ starts that make no sense

# One call of each kind of plan: (lens, news, prefix, wide prefix table): items by number, items by CTA, more than 32
# sequences, prefixes and own rows in one pass, prefixes in a pass of their own, in one on the tensor cores.
PLANS = [([90, 200, 30], [3, 7, 5], [], False), ([90, 200, 30], [40, 170, 25], [], False),
         ([300] * 60, [100] * 60, [200], False), ([64] * 40, [2] * 40, [], False), ([90, 40, 30], [3, 2, 1], [64], True),
         ([9] * 50, [1] * 50, [64], True), ([90, 40, 30], [9, 2, 5], [64], True), ([9] * 80, [3] * 80, [640], True)]


def guarded(count, dtype, fill):
    """A tensor of `count` elements with 4096 more on both sides, and a check that those are as they were."""
    whole = torch.full((count + 8192,), fill, dtype=dtype, device="cuda")
    return whole[4096:-4096], lambda: bool((whole[:4096] == fill).all() and (whole[-4096:] == fill).all())


@pytest.mark.parametrize("lens,news,prefix,wide", PLANS)
@pytest.mark.parametrize("what", ["good", "descending", "repeating", "behind", "negative", "groups descend", "groups behind"])
def test_starts_stay_inside(lens, news, prefix, wide, what):
    hq, hk, d, page, seqs, tokens = 8, 2, 128, 16, len(lens), sum(news)
    if "groups" in what and not prefix:
        return
    table, pages, _ = P.tables(lens + prefix * 2, page, 3)
    kc, vc = (x.cuda() for x in P.cache(pages, hk, page, d, F16, 5))
    q = torch.randn(tokens, hq, d, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    starts = [0] + torch.tensor(news).cumsum(0).tolist()
    groups = [0, seqs // 2, seqs]
    if what == "descending":
        starts[1:-1] = starts[1:-1][::-1]
    elif what == "repeating":  # every second sequence has all tokens
        starts = [i % 2 * tokens for i in range(seqs + 1)]
    elif what == "behind":
        starts[-1] = 10 ** 6
    elif what == "negative":
        starts[0] = -3
    elif what == "groups descend":
        groups = [seqs, 0, seqs]
    elif what == "groups behind":
        groups[-1] = 10 ** 6
    more = dict(q_start=ints(starts))
    if prefix:
        lines = table[seqs:, :-(-prefix[0] // page)]
        if wide:  # so wide that the prefixes run once a group
            lines = torch.cat([lines, torch.full((2, 192 * 2 ** 20 // ((seqs - 2) * page * hk * d * 4) + 1), -1)], 1)
        more.update(prefix_table=lines.to(torch.int32).contiguous().cuda(), prefix_lens=ints(prefix * 2), group_start=ints(groups))
    need = ops.paged_attention_workspace(tokens, hq, hk, d, seqs, 2 if prefix else 0, "cuda").numel()
    work, work_whole = guarded(need, torch.uint8, 171)
    out, out_whole = guarded(tokens * hq * d, F16, 7.0)
    out = out.view(tokens, hq, d)
    ops.paged_attention(q, kc, vc, table[:seqs, :-(-max(lens) // page)].contiguous().cuda(), ints(lens), out=out,
                        workspace=work, **more)
    torch.cuda.synchronize()
    assert work_whole() and out_whole()
    assert ops.device_error() == (0 if what == "good" else BAD_PAGE)
    if what in ("descending", "repeating"):
        assert (out == 7.0).all()
    elif what != "groups descend":
        assert torch.isfinite(out).all() and not (out[starts[1]:] == 7.0).all(-1).any()


# ------------------------------------------------------------------ results beside their inputs

@pytest.mark.parametrize("tokens", [3, 200])
def test_out_between_the_rows_of_q(tokens):
    """q and out as interleaved views of one buffer: by token, by head, and rows one after the other."""
    lens, page, hq, hk, d = [tokens], 16, 8, 2, 128
    table, pages, _ = P.tables(lens, page, 3)
    kc, vc = (x.cuda() for x in P.cache(pages, hk, page, d, F16, 5))
    q = torch.randn(tokens, hq, d, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    args = (kc, vc, table.cuda(), ints(lens))
    want = ops.paged_attention(q, *args, q_start=ints([0, tokens]))
    for shape, at in (((tokens, 2, hq, d), 1), ((tokens, hq, 2, d), 2), ((2, tokens, hq, d), 0), ((tokens, 2, hq, d), 1)):
        buffer = torch.full(shape, 7.0, dtype=F16, device="cuda")
        mine, out = buffer.select(at, 0), buffer.select(at, 1)
        mine.copy_(q)
        assert ops.paged_attention(mine, *args, q_start=ints([0, tokens]), out=out) is out
        assert torch.equal(out, want) and torch.equal(mine, q)


def test_caches_of_one_head_with_other_strides():
    """K by rows, V by heads: with one KV head the same layout, although torch gives other strides."""
    table, pages, _ = P.tables([40, 3], 16, 6)
    kc, vc = P.cache(pages, 1, 16, 64, F16, 7)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    k = torch.empty(pages, 16, 1, 64, dtype=F16, device="cuda").transpose(1, 2)
    k.copy_(kc)
    assert k.stride() != vc.stride()
    out = ops.paged_attention(q, k, vc.cuda(), table.cuda(), ints([40, 3]))
    assert torch.equal(out, ops.paged_attention(q, kc.cuda(), vc.cuda(), table.cuda(), ints([40, 3])))


# ------------------------------------------------------------------ memory

@pytest.mark.parametrize("seqs,tokens,prefix,most", [(512, 10, 40, 44), (1024, 12, 40, 44), (512, 1, 0, 8), (64, 1, 30, 8)])
def test_attention_allocates_for_the_plan_that_it_takes(seqs, tokens, prefix, most):
    """32 query and 8 KV heads of 128: MB beside the result.  Two segments of 256 rows a CTA take 39 MB, with up to 64 rows
    a tile and two CTAs an SM 20, with 16 rows 5."""
    page, hq, hk, d = 16, 32, 8, 128
    table = torch.zeros(seqs, 2, dtype=torch.int32).cuda()
    kc, vc = (x.cuda() for x in P.cache(4, hk, page, d, F16, 5))
    q = torch.zeros(seqs * tokens, hq, d, dtype=F16, device="cuda")
    more = {}
    if prefix:
        more = dict(prefix_table=torch.zeros(1, -(-prefix // page), dtype=torch.int32).cuda(), prefix_lens=ints([prefix]))
    if tokens > 1:
        more["q_start"] = ints([tokens * i for i in range(seqs + 1)])
    lens, out = ints([20] * seqs), torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.paged_attention(q, kc, vc, table, lens, out=out, **more)
    assert torch.cuda.max_memory_allocated() - before <= most * 2 ** 20


def test_group_starts_without_groups_are_not_read():
    """The C entry with groups 0 and a group_start all the same."""
    table, pages, _ = P.tables([40, 3], 16, 6)
    kc, vc = (x.cuda() for x in P.cache(pages, 2, 16, 64, F16, 7))
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).to(F16).cuda()
    table, lens, starts = table.cuda(), ints([40, 3]), ints([10 ** 6])
    want, out = ops.paged_attention(q, kc, vc, table, lens), torch.empty_like(q)
    cache = _lib.PagedCache(kc.data_ptr(), vc.data_ptr(), pages, 2, 16, 64, *kc.stride()[:3], 1, 0, _lib.TYPE_F16)
    call = _lib.PagedAttn(q.data_ptr(), out.data_ptr(), 2, 4, 256, 64, 256, 64, table.data_ptr(), lens.data_ptr(), 2,
                          table.shape[1], None, None, starts.data_ptr(), 0, 0, None, 0.125)
    work = torch.empty(_lib.lib().mllb_paged_attention_call_workspace(call, cache), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib().mllb_paged_attention(call, cache, work.data_ptr(), work.numel(), 0,
                                               torch.cuda.current_stream().cuda_stream), "attention")
    assert torch.equal(out, want) and ops.device_error() == 0
