"""Paged-cache operators on the GPU against plain fp64 forms (paged_util.py)."""
import math

import pytest
import torch

import paged_util as P
from mojo_llm_lab_b200 import _lib, ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
BAD_PAGE, BAD_PARENT = 1 << 8, 1 << 9


@pytest.fixture(autouse=True)
def no_device_error():
    ops.device_error()
    yield
    torch.cuda.synchronize()
    assert ops.device_error() == 0


def within(got, ref, bound, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} of {over.numel()} off, worst by {float(over.max()):.3e}"


# ------------------------------------------------------------------ append

def append_case(tokens, hq, hk, d, rot, src, dst, page, interleaved, norm, seed, per_seq=1, rows_first=False, base=0,
                scaling="none"):
    g = torch.Generator().manual_seed(seed)
    seqs = -(-tokens // per_seq)
    held = [(7 * i) % 50 for i in range(seqs)]
    table, pages, _ = P.tables([h + per_seq for h in held], page, seed)
    kc, vc = P.cache(pages, hk, page, d, dst, seed, rows_first)
    qkv = (torch.randn(tokens, (hq + 2 * hk) * d, generator=g) * 2).to(src)
    seq = (torch.arange(tokens) // per_seq).to(torch.int32)
    rows = (torch.tensor(held)[seq.long()] + torch.arange(tokens) % per_seq).to(torch.int32)
    gammas = [0.5 + torch.rand(d, generator=g) if norm else None for _ in range(2)]
    freqs, magnitude = ops.rope_frequencies(rot, scaling=scaling, factor=4.0 if scaling != "none" else 1.0, device="cpu")
    return dict(qkv=qkv, positions=(rows + base).to(torch.int32), rows=rows, seq=seq, table=table, kc=kc, vc=vc, hq=hq,
                freqs=freqs, q_gamma=gammas[0], k_gamma=gammas[1], interleaved=interleaved, magnitude=magnitude)


def run_append(c, seq=True, **kw):
    dev = {k: P.to_dev(v) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q = ops.paged_qkv_append(dev["qkv"], dev["positions"], dev["rows"], dev["table"], dev["kc"], dev["vc"], c["hq"],
                             dev["freqs"], seq=dev["seq"] if seq else None, q_gamma=dev["q_gamma"], k_gamma=dev["k_gamma"],
                             interleaved=c["interleaved"], magnitude=c["magnitude"], **kw)
    return q, dev["kc"], dev["vc"]


def check_append(c, q, kc, vc):
    ref_q, ref_k, ref_v, bound_q, bound_k = P.append(c["qkv"], c["positions"], c["rows"], c["seq"], c["table"], c["kc"],
                                                     c["vc"], c["hq"], c["freqs"], c["q_gamma"], c["k_gamma"],
                                                     c["interleaved"], c["magnitude"])
    live = c["rows"] >= 0
    within(q.cpu()[live], ref_q[live], bound_q[live], "q")
    page = c["kc"].shape[2]
    kc, vc = kc.cpu(), vc.cpu()
    want_k, want_v = c["kc"].clone(), c["vc"].clone()
    for t in torch.nonzero(live)[:, 0].tolist():
        r = int(c["rows"][t])
        slot = int(c["table"][int(c["seq"][t]), r // page])
        within(kc[slot, :, r % page], ref_k[t], bound_k[t], "k")
        want_k[slot, :, r % page] = kc[slot, :, r % page]
        want_v[slot, :, r % page] = ref_v[t].to(vc.dtype)
    assert torch.equal(kc, want_k), "K rows that no token names changed"
    assert torch.equal(vc, want_v), "V: one rounding of the input, and no other row"


@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (128, 2, True),
                                               (128, 50, False), (128, 50, True), (64, 64, False), (64, 16, True),
                                               (64, 22, False)])
@pytest.mark.parametrize("src,dst", [(F32, F16), (BF16, BF16), (F16, BF16)])
def test_append_layouts(d, rot, interleaved, src, dst):
    c = append_case(5, 6, 2, d, rot, src, dst, 16, interleaved, True, seed=d + rot, base=1000)
    check_append(c, *run_append(c, seq=False))


@pytest.mark.parametrize("tokens,hq,hk,norm,per_seq,page,rows_first", [
    (1, 32, 8, True, 1, 16, False), (1, 1, 1, False, 1, 16, True), (97, 32, 8, True, 40, 32, True),
    (300, 3, 1, False, 100, 128, False), (700, 5, 5, True, 350, 16, False)])
def test_append_sizes(tokens, hq, hk, norm, per_seq, page, rows_first):
    c = append_case(tokens, hq, hk, 128, 128, F32, F16, page, False, norm, seed=tokens, per_seq=per_seq,
                    rows_first=rows_first)
    check_append(c, *run_append(c))


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_append_far_positions(scaling):
    c = append_case(3, 4, 1, 64, 64, F32, F16, 16, False, False, seed=9, base=2_000_000_000, scaling=scaling)
    check_append(c, *run_append(c))


def test_append_only_one_gamma_and_zero_rows():
    c = append_case(2, 2, 1, 64, 64, F32, BF16, 16, False, True, seed=4)
    c["q_gamma"] = None
    c["qkv"][1] = 0.0  # a norm of nothing: 0 / sqrt(eps)
    check_append(c, *run_append(c))


def test_append_padding_and_strided_input():
    c = append_case(6, 4, 2, 128, 128, F32, F16, 16, True, True, seed=11)
    c["rows"][2] = -1
    c["rows"][5] = -7
    wide = torch.full((6, c["qkv"].shape[1] + 64), math.nan)
    wide[:, 32:-32] = c["qkv"]
    q_out = torch.full((6, 4, 128), 7.0, dtype=F16, device="cuda")
    dev = wide.cuda()[:, 32:-32]
    kc, vc = P.to_dev(c["kc"]), P.to_dev(c["vc"])
    got = ops.paged_qkv_append(dev, c["positions"].cuda(), c["rows"].cuda(), c["table"].cuda(), kc, vc, 4,
                               c["freqs"].cuda(), q_gamma=c["q_gamma"].cuda(), k_gamma=c["k_gamma"].cuda(),
                               interleaved=True, q_out=q_out)
    assert got is q_out
    check_append(c, q_out, kc, vc)
    assert (q_out[[2, 5]] == 7.0).all()


def test_append_rows_without_a_page_store_nothing():
    c = append_case(5, 4, 2, 128, 128, F32, F16, 16, False, True, seed=12)
    for t, bad in ((0, -1), (1, c["kc"].shape[0]), (2, 2 ** 31 - 1)):
        c["table"][t] = bad
    c["rows"][3] = 16 * c["table"].shape[1]  # behind the table
    c["seq"][4] = 5  # no such sequence
    kc0, vc0 = c["kc"].clone(), c["vc"].clone()
    q, kc, vc = run_append(c)
    assert torch.equal(kc.cpu(), kc0) and torch.equal(vc.cpu(), vc0)
    assert torch.isfinite(q).all()
    assert ops.device_error() == BAD_PAGE


# ------------------------------------------------------------------ attention

def attention_case(lens, news=None, prefix=(), group_start=None, hq=8, hk=2, d=128, page=16, dtype=F16, seed=0,
                   rows_first=False, spread=2.0, apart=True):
    """apart: the prefixes' table is so wide (behind its pages stand numbers that are never read) that prefixes run
    once a group; else a call of this size has every sequence read its prefix again."""
    g = torch.Generator().manual_seed(seed)
    news = [1] * len(lens) if news is None else news
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    table, pages, _ = P.tables(list(lens) + list(prefix), page, seed, behind=2 ** 31 - 1)
    kc, vc = P.cache(pages, hk, page, d, dtype, seed, rows_first)
    for i, n in enumerate(list(lens) + list(prefix)):
        if n % page:
            kc[int(table[i, n // page]), :, n % page:] = math.nan
            vc[int(table[i, n // page]), :, n % page:] = math.nan
    q = (torch.randn(starts[-1], hq, d, generator=g) * spread).to(dtype)
    b = len(lens)
    width = max(1, -(-max(lens) // page))
    c = dict(q=q, kc=kc, vc=vc, table=table[:b, :width].contiguous(), lens=list(lens), starts=starts,
             one=all(n == 1 for n in news))
    if prefix:
        c["prefix_table"] = table[b:, :max(1, -(-max(prefix) // page))].contiguous()
        c["prefix_lens"] = list(prefix)
        c["group_start"] = [0, b] if group_start is None else group_start
        if apart and b > len(prefix):
            columns = 192 * 2 ** 20 // ((b - len(prefix)) * page * hk * d * 4) + 1
            wide = torch.full((len(prefix), max(columns, c["prefix_table"].shape[1])), 2 ** 31 - 1, dtype=torch.int32)
            wide[:, :c["prefix_table"].shape[1]] = c["prefix_table"]
            c["prefix_table"] = wide
    return c


def run_attention(c, **kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    more = {}
    if "prefix_table" in c:
        more = dict(prefix_table=c["prefix_table"].cuda(), prefix_lens=i32(c["prefix_lens"]), group_start=i32(c["group_start"]))
    if not c["one"]:
        more["q_start"] = i32(c["starts"])
    return ops.paged_attention(kw.pop("q", None) if "q" in kw else c["q"].cuda(), P.to_dev(c["kc"]), P.to_dev(c["vc"]),
                               c["table"].cuda(), i32(c["lens"]), **more, **kw)


def check_attention(c, out, scale=None):
    ref, bound = P.attention(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], c.get("prefix_table"),
                             c.get("prefix_lens"), c.get("group_start"), scale)
    within(out, ref, bound)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 128, 1000, 5001])
@pytest.mark.parametrize("hq,hk,d,page,dtype", [(8, 2, 128, 16, F16), (3, 3, 64, 64, BF16)])
def test_attention_lengths(n, hq, hk, d, page, dtype):
    c = attention_case([n], hq=hq, hk=hk, d=d, page=page, dtype=dtype, seed=n)
    check_attention(c, run_attention(c))


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 1), (16, 1), (17, 1), (40, 1), (64, 1), (65, 1), (200, 2), (32, 8), (21, 7)])
def test_attention_heads(hq, hk):
    c = attention_case([130, 0, 77], hq=hq, hk=hk, seed=hq)
    check_attention(c, run_attention(c))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("rows_first", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_pages(page, rows_first, d):
    c = attention_case([page + 5, 3 * page, 1], prefix=[2 * page + 1], page=page, d=d, rows_first=rows_first, seed=page,
                       dtype=BF16)
    check_attention(c, run_attention(c))


@pytest.mark.parametrize("seqs,prefix,group_start,hq,hk", [
    (2, [100], None, 4, 1), (5, [1019], None, 16, 4), (20, [300], None, 8, 2), (40, [2000], None, 8, 2),
    (80, [513], None, 8, 2), (33, [700, 65], [0, 30, 33], 8, 2), (9, [64, 0, 128], [0, 4, 6, 9], 4, 2),
    (12, [200, 90], [2, 5, 9], 4, 1), (7, [50, 60, 70], [0, 3, 3, 7], 4, 1), (3, [40, 50, 60], [0, 1, 2, 3], 4, 2),
    (150, [1025], None, 10, 2)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("apart", [True, False])
def test_attention_shared_prefixes(seqs, prefix, group_start, hq, hk, dtype, apart):
    lens = [(37 * i) % 150 for i in range(seqs)]
    c = attention_case(lens, prefix=prefix, group_start=group_start, hq=hq, hk=hk, seed=seqs, dtype=dtype, apart=apart)
    check_attention(c, run_attention(c))


@pytest.mark.parametrize("lens,news,prefix,hq,hk,d", [
    ([5], [5], [], 4, 2, 128), ([200], [200], [], 4, 1, 128), ([333], [100], [], 8, 2, 64),
    ([70, 300, 9], [70, 129, 9], [], 4, 2, 128), ([70, 300, 9], [3, 129, 0], [], 4, 2, 64),
    ([4, 0, 6], [9, 3, 6], [], 4, 2, 128),          # more tokens than rows: the first see nothing
    ([4, 0, 6], [9, 3, 6], [33], 4, 2, 128),        # ... or the prefix alone
    ([200, 150, 90], [64, 2, 90], [500], 8, 2, 128), ([600, 550], [600, 400], [333], 8, 2, 128),
    ([64, 64, 64, 64], [4, 4, 3, 2], [1000], 8, 2, 128),
    ([100, 90, 60], [12, 9, 11], [], 8, 2, 128), ([600, 511, 30], [12, 9, 11], [], 8, 2, 64),  # short, long tables
    ([600, 511, 30], [12, 9, 11], [70], 8, 2, 128),
    (list(range(70, 110)), list(range(70, 110)), [], 8, 2, 64),  # items of one or two tiles: shares start anywhere in them
    ([130] * 30, [100 + i % 7 for i in range(30)], [65], 4, 1, 128), ([1500], [1500], [], 4, 2, 64), ([1100], [1030], [129], 2, 1, 64)])
@pytest.mark.parametrize("dtype,apart", [(F16, True), (BF16, True), (F16, False)])
def test_attention_many_tokens(lens, news, prefix, hq, hk, d, dtype, apart):
    c = attention_case(lens, news, prefix, hq=hq, hk=hk, d=d, dtype=dtype, seed=sum(lens), apart=apart)
    check_attention(c, run_attention(c))


def test_attention_empty_rows_are_zero():
    c = attention_case([0, 0, 40], seed=3)
    c["table"] = c["table"].clone()
    out = torch.full((3, 8, 128), math.nan, dtype=F16, device="cuda")
    assert run_attention(c, out=out) is out
    assert (out[:2] == 0).all()
    check_attention(c, out)


def test_attention_all_empty():
    c = attention_case([0, 0], prefix=[0], seed=3)
    assert (run_attention(c) == 0).all()


@pytest.mark.parametrize("prefix", [[], [90]])
def test_attention_strides_and_rows_behind_the_last_token(prefix):
    c = attention_case([90, 200], [3, 70], prefix, seed=21)
    n = c["q"].shape[0]
    wide = torch.zeros(n + 9, 3, 8, 128, dtype=F16)
    wide[:n, 1] = c["q"]
    wide[n:] = math.nan
    q = wide.cuda()[:, 1]
    buffer = torch.full((n + 9, 8, 2, 128), 7.0, dtype=F16, device="cuda")
    out = buffer[:, :, 0]
    run_attention(c, q=q, out=out)
    check_attention(c, out[:n])
    assert (out[n:] == 7.0).all() and (buffer[:, :, 1] == 7.0).all()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 1e-20])
def test_attention_scales(scale):
    c = attention_case([70, 300], prefix=[100], spread=0.3, seed=5)
    check_attention(c, run_attention(c, scale=scale), scale)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 1e-20])
@pytest.mark.parametrize("hq", [8, 6])
def test_attention_scales_of_many_tokens(scale, hq):
    c = attention_case([300, 170], [200, 170], [100], hq=hq, spread=0.3, seed=5)
    check_attention(c, run_attention(c, scale=scale), scale)


def test_attention_rising_scores():
    """Scores that grow from tile to tile, so that the running maximum has to move again and again; and huge ones."""
    for grow in (0.02, 0.4):
        c = attention_case([700], [120], [650], hq=4, hk=2, spread=1.0, seed=3)
        c["q"] = c["q"].abs()
        for lens, table in ((650, c["prefix_table"][0]), (700, c["table"][0])):
            for at in range(lens):
                c["kc"][int(table[at // 16]), :, at % 16] = (at if lens == 650 else 650 + at) * grow / 128
        check_attention(c, run_attention(c))


def test_attention_peaked_scores():
    """One key outweighs all others by far, early or late: the running maximum's corrections."""
    for at in (0, 63, 64, 500, 999):
        c = attention_case([1000], spread=1.0, seed=at)
        slot = int(c["table"][0, at // 16])
        c["kc"][slot, :, at % 16] = 20.0 * torch.sign(c["q"][0, ::4].float()).to(F16)
        check_attention(c, run_attention(c))


@pytest.mark.parametrize("apart", [True, False])
def test_attention_bad_pages_are_flagged_and_stay_inside(apart):
    c = attention_case([200, 100, 64], prefix=[80], seed=8, apart=apart)
    good = run_attention(c).cpu()
    c["table"][0, 3], c["table"][0, 5] = -5, c["kc"].shape[0]
    out = run_attention(c)
    assert torch.isfinite(out).all() and torch.equal(out.cpu()[1:], good[1:])
    assert ops.device_error() == BAD_PAGE
    # Lengths outside the table count as its ends.
    c = attention_case([208, 100], seed=8)
    good = run_attention(c).cpu()
    c["lens"] = [10 ** 6, -4]
    out = run_attention(c).cpu()
    assert torch.equal(out[0], good[0]) and (out[1] == 0).all()
    assert ops.device_error() == BAD_PAGE


@pytest.mark.parametrize("apart", [True, False])
def test_attention_starts_that_make_no_sense_stay_inside(apart):
    c = attention_case([90, 200, 30], [3, 70, 5], [64], seed=22, apart=apart)
    c["starts"] = [0, 10 ** 6, -3, 78]
    c["group_start"] = [7, -2]
    run_attention(c)
    torch.cuda.synchronize()
    ops.device_error()


def test_attention_offsets_past_32_bits():
    """A cache of more than 2^31 elements, with the sequence's pages at its far end."""
    page, hk, d = 128, 8, 128
    pages = 2 ** 31 // (page * hk * d) + 40
    kc = torch.zeros(pages, hk, page, d, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    c = attention_case([300, 170], prefix=[140], hq=16, hk=hk, page=page, dtype=BF16, seed=6)
    shift = pages - c["kc"].shape[0]
    kc[shift:], vc[shift:] = c["kc"].cuda(), c["vc"].cuda()
    far = {k: torch.where(c[k] < 2 ** 30, c[k] + shift, c[k]).cuda() for k in ("table", "prefix_table")}
    lens, plens = torch.tensor(c["lens"], dtype=torch.int32).cuda(), torch.tensor([140], dtype=torch.int32).cuda()
    out = ops.paged_attention(c["q"].cuda(), kc, vc, far["table"], lens, far["prefix_table"], plens)
    check_attention(c, out)
    # The append writes there too.
    a = append_case(2, 16, hk, d, 128, BF16, BF16, page, False, True, seed=2)
    at = a["table"] + (pages - a["kc"].shape[0])
    ops.paged_qkv_append(a["qkv"].cuda(), a["positions"].cuda(), a["rows"].cuda(), at.cuda(), kc, vc, 16,
                         a["freqs"].cuda(), q_gamma=a["q_gamma"].cuda(), k_gamma=a["k_gamma"].cuda())
    tail = kc[int(at[0, 0]), :, int(a["rows"][0])].cpu()
    ref = P.append(a["qkv"], a["positions"], a["rows"], a["seq"], a["table"], a["kc"], a["vc"], 16, a["freqs"],
                   a["q_gamma"], a["k_gamma"], False, 1.0)
    within(tail, ref[1][0], ref[4][0])


def test_attention_on_another_stream_and_twice_at_once():
    """Calls on two streams at the same time, each with its own workspace."""
    a, b = attention_case([700, 90], prefix=[300], seed=1), attention_case([400, 1000, 3], seed=2)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for c, s in zip((a, b), streams):
        with torch.cuda.stream(s):
            outs.append(run_attention(c))
    torch.cuda.synchronize()
    check_attention(a, outs[0])
    check_attention(b, outs[1])


@pytest.mark.parametrize("prefix,apart", [([], False), ([150], False), ([150], True)])
def test_captured_attention_follows_lengths(prefix, apart):
    """One captured launch, replayed while the lengths grow across tiles and pages."""
    c = attention_case([200, 180, 140], prefix=prefix, seed=31, apart=apart)
    q, kc, vc, table = c["q"].cuda(), P.to_dev(c["kc"].nan_to_num()), P.to_dev(c["vc"].nan_to_num()), c["table"].cuda()
    c["kc"], c["vc"] = kc.cpu(), vc.cpu()
    lens = torch.tensor([1, 1, 1], dtype=torch.int32).cuda()
    more = {}
    if prefix:
        more = dict(prefix_table=c["prefix_table"].cuda(), prefix_lens=torch.tensor(prefix, dtype=torch.int32).cuda())
    work = ops.paged_attention_workspace(3, 8, 2, 128, 3, len(prefix), "cuda")
    out = torch.empty_like(q)
    ops.paged_attention(q, kc, vc, table, lens, out=out, workspace=work, **more)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, kc, vc, table, lens, out=out, workspace=work, **more)
    for now in ([1, 1, 1], [0, 64, 65], [16, 17, 128], [200, 180, 140], [33, 0, 0]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        work.fill_(255)  # a workspace holds nothing between calls
        graph.replay()
        torch.cuda.synchronize()
        c["lens"] = now
        check_attention(c, out)


@pytest.mark.parametrize("lens,news,prefix", [
    ([700, 90, 1], None, []), ([300, 170], [200, 170], [100]), ([64] * 9, None, [500]), ([30] * 70, None, [300])])
def test_attention_into_its_queries(lens, news, prefix):
    c = attention_case(lens, news, prefix, seed=17)
    want = run_attention(c)
    q = c["q"].cuda()
    assert run_attention(c, q=q, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("news", [3, 200])
def test_attention_of_one_query_for_all_tokens(news):
    """q with stride 0 over the tokens."""
    c = attention_case([300], [news], seed=18)
    one = c["q"][:1].cuda()
    out = run_attention(c, q=one.expand(news, -1, -1))
    c["q"] = c["q"][:1].expand(news, -1, -1).contiguous()
    check_attention(c, out)


def test_attention_most_sequences():
    """2047 sequences and their one prefix, as one softmax and apart; one more is refused."""
    lens = [i % 19 for i in range(2047)]
    for apart in (False, True):
        c = attention_case(lens, prefix=[33], hq=2, hk=1, d=64, seed=19, apart=apart)
        check_attention(c, run_attention(c))
    c = attention_case(lens + [3], prefix=[33], hq=2, hk=1, d=64, seed=19, apart=False)
    with pytest.raises(_lib.MllbError, match="2048"):
        run_attention(c)


# ------------------------------------------------------------------ reorder

@pytest.mark.parametrize("batch,beams,layers,heads,page,d,dtype,rows_first", [
    (1, 4, 1, 2, 16, 128, F16, False), (3, 8, 3, 1, 32, 64, BF16, True), (2, 1, 2, 2, 16, 64, F16, False),
    (5, 3, None, 8, 64, 128, BF16, False), (1, 40, 2, 3, 16, 128, F16, True)])
def test_reorder(batch, beams, layers, heads, page, d, dtype, rows_first):
    g = torch.Generator().manual_seed(batch * beams)
    r = batch * beams
    lens = torch.tensor([(5 * page // 2 + 3 * b) if b else 2 * page for b in range(batch)]).repeat_interleave(beams).to(torch.int32)
    lens[0] = 1  # beams of an entry need not be of one length
    table, pages, spare = P.tables(lens.tolist(), page, 1, spare=r)
    kc, vc = P.cache(pages, heads, page, d, dtype, 3, rows_first, layers)
    parents = torch.randint(0, beams, (batch, beams), generator=g).to(torch.int32)
    kd, vd = P.to_dev(kc), P.to_dev(vc)
    got = ops.beam_reorder(parents.cuda(), table.cuda(), lens.cuda(), spare.cuda(), kd, vd)
    want = P.reorder(parents, table, lens, spare, [kc, vc], page)
    for x, y in zip(got, want[:3]):
        assert torch.equal(x.cpu(), y)
    assert torch.equal(kd.cpu(), want[3][0]) and torch.equal(vd.cpu(), want[3][1])


def test_reorder_rows_that_end_and_bad_parents():
    lens = torch.tensor([20, 20, 20, 20], dtype=torch.int32)
    table, pages, spare = P.tables(lens.tolist(), 16, 1, spare=4)
    kc, vc = P.cache(pages, 2, 16, 64, F16, 3)
    kd, vd = kc.cuda(), vc.cuda()
    parents = torch.tensor([[1, -1, 1, 4]], dtype=torch.int32)
    got = ops.beam_reorder(parents.cuda(), table.cuda(), lens.cuda(), spare.cuda(), kd, vd)
    want = P.reorder(parents, table, lens, spare, [kc, vc], 16)
    for x, y in zip(got, want[:3]):
        assert torch.equal(x.cpu(), y)
    assert torch.equal(kd.cpu(), want[3][0])
    assert ops.device_error() == BAD_PARENT
    # A fresh page outside the cache, a length outside the table: flagged, and nothing is copied.
    bad = spare.clone()
    bad[2] = pages
    before = kd.clone()
    table_out, _, used = ops.beam_reorder(parents.clamp(0, 3).cuda(), table.cuda(), lens.cuda(), bad.cuda(), kd, vd)
    assert int(used[2]) == 0 and torch.equal(kd, before) and torch.equal(table_out[2].cpu(), table[1])
    assert ops.device_error() == BAD_PAGE
    ops.beam_reorder(torch.zeros(1, 4, dtype=torch.int32).cuda(), table.cuda(), (lens + 100).cuda(), spare.cuda(), kd, vd)
    assert torch.equal(kd, before)
    assert ops.device_error() == BAD_PAGE


# ------------------------------------------------------------------ a run of them

def test_beam_decoding_steps():
    """Beams of two prompts for 40 steps, as a decode loop runs them: append, attention over the shared prompt and the
    beams' own pages, selection, reordering; against each beam's whole history, kept flat, in fp64."""
    torch.manual_seed(5)
    g = torch.Generator().manual_seed(5)
    batch, beams, hq, hk, d, page, vocab, steps = 2, 3, 4, 2, 64, 16, 500, 40
    prompt, r = [37, 64], 6
    freqs, _ = ops.rope_frequencies(d, device="cpu")
    width = -(-steps // page)
    prefix_table, used_pages, _ = P.tables(prompt, page, 2, spare=0)
    pages = used_pages + 3 * r * (width + 1)
    kc, vc = P.cache(pages, hk, page, d, F16, 5)
    history = [(P.rows_of(kc, prefix_table[b], prompt[b]), P.rows_of(vc, prefix_table[b], prompt[b])) for b in range(batch)
               for _ in range(beams)]
    embed = torch.randn(vocab, (hq + 2 * hk) * d, generator=g) * 1.5
    head = torch.randn(hq * d, vocab, generator=g) * 0.4
    kd, vd, ed, hd = kc.cuda(), vc.cuda(), embed.cuda(), head.cuda()
    plens = torch.tensor(prompt, dtype=torch.int32).cuda()
    group_start = torch.tensor([0, beams, r], dtype=torch.int32).cuda()
    free = list(range(used_pages, pages))
    table = torch.full((r, width), -1, dtype=torch.int32)
    tokens = torch.arange(r)
    scores = torch.tensor([[0.0] + [-math.inf] * (beams - 1)] * batch).cuda()
    lens = torch.zeros(r, dtype=torch.int32)
    for step in range(steps):
        if step % page == 0:
            for i in range(r):
                table[i, step // page] = free.pop()
        pos = torch.tensor([prompt[i // beams] + step for i in range(r)], dtype=torch.int32)
        x = embed[tokens]
        q = ops.paged_qkv_append(ed[tokens.cuda()], pos.cuda(), lens.cuda(), table.cuda(), kd, vd, hq, freqs.cuda())
        lens = lens + 1
        out = ops.paged_attention(q, kd, vd, table.cuda(), lens.cuda(), prefix_table.cuda(), plens, group_start)
        _, rk, rv, _, _ = P.append(x, pos, lens, None, table, kc, vc, hq, freqs, None, None, False, 1.0)
        ref = torch.zeros(r, hq, d, dtype=torch.float64)
        for i in range(r):
            k = torch.cat([history[i][0], rk[i][:, None].half().double()], 1)
            v = torch.cat([history[i][1], rv[i][:, None].half().double()], 1)
            history[i] = k, v
            s = torch.einsum("hrd,hld->hrl", q[i].double().cpu().view(hk, hq // hk, d), k) * d ** -0.5
            ref[i] = torch.einsum("hrl,hld->hrd", s.softmax(-1), v).reshape(hq, d)
        # Weights and result rounded to fp16, and K off by one step where fp32 and fp64 round it apart.
        assert (out.double().cpu() - ref).abs().max() <= 2.0 ** -8 * ref.abs().max()
        logits = (out.float().view(r, -1) @ hd).view(batch, beams, vocab)
        scores, picked, parents = ops.beam_select(logits, scores)
        want = P.select(logits.cpu(), scores_before.cpu() if step else torch.tensor([[0.0] + [-math.inf] * (beams - 1)] * batch),
                        beams, None, -1)
        assert torch.equal(picked.cpu(), want[1]) and torch.equal(parents.cpu(), want[2])
        scores_before = scores
        fresh = torch.tensor([free.pop() for _ in range(r)], dtype=torch.int32)
        new_table, new_lens, used = ops.beam_reorder(parents, table.cuda(), lens.cuda(), fresh.cuda(), kd, vd)
        flat = (parents.cpu().long() + torch.arange(batch)[:, None] * beams).view(-1)
        history = [history[int(i)] for i in flat]
        table, lens = new_table.cpu(), new_lens.cpu()
        held = set(table.flatten().tolist())
        free = sorted((set(free) | {int(f) for f in fresh} | set(range(used_pages, pages))) - held - {-1})
        tokens = picked.cpu().view(-1).long()


def test_captured_step_of_all_operators():
    """Append, attention, selection and reordering in one graph, replayed on other states: as the calls one by one."""
    batch, beams, hq, hk, d, page, vocab, r = 2, 3, 4, 2, 64, 16, 300, 6
    freqs, _ = ops.rope_frequencies(d)
    g = torch.Generator().manual_seed(9)
    shapes = dict(qkv=(r, (hq + 2 * hk) * d), head=(hq * d, vocab))
    fixed = {k: torch.randn(*v, generator=g).cuda() for k, v in shapes.items()}
    kc, vc = (torch.randn(40, hk, page, d, generator=g).to(F16).cuda() for _ in range(2))
    i32 = dict(dtype=torch.int32, device="cuda")
    table, fresh = torch.arange(12, **i32).view(r, 2), torch.arange(20, 20 + r, **i32)
    prefix, plens, starts = torch.arange(30, 34, **i32).view(2, 2), torch.tensor([20, 32], **i32), torch.tensor([0, 3, 6], **i32)
    state = dict(rows=torch.zeros(r, **i32), lens=torch.ones(r, **i32), positions=torch.zeros(r, **i32),
                 scores=torch.zeros(batch, beams, device="cuda"), kc=kc, vc=vc)

    def step(s):
        q = ops.paged_qkv_append(fixed["qkv"], s["positions"], s["rows"], table, s["kc"], s["vc"], hq, freqs)
        out = ops.paged_attention(q, s["kc"], s["vc"], table, s["lens"], prefix, plens, starts)
        logits = (out.view(r, -1, 1).float() * fixed["head"]).sum(1).view(batch, beams, vocab)
        scores, tokens, parents = ops.beam_select(logits, s["scores"])
        return (q, out, scores, tokens, parents, *ops.beam_reorder(parents, table, s["lens"], fresh, s["kc"], s["vc"]))

    step({k: v.clone() for k, v in state.items()})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(state)
    for at in (0, 5, 16, 30):
        state["rows"].fill_(at)
        state["lens"].fill_(at + 1)
        state["positions"].fill_(at + 20)
        state["scores"].copy_(torch.randn(batch, beams, generator=g))
        state["kc"].normal_()
        state["vc"].normal_()
        copy = {k: v.clone() for k, v in state.items()}
        graph.replay()
        want = step(copy)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(state["kc"], copy["kc"]) and torch.equal(state["vc"], copy["vc"])
    assert ops.device_error() == 0
