"""Beam selection on the GPU against a plain fp64 sort of every candidate."""
import math

import pytest
import torch

import paged_util as P
from mojo_llm_lab_b200 import ops

pytestmark = pytest.mark.gpu


def check(logits, scores, n, done=None, end_token=-1, device_logits=None, **kw):
    dev = logits.cuda() if device_logits is None else device_logits
    got = ops.beam_select(dev, scores.cuda(), n=n, done=None if done is None else done.cuda(), end_token=end_token, **kw)
    want = P.select(logits, scores, n, done, end_token)
    assert torch.equal(got[1].cpu(), want[1]), "tokens"
    assert torch.equal(got[2].cpu(), want[2]), "parents"
    s, ref = got[0].double().cpu(), want[0]
    assert torch.equal(s.isinf(), ref.isinf())
    fine = ref.isfinite()
    # One rounding to fp32, and the logarithm's error, the relative one of the sum.  A term 2^t, t = d log2(e) in fp32:
    # the unit's 2 steps (2^-22), and t off by half a step, 2^-20 up to |t| = 32, which changes it by ln 2 times that;
    # terms below 2^-32 are 2^-14 of the sum at most.  Equal logits have equal errors, so nothing averages out:
    # 2^-22 + 0.7 x 2^-20 < 2^-20.
    assert ((s - ref)[fine].abs() <= 2.0 ** -24 * ref[fine].abs() + 2.0 ** -20).all()
    return got


def random(batch, beams, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(batch, beams, vocab, generator=g) * spread).to(dtype)
    return logits, -torch.rand(batch, beams, generator=g) * 8


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,n", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 100, 6), (1, 4, 4096, 4), (3, 2, 4097, 5),
                                                 (1, 5, 12288, 64), (2, 64, 999, 64), (1, 8, 50001, 16), (2, 4, 151936, 8)])
def test_select(batch, beams, vocab, n, dtype):
    check(*random(batch, beams, vocab, dtype, vocab + n), n)


def test_select_ties_go_to_the_lowest_place():
    logits = torch.zeros(2, 3, 9000)
    logits[1, 1, 8000:] = 1.0
    check(logits, torch.zeros(2, 3), 8)
    check(logits.bfloat16(), torch.tensor([[0.0, 0.0, 0.0], [-1.0, -1.0, -1.0]]), 40)
    signed = torch.zeros(1, 1, 5000)
    signed[0, 0, ::2] = -0.0  # the two zeros are one value
    check(signed, torch.zeros(1, 1), 5)


def test_select_order_that_defeats_the_threshold():
    """All large logits in one thread's share, or sorted: more keys reach the threshold than are wanted."""
    up = torch.arange(40000, dtype=torch.float32).view(1, 2, 20000) * 1e-3
    check(up, torch.zeros(1, 2), 64)
    check(up.flip(2), torch.zeros(1, 2), 64)
    one = torch.full((1, 1, 4096), -9.0)
    one[0, 0, torch.arange(16) * 256] = torch.arange(16.0)  # one thread's (unvectorised)
    check(one, torch.zeros(1, 1), 10)
    many = torch.full((1, 64, 4096 * 3), -5.0)
    many[0, 0] = torch.linspace(0, 1, 4096 * 3)
    check(many, torch.zeros(1, 64), 64)


def test_select_first_step_and_banned_tokens():
    """One live beam of several, most tokens not allowed: places without a candidate are marked."""
    logits, scores = random(2, 4, 3000, torch.float32, 8)
    scores[:, 1:] = -math.inf
    check(logits, scores, 4)
    logits[0, 0] = -math.inf
    logits[0, 0, 2990:2992] = 1.0
    got = check(logits, scores, 5)
    assert got[1][0].tolist() == [2990, 2991, -1, -1, -1] and got[2][0].tolist() == [0, 0, -1, -1, -1]
    assert (got[0][0, 2:] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_select_masks_of_the_lowest_value(dtype):
    """Tokens masked with the type's lowest value are candidates still: long runs of equal keys, few others among them."""
    logits, scores = random(2, 3, 20000, dtype, 15)
    low = torch.finfo(dtype).min
    logits[0, 0, 40:] = low
    logits[0, 1] = low
    logits[0, 2, :19995] = low
    logits[1, :, 3000:16500] = -math.inf
    logits[1, 1, :3000] = low
    check(logits, scores, 6)
    check(logits, scores, 64)


@pytest.mark.parametrize("vocab,pad", [(9000, 0), (9001, 0), (9003, 5), (40000, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_many_rows(vocab, pad, dtype):
    """So many rows that a CTA takes several steps of one, ending inside a step and inside a vector."""
    logits, scores = random(150, 4, vocab, dtype, 16)
    wide = torch.full((150, 4, vocab + pad), math.nan, dtype=dtype)
    wide[..., :vocab] = logits
    check(logits, scores, 5, device_logits=wide.cuda()[..., :vocab])
    logits[..., 100:] = logits[..., 7:8]  # equal ones from there on
    check(logits, scores, 5)


def test_select_not_numbers():
    logits, scores = random(1, 3, 5000, torch.float32, 9)
    logits[0, 0, 100:200] = math.nan
    logits[0, 1, 77] = math.inf
    logits[0, 2] = math.nan
    check(logits, scores, 6)
    scores[0, 0] = math.nan
    check(logits, scores, 6)


@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
def test_select_done_beams(kind):
    logits, scores = random(3, 4, 6000, torch.bfloat16, 10)
    done = torch.tensor([[0, 1, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0]]).to(kind)
    scores[0, 1] = 0.0
    logits[0, 1] = math.nan  # not read
    got = check(logits, scores, 8, done, 17)
    assert got[1][0, 0] == 17 and got[2][0, 0] == 1 and got[0][0, 0] == 0.0
    assert (got[1][1, :4] == 17).all() and (got[1][1, 4:] == -1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [1, 8])
def test_select_strided_logits(dtype, pad):
    """Rows that are slices of wider ones, on 16-byte boundaries or not."""
    logits, scores = random(2, 3, 5001, dtype, 11)
    wide = torch.full((2, 4, 5001 + pad + 6), math.nan, dtype=dtype)
    wide[:, :3, pad:pad + 5001] = logits
    check(logits, scores, 6, device_logits=wide.cuda()[:, :3, pad:pad + 5001])
    turned = logits.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    check(logits, scores, 6, device_logits=turned)


def test_select_captured_and_on_another_stream():
    logits, scores = random(2, 4, 20000, torch.float32, 12)
    dev, sc = logits.cuda(), scores.cuda()
    out = (torch.empty(2, 6, device="cuda"), torch.empty(2, 6, dtype=torch.int32, device="cuda"),
           torch.empty(2, 6, dtype=torch.int32, device="cuda"))
    ops.beam_select(dev, sc, n=6, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_select(dev, sc, n=6, out=out)
    for seed in (13, 14):
        logits, scores = random(2, 4, 20000, torch.float32, seed)
        dev.copy_(logits)
        sc.copy_(scores)
        graph.replay()
        torch.cuda.synchronize()
        want = P.select(logits, scores, 6, None, -1)
        assert torch.equal(out[1].cpu(), want[1]) and torch.equal(out[2].cpu(), want[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(logits, scores, 6)


def test_select_into_its_scores_and_shared_logits():
    """New scores written over the old ones; logits that all beams share (stride 0)."""
    logits, scores = random(3, 5, 7000, torch.float32, 21)
    dev, sc = logits[:, :1].cuda().expand(3, 5, 7000), scores.cuda()
    want = P.select(logits[:, :1].expand(3, 5, 7000).contiguous(), scores, 5, None, -1)
    out = (sc, torch.empty(3, 5, dtype=torch.int32, device="cuda"), torch.empty(3, 5, dtype=torch.int32, device="cuda"))
    alone = ops.beam_select(dev, sc)
    ops.beam_select(dev, sc, out=out)
    assert torch.equal(out[1].cpu(), want[1]) and torch.equal(out[2].cpu(), want[2])
    assert all(torch.equal(x, y) for x, y in zip(out, alone))
