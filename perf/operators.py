"""What is measured of the paged-cache operators: inputs, plain forms, exact values and work.

The operators of one decode step of a batch of sequences or beams over a paged KV cache:

    append     norms of q and k, rotary positions and the K/V append into pages   (ops.paged_qkv_append)
    attention  sequences that share prefixes, over prefix pages and own pages      (ops.paged_attention)
    select     the n best continuations over beams x vocabulary                    (ops.beam_select)
    reorder    page tables by parent beam, with a copy of the part-full page       (ops.beam_reorder)

`own` is False: `run` computes the plain form; True: `run` calls the framework.
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_FLT_MAX = torch.finfo(torch.float32).max


# ------------------------------------------------------------------------------------------------ cases

def _append(name, **kw):
    c = dict(op="append", tokens=1, seqs=1, start=0, q_heads=32, kv_heads=8, dim=128, rot=128, interleaved=False,
             scaling="none", norm=True, src="float32", cache="float16", page=16)
    return dict(c, **kw, **({"name": name} if name else {}))


def _attention(name, **kw):
    c = dict(op="attention", seqs=1, groups=1, prefix=0, tail=0, new=1, q_heads=32, kv_heads=8, dim=128, page=16,
             type="float16", rows_first=False)
    return dict(c, **kw, **({"name": name} if name else {}))


def _select(name, **kw):
    c = dict(op="select", batch=1, beams=4, vocab=151936, n=4, type="float32", done=False)
    return dict(c, **kw, **({"name": name} if name else {}))


def _reorder(name, **kw):
    c = dict(op="reorder", batch=1, beams=4, layers=36, kv_heads=8, dim=128, page=16, rows=23, type="float16")
    return dict(c, **kw, **({"name": name} if name else {}))


def listed():
    return [
        # The newest token of one sequence: latency is all there is.
        _append("append one token", start=4096),
        # A decode step of a batch in bfloat16, half of each head rotated in interleaved pairs, no norms.
        _append("append 77 sequences", tokens=77, seqs=77, start=3900, rot=64, interleaved=True, norm=False,
                src="bfloat16", cache="bfloat16", page=32),
        # Prompts of several sequences, positions stretched for a long context.
        _append("append prompts", tokens=8190, seqs=3, start=30000, scaling="yarn", page=64),
        # One sequence at the context of the decode benchmark.
        _attention("attend one sequence", tail=4096),
        # A few beams over one prompt of odd length, heads of 64, cache rows ahead of heads.
        _attention("attend 5 beams", seqs=5, prefix=1019, tail=37, q_heads=16, kv_heads=4, dim=64, type="bfloat16",
                   rows_first=True),
        # Ragged own contexts, nothing shared: a plain batch of a server.
        _attention("attend 48 ragged", seqs=48, tail=5000, page=32, type="bfloat16"),
        # Two long documents with many questions about each: as much for the tensor cores as for HBM.
        _attention("attend 128 on 2 documents", seqs=128, groups=2, prefix=32768, tail=512, page=64),
        # Prompts of several sequences behind one system prompt: causal over their own rows.
        _attention("attend prompts", seqs=4, prefix=1500, tail=1100, new=1024, page=32, type="bfloat16"),
        # Beams of one sentence.
        _select("select 4 beams"),
        # A batch of sentences, some beams done, twice as many candidates as beams.
        _select("select 32 x 8 beams", batch=32, beams=8, n=16, type="bfloat16", done=True),
        # Beams of one sentence, and of a batch, over all layers' caches.
        _reorder("reorder 4 beams"),
        _reorder("reorder 16 x 8 beams", batch=16, beams=8, rows=45, page=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "select", "reorder"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = dict(kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 8]))
    dim, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256])
    kind = rng.choice(["float16", "bfloat16"])
    if op == "append":
        tokens = _log(rng, 1, 8190)
        rot = rng.choice([dim, dim // 2, dim // 4, rng.randrange(2, dim + 1, 2)])
        return _append(None, tokens=tokens, seqs=rng.randint(1, min(tokens, 64)), start=_log(rng, 1, 100000), dim=dim,
                       rot=rot, interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "yarn"]),
                       norm=rng.random() < 0.6, src=rng.choice(["float32", "float16", "bfloat16"]), cache=kind,
                       page=page, **heads)
    if op == "attention":
        heads["q_heads"] = min(heads["q_heads"], 32)
        heads["q_heads"] -= heads["q_heads"] % kv_heads
        common = dict(dim=dim, page=page, type=kind, rows_first=rng.random() < 0.5, **heads)
        what = rng.choice(["one", "batch", "prefix", "prefix", "prompt"])
        if what == "one":
            return _attention(None, tail=_log(rng, 1, 100000), **common)
        if what == "batch":
            return _attention(None, seqs=_log(rng, 2, 48), tail=_log(rng, 1, 4000), **common)
        if what == "prefix":
            groups = rng.choice([1, 1, 2, 3])
            return _attention(None, seqs=groups * _log(rng, 1, 40), groups=groups, prefix=_log(rng, 10, 32000),
                              tail=_log(rng, 1, 1000), **common)
        new = _log(rng, 2, 700)
        return _attention(None, seqs=rng.randint(1, 4), prefix=rng.choice([0, _log(rng, 10, 1500)]), new=new,
                          tail=new + _log(rng, 1, 500), **common)
    if op == "select":
        beams = rng.randint(1, 12)
        return _select(None, batch=_log(rng, 1, 20), beams=beams, vocab=_log(rng, 1000, 151936),
                       n=rng.randint(1, 2 * beams), type=rng.choice(["float32", "float16", "bfloat16"]),
                       done=rng.random() < 0.5)
    return _reorder(None, batch=_log(rng, 1, 16), beams=rng.randint(1, 8), layers=rng.randint(1, 36), kv_heads=kv_heads,
                    dim=dim, page=page, rows=_log(rng, 1, 300), type=kind)


# ------------------------------------------------------------------------------------------------ inputs

def _frequencies(rot, scaling):
    """Radians a position for each pair, and the factor on cosines and sines: base 5e6, contexts of 32768 stretched 4 x."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    freqs, base, factor, original = 5e6 ** (-2 * i / rot), 5e6, 4.0, 32768
    if scaling == "linear":
        return freqs / factor, 1.0
    if scaling == "yarn":
        # Pairs that turn more than 32 times over the original context stay, those below one turn are stretched,
        # with a ramp over the pair's index between.
        at = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return freqs * (1 - ramp) + freqs / factor * ramp, 0.1 * math.log(factor) + 1.0
    return freqs, 1.0


def _tails(case):
    """Own rows of each sequence, the attended tokens among them: ragged, the second sequence of a decode batch none."""
    t, n = case["tail"], case["new"]
    lens = [t - (i * 7919) % (t // 2 + 1) for i in range(case["seqs"])]
    if n > 1:
        lens = [max(x, k) for x, k in zip(lens, _news(case))]
    elif case["prefix"] and case["seqs"] > 1:
        lens[1] = 0
    return lens


def _news(case):
    return [case["new"] - (i * 131) % (case["new"] // 3 + 1) for i in range(case["seqs"])]


def _tables(lens, page, gen, spare=0):
    """A page table (-1 behind each sequence's last page) over randomly placed pages, and the number of pages."""
    need = [-(-x // page) for x in lens]
    width = max(max(need), 1)
    order = torch.randperm(sum(need) + spare, generator=gen).to(torch.int32)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, sum(need) + spare


def _caches(pages, case, kind, g, layers=None):
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    shape = (pages, p, h, d) if case.get("rows_first") else (pages, h, p, d)
    shape = shape if layers is None else (layers,) + shape
    made = [torch.randn(shape, generator=g, device="cuda", dtype=kind) for _ in range(2)]
    return [x.transpose(1, 2) if case.get("rows_first") else x for x in made]


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["op"]](case, cpu, g)


def _prepare_append(case, cpu, g):
    t, n, d = case["tokens"], case["seqs"], case["dim"]
    per = [t // n + (i < t % n) for i in range(n)]
    base = [(i * 577) % (case["start"] // 4 + 1) for i in range(n)]  # rows already held
    table, pages = _tables([b + k for b, k in zip(base, per)], case["page"], cpu)
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(per)).to(torch.int32)
    rows = torch.cat([torch.arange(b, b + k) for b, k in zip(base, per)]).to(torch.int32)
    width = (case["q_heads"] + 2 * case["kv_heads"]) * d
    freqs, magnitude = _frequencies(case["rot"], case["scaling"])
    kc, vc = _caches(pages, case, _TYPES[case["cache"]], g)
    gammas = [(0.5 + torch.rand(d, generator=g, device="cuda")) if case["norm"] else None for _ in range(2)]
    qkv = (torch.randn(t, width, generator=g, device="cuda") * 3).to(_TYPES[case["src"]])
    return dict(case=case, qkv=qkv, positions=(rows + case["start"]).to(torch.int32).cuda(), rows=rows.cuda(),
                seq=None if t == n else seq.cuda(), table=table.cuda(), k_cache=kc, v_cache=vc, freqs=freqs.cuda(),
                magnitude=magnitude, q_gamma=gammas[0], k_gamma=gammas[1],
                q_out=torch.empty(t, case["q_heads"], d, device="cuda", dtype=kc.dtype))


def _prepare_attention(case, cpu, g):
    kind, page = _TYPES[case["type"]], case["page"]
    tails, b, groups = _tails(case), case["seqs"], case["groups"]
    all_lens = tails + [case["prefix"]] * (groups if case["prefix"] else 0)
    table, pages = _tables(all_lens, page, cpu)
    kc, vc = _caches(pages, case, kind, g)
    # Rows behind a sequence's last are whatever an earlier user of the page left there: not numbers at all.
    for i, x in enumerate(all_lens):
        if x % page:
            last = int(table[i, x // page])
            kc[last, :, x % page:] = math.nan
            vc[last, :, x % page:] = math.nan
    news = _news(case) if case["new"] > 1 else [1] * b
    starts = torch.tensor([0] + news).cumsum(0).to(torch.int32)
    q = (torch.randn(sum(news), case["q_heads"], case["dim"], generator=g, device="cuda") * 2).to(kind)
    s = dict(case=case, q=q, k_cache=kc, v_cache=vc, new_most=max(news), tail_most=max(max(tails), 1),
             table=table[:b, :-(-max(max(tails), 1) // page)].contiguous().cuda(),
             lens=torch.tensor(tails, dtype=torch.int32).cuda(),
             q_start=starts.cuda() if case["new"] > 1 else None, prefix_table=None, prefix_lens=None, group_start=None,
             out=torch.empty_like(q))
    if case["prefix"]:
        s["prefix_table"] = table[b:, :-(-case["prefix"] // page)].contiguous().cuda()
        s["prefix_lens"] = torch.full((groups,), case["prefix"], dtype=torch.int32).cuda()
        s["group_start"] = (torch.arange(groups + 1) * (b // groups)).to(torch.int32).cuda() if groups > 1 else None
    return s


def _prepare_select(case, cpu, g):
    b, w, v = case["batch"], case["beams"], case["vocab"]
    logits = (torch.randn(b, w, v, generator=g, device="cuda") * 3).to(_TYPES[case["type"]])
    # A tenth of the vocabulary is not allowed next.
    logits[:, :, torch.rand(v, generator=g, device="cuda") < 0.1] = -math.inf
    scores = -torch.rand(b, w, generator=g, device="cuda") * 10 - 5
    done = torch.rand(b, w, generator=g, device="cuda") < 0.2 if case["done"] else None
    if done is not None:
        done[:, 0] = False  # a batch entry whose beams are all done has left the batch
    return dict(case=case, logits=logits, scores=scores, done=done, end_token=v - 7)


def _reorder_rows(case):
    """Rows held, the same for all beams of a batch entry."""
    return [case["rows"] - (i * 7) % (case["rows"] // 2 + 1) for i in range(case["batch"])]


def _prepare_reorder(case, cpu, g):
    b, w, page = case["batch"], case["beams"], case["page"]
    lens = _reorder_rows(case)
    full, r = [x // page for x in lens], b * w
    order = torch.randperm(sum(full) + 2 * r, generator=cpu).to(torch.int32)
    width = max(full) + 1
    table, at = torch.full((r, width), -1, dtype=torch.int32), 2 * r
    for i, k in enumerate(full):  # whole pages are shared by the beams, the part-full one is a beam's own
        table[i * w:(i + 1) * w, :k] = order[at:at + k]
        if lens[i] % page:
            table[i * w:(i + 1) * w, k] = order[i * w:(i + 1) * w]
        at += k
    half = (w + 1) // 2  # half of the beams go on, most of them twice
    parents = torch.stack([torch.randperm(w, generator=cpu)[:half].repeat(2)[:w][torch.randperm(w, generator=cpu)]
                           for _ in range(b)]).to(torch.int32)
    kc, vc = _caches(sum(full) + 2 * r, case, _TYPES[case["type"]], g, case["layers"])
    lens = torch.tensor(lens, dtype=torch.int32).repeat_interleave(w)
    return dict(case=case, parents=parents.cuda(), table=table.cuda(), lens=lens.cuda(), fresh=order[r:2 * r].cuda(),
                k_cache=kc, v_cache=vc)


# ------------------------------------------------------------------------------------------------ passes

def run(s):
    return {"append": _run_append, "attention": _run_attention, "select": _run_select,
            "reorder": _run_reorder}[s["case"]["op"]](s)


def _run_append(s):
    c = s["case"]
    if own:
        from mojo_llm_lab_b200 import ops
        q = ops.paged_qkv_append(s["qkv"], s["positions"], s["rows"], s["table"], s["k_cache"], s["v_cache"],
                                 c["q_heads"], s["freqs"], seq=s["seq"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"],
                                 interleaved=c["interleaved"], magnitude=s["magnitude"], q_out=s["q_out"])
        return q, s["k_cache"], s["v_cache"]
    t, hq, hk, d, rot = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s["qkv"].float().view(t, hq + 2 * hk, d)
    qk, v = x[:, :hq + hk], x[:, hq + hk:]
    if c["norm"]:
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6)
        qk = torch.cat([qk[:, :hq] * s["q_gamma"], qk[:, hq:] * s["k_gamma"]], 1)
    angle = s["positions"].double()[:, None] * s["freqs"]  # far positions lose their angle in 32 bits
    cos = (angle.cos() * s["magnitude"]).float()[:, None]
    sin = (angle.sin() * s["magnitude"]).float()[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = qk[..., first], qk[..., second]
    y = qk.clone()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    kind, page = s["k_cache"].dtype, c["page"]
    rows = s["rows"].long()
    seq = torch.arange(t, device=rows.device) if s["seq"] is None else s["seq"].long()
    pages = s["table"][seq, rows // page].long()
    s["k_cache"][pages, :, rows % page] = y[:, hq:].to(kind)
    s["v_cache"][pages, :, rows % page] = v.to(kind)
    return y[:, :hq].to(kind), s["k_cache"], s["v_cache"]


def _gather(cache, table, lens):
    """[n, heads, rows, dim] in 32 bits of n sequences' pages, zeros from each one's length on, and which rows those are."""
    n, p = table.shape
    x = cache[table.clamp(min=0).long()].float()  # [n, p, heads, page, dim]
    x = x.transpose(1, 2).reshape(n, cache.shape[1], p * cache.shape[2], cache.shape[3])
    held = torch.arange(x.shape[2], device=x.device) < lens[:, None]
    return torch.where(held[:, None, :, None], x, 0.0), held


def _run_attention(s):
    c = s["case"]
    if own:
        from mojo_llm_lab_b200 import ops
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                   prefix_table=s["prefix_table"], prefix_lens=s["prefix_lens"],
                                   group_start=s["group_start"], q_start=s["q_start"], out=s["out"])
    b, hq, hk, d, n = c["seqs"], c["q_heads"], c["kv_heads"], c["dim"], s["new_most"]
    q = s["q"].float() / math.sqrt(d)
    if s["q_start"] is None:
        count = torch.ones(b, dtype=torch.int64, device=q.device)
        at = torch.arange(b, device=q.device)[:, None]
    else:
        count = (s["q_start"][1:] - s["q_start"][:-1]).long()
        at = s["q_start"][:-1, None] + torch.arange(n, device=q.device)
    at = at.clamp(max=q.shape[0] - 1)
    # [sequence, kv head, query head of it, token, dim]
    q = q[at].view(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    k, held = _gather(s["k_cache"], s["table"], s["lens"])
    v, _ = _gather(s["v_cache"], s["table"], s["lens"])
    # Token j of a sequence's last `count` sees its own rows up to itself.
    seen = s["lens"][:, None] - count[:, None] + torch.arange(n, device=q.device) + 1
    seen = torch.arange(k.shape[2], device=q.device) < seen[..., None]
    own_scores = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).view(b, hk, hq // hk, n, -1)
    own_scores = torch.where((seen & held[:, None])[:, None, None], own_scores, -math.inf)
    top = own_scores.amax(-1, keepdim=True)
    if s["prefix_table"] is not None:
        g = s["prefix_table"].shape[0]
        pk, pheld = _gather(s["k_cache"], s["prefix_table"], s["prefix_lens"])
        pv, _ = _gather(s["v_cache"], s["prefix_table"], s["prefix_lens"])
        # A group's queries side by side: [group, kv head, sequences x query heads x tokens, dim]
        pq = q.reshape(g, b // g, hk, -1, d).transpose(1, 2).reshape(g, hk, -1, d)
        scores = torch.matmul(pq, pk.transpose(-1, -2))
        scores = scores.masked_fill(~pheld[:, None, None], -math.inf)
        back = lambda x: x.view(g, hk, b // g, hq // hk, n, -1).transpose(1, 2).reshape(b, hk, hq // hk, n, -1)  # noqa: E731
        there = lambda x: x.view(g, b // g, hk, hq // hk, n, -1).transpose(1, 2).reshape(g, hk, -1, x.shape[-1])  # noqa: E731
        top = torch.maximum(top, back(scores.amax(-1, keepdim=True)))
    safe = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(own_scores - safe)
    total, y = w.sum(-1, keepdim=True), torch.matmul(w.flatten(2, 3), v).view(b, hk, hq // hk, n, d)
    if s["prefix_table"] is not None:
        w = torch.exp(scores - there(safe))
        total, y = total + back(w.sum(-1, keepdim=True)), y + back(torch.matmul(w, pv))
    y = torch.where(total > 0, y / total, 0.0)
    y = y.permute(0, 3, 1, 2, 4).reshape(b * n, hq, d).to(s["q"].dtype)
    if s["q_start"] is None:
        return y
    token = torch.arange(s["q"].shape[0], device=q.device)
    which = torch.searchsorted(s["q_start"], token, right=True) - 1
    return y[which * n + token - s["q_start"][which]]


def _run_select(s):
    c = s["case"]
    if own:
        from mojo_llm_lab_b200 import ops
        return ops.beam_select(s["logits"], s["scores"], n=c["n"], done=s["done"], end_token=s["end_token"])
    b, w, v, n = c["batch"], c["beams"], c["vocab"], c["n"]
    # In 64 bits: candidates of different beams lie close.
    x = s["logits"].double().nan_to_num(nan=-math.inf, posinf=_FLT_MAX, neginf=-math.inf)
    top = x.amax(-1, keepdim=True)
    total = top + (x - top).exp().sum(-1, keepdim=True).log()
    x = (x - total).nan_to_num(nan=-math.inf, neginf=-math.inf) + s["scores"].double()[..., None]
    if s["done"] is not None:
        only = torch.full_like(x, -math.inf)
        only[..., s["end_token"]] = s["scores"].double()
        x = torch.where(s["done"][..., None], only, x)
    # More than are wanted, so that equal ones at the border can be put in order of their places.
    x = x.view(b, w * v)
    best, place = x.topk(min(n + 32, w * v), dim=1)
    place, order = place.sort(1)
    best, order = best.gather(1, order).sort(dim=1, descending=True, stable=True)
    place = place.gather(1, order)[:, :n]
    return best[:, :n].float(), (place % v).to(torch.int32), (place // v).to(torch.int32)


def _run_reorder(s):
    c = s["case"]
    if own:
        from mojo_llm_lab_b200 import ops
        table, lens, used = ops.beam_reorder(s["parents"], s["table"], s["lens"], s["fresh"], s["k_cache"], s["v_cache"])
        return table, lens, used, s["k_cache"], s["v_cache"]
    b, w, page = c["batch"], c["beams"], c["page"]
    r = b * w
    row = torch.arange(r, device=s["table"].device)
    parent = (s["parents"].long() + torch.arange(b, device=row.device)[:, None] * w).view(-1)
    table, lens = s["table"][parent], s["lens"][parent]
    part = (lens % page).long()
    earlier = ((parent[:, None] == parent) & (row[:, None] > row)).any(1)
    copied = earlier & (part > 0)
    at = (lens // page).long()
    last = torch.where(copied, table.gather(1, at.clamp(max=table.shape[1] - 1)[:, None])[:, 0].long(), 0)
    fresh = s["fresh"].long()
    take = (copied[:, None] & (torch.arange(page, device=row.device) < part[:, None]))[None, :, None, :, None]
    for cache in (s["k_cache"], s["v_cache"]):
        cache[:, fresh] = torch.where(take, cache[:, last], cache[:, fresh])
    column = torch.arange(table.shape[1], device=row.device)
    table = torch.where(copied[:, None] & (column == at[:, None]), s["fresh"][:, None], table)
    return table, lens, copied.to(torch.int32), s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------ work

def _seen(case):
    """(query row, key) pairs of one query head."""
    news = _news(case) if case["new"] > 1 else [1] * case["seqs"]
    own_rows = sum(max(0, x - n + j + 1) for x, n in zip(_tails(case), news) for j in range(n))
    return own_rows + sum(news) * case["prefix"], sum(news)


def work(case):
    c = case
    size = lambda t: _TYPES[t].itemsize  # noqa: E731
    if c["op"] == "append":
        heads = c["q_heads"] + 2 * c["kv_heads"]
        values = c["tokens"] * heads * c["dim"]
        return dict(bytes=values * (size(c["src"]) + size(c["cache"])) + c["tokens"] * 16 + c["rot"] * 4,
                    flops=values * (4 if c["norm"] else 0) + c["tokens"] * (c["q_heads"] + c["kv_heads"]) * c["rot"] * 3)
    if c["op"] == "attention":
        pairs, tokens = _seen(c)
        keys = sum(_tails(c)) + c["groups"] * c["prefix"]
        return dict(bytes=2 * 2 * keys * c["kv_heads"] * c["dim"] + 2 * 2 * tokens * c["q_heads"] * c["dim"],
                    flops=4 * pairs * c["q_heads"] * c["dim"])
    if c["op"] == "select":
        rows = c["batch"] * c["beams"]
        return dict(bytes=rows * c["vocab"] * size(c["type"]) + rows * 5 + c["batch"] * c["n"] * 12,
                    flops=rows * c["vocab"] * 4)
    further = c["beams"] - (c["beams"] + 1) // 2
    rows = sum(x % c["page"] for x in _reorder_rows(c)) * further
    table = c["batch"] * c["beams"] * (max(_reorder_rows(c)) // c["page"] + 1) * 4
    return dict(bytes=rows * c["layers"] * 2 * c["kv_heads"] * c["dim"] * 2 * 2 + 2 * table + c["batch"] * c["beams"] * 20,
                flops=0)


# ------------------------------------------------------------------------------------------------ exact values

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "select": _exact_select,
            "reorder": _exact_reorder}[case["op"]](s)


def _exact_append(s):
    """Each pair as a complex number times magnitude x e^(i angle)."""
    c = s["case"]
    t, hq, hk, d, rot = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"], c["rot"]
    q, k, v = s["qkv"].double().view(t, -1, d).split([hq, hk, hk], 1)
    done = []
    for x, gamma in ((q, s["q_gamma"]), (k, s["k_gamma"])):
        if gamma is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * gamma.double()
        turned, rest = x[..., :rot], x[..., rot:]
        pairs = turned.unflatten(-1, (rot // 2, 2)) if c["interleaved"] else turned.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        angle = torch.outer(s["positions"].double(), s["freqs"])
        z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]
        z = torch.view_as_real(z)
        z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
        done.append(torch.cat([z, rest], -1))
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    seq = range(t) if s["seq"] is None else s["seq"].tolist()
    slot = torch.tensor([int(p) for p in s["table"].cpu()[torch.tensor(list(seq)).long(), s["rows"].cpu().long() // c["page"]]])
    slot, row = slot.cuda(), s["rows"].long() % c["page"]
    kc[slot, :, row], vc[slot, :, row] = done[1], v
    return done[0], kc, vc


def _exact_attention(s):
    """Sequence by sequence: prefix and own rows in one softmax."""
    c = s["case"]
    b, hq, hk, d, page = c["seqs"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    starts = list(range(b + 1)) if s["q_start"] is None else s["q_start"].tolist()
    lens, out = s["lens"].tolist(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    rows = lambda cache, table, n: cache[table[:-(-n // page)].long()].double().permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n]  # noqa: E731
    shared = None
    for i in range(b):
        if c["prefix"] and i % (b // c["groups"]) == 0:
            t = s["prefix_table"][i // (b // c["groups"])]
            shared = rows(s["k_cache"], t, c["prefix"]), rows(s["v_cache"], t, c["prefix"])
        k, v = rows(s["k_cache"], s["table"][i], lens[i]), rows(s["v_cache"], s["table"][i], lens[i])
        if shared is not None:
            k, v = torch.cat([shared[0], k], 1), torch.cat([shared[1], v], 1)
        n = starts[i + 1] - starts[i]
        if not k.shape[1]:
            continue
        q = s["q"][starts[i]:starts[i + 1]].double().unflatten(1, (hk, hq // hk))
        x = torch.einsum("nhrd,hld->hrnl", q, k) / d ** 0.5
        hidden = torch.ones(n, k.shape[1], dtype=torch.bool, device="cuda").triu(k.shape[1] - n + 1)
        if n > 1:
            x = x.masked_fill(hidden, -math.inf)
        elif lens[i] == 0 and not c["prefix"]:
            continue
        out[starts[i]:starts[i + 1]] = torch.einsum("hrnl,hld->nhrd", x.softmax(-1), v).flatten(1, 2)
    return out


def _exact_select(s):
    c = s["case"]
    found = []
    for i in range(c["batch"]):
        each = s["logits"][i].double().log_softmax(-1) + s["scores"][i].double()[:, None]
        if s["done"] is not None:
            each = each[~s["done"][i]]
            each = torch.cat([each.flatten(), s["scores"][i][s["done"][i]].double()])
        found.append(each.flatten().sort(descending=True).values[:c["n"]])
    return torch.stack(found), None, None


def _exact_reorder(s):
    return None
