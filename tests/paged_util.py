"""Plain fp64 forms of the paged-cache operators, on the CPU, and builders of their inputs."""
import math

import torch

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}


def tables(lens, page, seed, spare=3, behind=-1, width=None):
    """Page table over pages in random order, `behind` behind each sequence's last page; and the pages needed."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1) if width is None else width), behind, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, sum(need) + spare, order[at:]


def cache(pages, heads, page, dim, dtype, seed, rows_first=False, layers=None):
    g = torch.Generator().manual_seed(seed)
    shape = (pages, page, heads, dim) if rows_first else (pages, heads, page, dim)
    shape = shape if layers is None else (layers, *shape)
    made = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
    return [x.transpose(-2, -3) if rows_first else x for x in made]


def to_dev(x):
    """On the GPU with the same strides."""
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
    y.copy_(x)
    return y


def rows_of(c, line, n):
    """[heads, n, dim] in fp64."""
    page = c.shape[2]
    if n == 0:
        return torch.zeros(c.shape[1], 0, c.shape[3], dtype=torch.float64)
    return c[line[:-(-n // page)].long()].double().transpose(0, 1).reshape(c.shape[1], -1, c.shape[3])[:, :n]


def attention(q, kc, vc, table, lens, starts, prefix_table=None, prefix_lens=None, group_start=None, scale=None):
    """(out, bound): fp64 result, and what a kernel of the documented precision may be off by, element by element."""
    tokens, hq, d = q.shape
    hk = kc.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    h = HALF[q.dtype]
    for b in range(len(lens)):
        k, v = rows_of(kc, table[b], lens[b]), rows_of(vc, table[b], lens[b])
        shared = 0
        for g in range(0 if prefix_table is None else len(prefix_lens)):
            if group_start[g] <= b < group_start[g + 1]:
                shared = prefix_lens[g]
                k = torch.cat([rows_of(kc, prefix_table[g], shared), k], 1)
                v = torch.cat([rows_of(vc, prefix_table[g], shared), v], 1)
        n = starts[b + 1] - starts[b]
        for j in range(n):
            seen = shared + min(max(lens[b] - n + j + 1, 0), lens[b])
            if seen == 0:
                continue
            t = starts[b] + j
            qt = q[t].double().view(hk, hq // hk, d)
            s = torch.einsum("hrd,hld->hrl", qt, k[:, :seen]) * scale
            w = s.softmax(-1)
            out[t] = torch.einsum("hrl,hld->hrd", w, v[:, :seen]).reshape(hq, d)
            mag = torch.einsum("hrl,hld->hrd", w, v[:, :seen].abs()).reshape(hq, d)
            # Scores: d products added in fp32, with at most one truncation (2^-23) an addition.  An error e of the
            # scores changes each weight by a factor within 1 +- 2 e (numerator and denominator).
            e = d * 2.0 ** -23 * (torch.einsum("hrd,hld->hrl", qt.abs(), k[:, :seen].abs()).amax() * abs(scale)) \
                + 2.0 ** -22 * s.abs().amax() + 2.0 ** -21
            # Weights rounded to the type (half a step), products with V added in fp32, segments joined.
            bound[t] = mag * (h + 2 * e + (seen / 8 + 64) * 2.0 ** -23) + h * out[t].abs()
            if q.dtype == torch.float16:  # weights below 2^-14 have steps of 2^-24
                bound[t] += seen * 2.0 ** -25 * v[:, :seen].abs().amax() + 2.0 ** -25
    return out, bound


def append(qkv, positions, rows, seq, table, kc, vc, hq, freqs, q_gamma, k_gamma, interleaved, magnitude, eps=1e-6):
    """(q, k rows, v rows, bounds of q and k): fp64."""
    tokens, hk, d, rot = qkv.shape[0], kc.shape[1], kc.shape[3], 2 * len(freqs)
    x = qkv.double().view(tokens, -1, d)
    q, k, v = x.split([hq, hk, hk], 1)
    res = []
    for y, gamma in ((q, q_gamma), (k, k_gamma)):
        if gamma is not None:
            y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
        ang = positions.double()[:, None] * freqs.double()
        c, s = ang.cos()[:, None] * magnitude, ang.sin()[:, None] * magnitude
        lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        z, size = y.clone(), y.abs().clone()
        z[..., lo], z[..., hi] = y[..., lo] * c - y[..., hi] * s, y[..., hi] * c + y[..., lo] * s
        both = (y[..., lo].abs() + y[..., hi].abs()) * max(abs(magnitude), 1e-30)
        size[..., lo], size[..., hi] = both, both
        # fp32: a sum of d squares over 5 + d / 32 additions, a square root, three products and a rotation whose angle
        # is off by half a step of half a turn and whose sine by 2 steps: 32 half steps cover them.
        bound = 32 * 2.0 ** -24 * size + HALF[kc.dtype] * (z.abs() + 32 * 2.0 ** -24 * size)
        res.append((z, bound + (2.0 ** -25 if kc.dtype == torch.float16 else 0.0)))
    return res[0][0], res[1][0], v, res[0][1], res[1][1]


def select(logits, scores, n, done, end_token):
    """(scores fp64, tokens, parents) by sorting everything: scores, then beams, then logits, then tokens."""
    batch, beams, vocab = logits.shape
    big = torch.finfo(torch.float32).max
    out = []
    for b in range(batch):
        found = []
        for w in range(beams):
            cum = float(scores[b, w])
            if done is not None and bool(done[b, w]):
                if cum > -math.inf:
                    found.append((-cum, w, 0.0, end_token))
                continue
            x = logits[b, w].double()
            x = torch.where(x.isnan(), -math.inf, x.clamp(max=big))
            if not bool((x > -math.inf).any()) or not cum > -math.inf:
                continue
            d = x - x.max()  # first: beside logits of 1e38 a logarithm of the sum would vanish
            s = cum + (d - d.exp().sum().log())
            order = torch.sort(x, descending=True, stable=True).indices[:n]
            found += [(-float(s[i]), w, -float(x[i]), int(i)) for i in order if float(s[i]) > -math.inf]
        found = sorted(found)[:n]
        found += [(math.inf, -1, 0.0, -1)] * (n - len(found))
        out.append([(-s, v, w) for s, w, _, v in found])
    t = torch.tensor(out, dtype=torch.float64)
    return t[..., 0], t[..., 1].to(torch.int32), t[..., 2].to(torch.int32)


def reorder(parents, table, lens, fresh, caches, page):
    """(table, lens, used, caches) row by row."""
    batch, beams = parents.shape
    new_table, new_lens, used = table.clone(), lens.clone(), torch.zeros_like(lens)
    caches = [c.clone() for c in caches]
    for b in range(batch):
        taken = set()
        for w in range(beams):
            r, p = b * beams + w, int(parents[b, w])
            if not 0 <= p < beams:
                new_table[r], new_lens[r] = -1, 0
                continue
            src = b * beams + p
            new_table[r], new_lens[r] = table[src], lens[src]
            part, slot = int(lens[src]) % page, int(lens[src]) // page
            if p in taken and part:
                old = int(table[src, slot])
                new_table[r, slot], used[r] = fresh[r], 1
                for c in caches:
                    c[..., int(fresh[r]), :, :part, :] = c[..., old, :, :part, :]
            taken.add(p)
    return new_table, new_lens, used, caches
