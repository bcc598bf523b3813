"""Batches of drafted token trees for the tests of their operators, and the formulas in 64 bits, request by request."""
import math
import random

import torch


def make_trees(nodes, seed=0, width=3, roots=1):
    """Parents of each request's nodes: random earlier ones; the first ``roots`` nodes (and some others, where more than one) have none."""
    rng, out = random.Random(seed), []
    for n in nodes:
        parents = []
        for i in range(n):
            if i < roots or (roots > 1 and rng.random() < 0.1):
                parents.append(-1)
            else:
                parents.append(rng.randrange(max(0, i - 3 * width), i))
        out.append(parents)
    return out


def ways_of(parents):
    ways = []
    for i, up in enumerate(parents):
        ways.append((ways[up] if up >= 0 else []) + [i])
    return ways


def tree_batch(prefix, nodes, hq, hkv, D, seed=0, dtype=torch.bfloat16, cache=None, head_major=True, page=1, roots=1, spare=0, device="cuda",
               trees=None, std=1.0):
    """Tensors of a batch: slots shuffled page by page, request rows not in the batch's order, ``spare`` rows behind the last tree."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    trees = make_trees(nodes, seed, roots=roots) if trees is None else trees
    B, T = len(nodes), sum(nodes) + spare
    lens = [p + n for p, n in zip(prefix, nodes)]
    pages = [-(-s // page) for s in lens]
    order = list(range(1, sum(pages) + 3))
    rng.shuffle(order)
    slots = (max(order) + 1) * page
    rows = list(range(B))
    rng.shuffle(rows)
    table = torch.zeros((B + 2, max(lens) + 5), dtype=torch.int32)
    at = 0
    for b, s in enumerate(lens):
        table[rows[b], :s] = torch.tensor([order[at + i // page] * page + i % page for i in range(s)], dtype=torch.int32)
        at += pages[b]

    def normal(*shape):
        return torch.randn(shape, generator=g) * std

    store = dtype if cache is None else cache
    shape = (hkv, slots, D) if head_major else (slots, hkv, D)
    k, v = (normal(*shape).to(device).to(store) for _ in range(2))
    if head_major:
        k, v = k.transpose(0, 1), v.transpose(0, 1)
    parents = [p for t in trees for p in t] + [-1] * spare
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=normal(T, hq, D).to(device).to(dtype), k=k, v=v, table=table.to(device), req=ints(rows), seq=ints(lens), prefix=ints(prefix),
                start=ints([sum(nodes[:i]) for i in range(B)]), parents=ints(parents), scale=D ** -0.5, trees=trees, slots=slots)


def exact_attention(c, window=None, logit_cap=0.0, sink=None, chunk=None, bounds=False):
    """The definition in 64 bits; rows that belong to no request are zero.  ``bounds``: also, per element, the largest error that a kernel
    may make which rounds weights and results to the activation type (half a step each: of the weighted sum of |v|, and of the result)
    and forms scores in 32 bits (D roundings of the sum of |q k|, and 2^-21 of the exponential, twice: numerator and denominator)."""
    q = c["q"].double()
    want, bound = torch.zeros_like(q), torch.zeros_like(q)
    hkv, D = c["k"].shape[1], q.shape[2]
    half = torch.finfo(c["q"].dtype).eps / 2
    for b, parents in enumerate(c["trees"]):
        pl, qs, n = int(c["prefix"][b]), int(c["start"][b]), len(parents)
        slots = c["table"][int(c["req"][b]), :pl + n].long()
        k, v = (t[slots].double() for t in (c["k"], c["v"]))
        for i, way in enumerate(ways_of(parents)):
            at = pl + len(way) - 1
            low = 0
            if window:
                low = max(0, at - window + 1)
            if chunk:
                low = at // chunk * chunk
            see = list(range(low, pl)) + [pl + node for up, node in enumerate(way) if pl + up >= low]
            kk, vv = k[see], v[see]
            x = q[qs + i].view(hkv, -1, D)
            s = torch.einsum("kgd,lkd->kgl", x, kk) * c["scale"]
            span = torch.einsum("kgd,lkd->kgl", x.abs(), kk.abs()).amax().item() * c["scale"]
            if logit_cap:
                s = logit_cap * torch.tanh(s / logit_cap)
            if sink is not None:
                s = torch.cat([s, sink.double().view(hkv, -1, 1)], dim=-1)
            w = torch.softmax(s, dim=-1)[..., :len(see)]
            o = torch.einsum("kgl,lkd->kgd", w, vv).reshape(-1, D)
            reach = torch.einsum("kgl,lkd->kgd", w, vv.abs()).reshape(-1, D)
            want[qs + i] = o
            bound[qs + i] = half * (o.abs() + reach) + reach * 2 * (D * 2 ** -24 * span + 2 ** -21)
    return (want, bound) if bounds else want


def exact_prologue(c, qkv, gains, inv_freq, hq, hkv, eps, delta=None):
    """(q, k, v) [T, heads, D] in 64 bits; rows of no request are zero."""
    T, D, half = qkv.shape[0], qkv.shape[1] // (hq + 2 * hkv), inv_freq.numel()
    x = qkv.double().view(T, hq + 2 * hkv, D)
    pos = torch.zeros(T, dtype=torch.float64)
    known = torch.zeros(T, dtype=torch.bool)
    for b, parents in enumerate(c["trees"]):
        qs = int(c["start"][b])
        for i, way in enumerate(ways_of(parents)):
            pos[qs + i] = int(c["prefix"][b]) + len(way) - 1 + (0 if delta is None else int(delta[b]))
            known[qs + i] = True
    z = torch.polar(torch.ones((T, half), dtype=torch.float64), torch.outer(pos, inv_freq.double().cpu())).to(qkv.device)

    def one(h, gain):
        if gain is not None:
            h = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gain.double()
        y = torch.complex(h[..., :half].contiguous(), h[..., half:2 * half].contiguous()) * z[:, None]
        return torch.cat([y.real, y.imag, h[..., 2 * half:]], dim=-1) * known.to(h.device)[:, None, None]

    return one(x[:, :hq], gains[0]), one(x[:, hq:hq + hkv], gains[1]), x[:, hq + hkv:]


def slots_of_rows(c):
    """Slot of every row of the batch's trees, in row order (the trees' rows follow each other)."""
    out = []
    for b, parents in enumerate(c["trees"]):
        pl = int(c["prefix"][b])
        out += c["table"][int(c["req"][b]), pl:pl + len(parents)].tolist()
    return out

