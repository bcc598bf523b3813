"""Eviction from the paged cache by accumulated attention weight, operator by operator.

A request's cache may be shortened: every kv head of every layer keeps the cached tokens that were attended to most, and the rows of the
kept ones move to the front, in their order.  Keys are cached with their positions turned in, so attention over what is left goes on as before.

* ``decode``   attention of one new token per request that also adds the weights of a group's heads to the cached tokens' sums;
* ``prompt``   the weights that the last queries of each prompt (or all of them) give to the cached tokens;
* ``select``   per layer, request and kv head: the last tokens, the first ones, and those of the largest sums;
* ``evict``    the kept rows of keys and values, and their sums, in all layers.

A case is one call of one of them.  Head sizes, layer counts and pages are those of the served models.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def listed():
    return [
        # one user, a short chat: the smallest step, latency alone
        _decode("decode-1x160", requests=1, context=160, heads=16, kv=8, dim=128, page=16),
        # a serving batch of unlike lengths whose slots were given one at a time
        _decode("decode-29x1900-fp16", requests=29, context=1900, spread=0.8, heads=32, kv=8, dim=128, page=1, dtype="fp16"),
        # long documents with wide heads (the hybrid's attention layers); old weights fade
        _decode("decode-3x30000-d256", requests=3, context=30000, spread=0.1, heads=8, kv=2, dim=256, page=16, decay=0.98),
        # a large batch over an 8-bit cache, few kv heads
        _decode("decode-32x4096-e4m3", requests=32, context=4096, spread=0.3, heads=32, kv=4, dim=128, page=16, cache="e4m3"),
        # the prompt of one user, looked at by its last 16 tokens
        _prompt("prompt-1x160-16", requests=1, context=160, new=160, last=16, heads=16, kv=8, dim=128, page=16),
        # a batch of prompts of the 8B model behind its last 32 tokens
        _prompt("prompt-8x2048-32", requests=8, context=2048, new=2048, last=32, heads=32, kv=8, dim=128, page=16),
        # the last chunk of a long document
        _prompt("prompt-1x32000-64", requests=1, context=32000, new=2000, last=64, heads=32, kv=8, dim=128, page=16),
        # every token of two prompts counts; odd lengths, slots one at a time
        _prompt("prompt-2x1500-all", requests=2, context=1500, new=1500, last=0, spread=0.3, heads=32, kv=8, dim=128, page=1, add=True),
        # one user's cache of all layers, halved
        _select("select-28x1x1200", layers=28, requests=1, context=1200, kv=8, keep=0.43, pool=1),
        # a batch of long prompts behind their last tokens: a quarter stays
        _select("select-36x8x8192", layers=36, requests=8, context=8192, spread=0.2, kv=8, keep=0.25, pool=7),
        # the kept rows of one user, and of a batch whose slots were given one at a time
        _evict("evict-28x1x1200", layers=28, requests=1, context=1200, kv=8, dim=128, keep=0.43, page=16),
        _evict("evict-36x4x4000", layers=36, requests=4, context=4000, spread=0.4, kv=8, dim=128, keep=0.25, page=1),
    ]


def _named(name, case):
    return dict(case, name=name) if name else case


def _decode(name, *, requests, context, heads, kv, dim, page, spread=0.0, cache="same", dtype="bf16", decay=1.0, cap=0.0, sink=False):
    return _named(name, dict(op="decode", requests=requests, context=context, spread=spread, heads=heads, kv=kv, dim=dim, page=page,
                             cache=cache, dtype=dtype, decay=decay, cap=cap, sink=sink))


def _prompt(name, *, requests, context, new, last, heads, kv, dim, page, spread=0.0, cache="same", dtype="bf16", add=False, cap=0.0, sink=False):
    return _named(name, dict(op="prompt", requests=requests, context=context, new=new, last=last, spread=spread, heads=heads, kv=kv, dim=dim,
                             page=page, cache=cache, dtype=dtype, add=add, cap=cap, sink=sink))


def _select(name, *, layers, requests, context, kv, keep, pool, spread=0.0, first=4, recent=32):
    return _named(name, dict(op="select", layers=layers, requests=requests, context=context, spread=spread, kv=kv, keep=keep, pool=pool,
                             first=first, recent=recent))


def _evict(name, *, layers, requests, context, kv, dim, keep, page, spread=0.0, cache="same", dtype="bf16"):
    return _named(name, dict(op="evict", layers=layers, requests=requests, context=context, spread=spread, kv=kv, dim=dim, keep=keep, page=page,
                             cache=cache, dtype=dtype))


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "select", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([1, 16])
    cache = rng.choice(["same", "same", "e4m3", "e5m2"])
    dim, kv, group = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    spread = round(rng.uniform(0.0, 0.9), 2)
    if op == "decode":
        requests = _log_int(rng, 1, 64)
        context = _log_int(rng, 1, min(30000, 90000 // requests, 52000 * 1024 // (requests * kv * dim)))
        return _decode(None, requests=requests, context=context, spread=spread, heads=kv * group, kv=kv, dim=dim, page=page, cache=cache,
                       dtype=dtype, decay=rng.choice([1.0, 1.0, 0.9]), cap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.25)
    if op == "prompt":
        requests, last = _log_int(rng, 1, 16), rng.choice([1, 8, 16, 32, 64, 100, 0])
        width = kv * group * dim
        if last == 0:
            context = _log_int(rng, 1, min(3000, math.isqrt(14_000_000_000 // (requests * width))))
        else:
            context = _log_int(rng, 1, min(32000 // requests, 20000 * 1024 // (requests * kv * dim), 8_000_000_000 // (requests * last * width)))
        return _prompt(None, requests=requests, context=context, new=context if last == 0 or rng.random() < 0.5 else min(context, 500), last=last,
                       spread=spread, heads=kv * group, kv=kv, dim=dim, page=page, cache=cache, dtype=dtype, add=rng.random() < 0.3,
                       cap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.25)
    layers, requests = rng.randint(1, 36), _log_int(rng, 1, 8)
    if op == "select":
        context = _log_int(rng, 1, min(30000, 11_500_000 // (layers * requests * kv)))
        return _select(None, layers=layers, requests=requests, context=context, spread=spread, kv=kv, keep=round(rng.uniform(0.05, 1.0), 2),
                       pool=rng.choice([1, 1, 5, 7, 13]), first=rng.choice([0, 4, 9]), recent=rng.choice([0, 1, 32, 64]))
    context = _log_int(rng, 1, min(30000, 140_000_000 // (layers * requests * kv * dim)))
    return _evict(None, layers=layers, requests=requests, context=context, spread=spread, kv=kv, dim=dim, keep=round(rng.uniform(0.05, 1.0), 2),
                  page=page, cache=cache, dtype=dtype)


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens of each request, the new ones included: spread evenly around the mean, in an order that mixes them."""
    n, spread = case["requests"], case["spread"]
    at = [(((i * 7) % n if n % 7 else i) + 0.5) / n * 2 - 1 for i in range(n)]
    return [max(1, int(round(case["context"] * (1 + spread * a)))) for a in at]


def _new(case):
    """New tokens of each prompt; what stands in front of them was cached before."""
    return [n if case["new"] == case["context"] else min(n, case["new"]) for n in _lengths(case)]


def _observed(case):
    return [min(n, case["last"]) if case["last"] else n for n in _new(case)]


def _budgets(case):
    return [max(1, int(n * case["keep"])) for n in _lengths(case)]


def _table(case, lens, rng):
    """(rows of the request table, number of slots): pages in the order that a used allocator gives them."""
    page = case["page"]
    pages = [-(-t // page) for t in lens]
    order = list(range(1, sum(pages) + 1))
    if page == 1:
        rng.shuffle(order)
    else:       # runs of pages: what is freed together is given together
        runs = [order[i:i + 8] for i in range(0, len(order), 8)]
        rng.shuffle(runs)
        order = [p for r in runs for p in r]
    rows, at = [], 0
    for t, p in zip(lens, pages):
        rows.append([order[at + i // page] * page + i % page for i in range(t)])
        at += p
    return rows, (sum(pages) + 1) * page


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1_000_003 + 29)
    lens, batch, kv = _lengths(case), case["requests"], case["kv"]
    longest = max(lens)
    room = longest + 64                                 # what the request table and the sums have per request
    order = list(range(batch))
    random.Random(int(seed) + 9).shuffle(order)         # the request table's rows are not the batch's
    s = dict(case=case, req=_ints(order), seq=_ints(lens), longest=longest)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    def sums(*shape):       # of a cache in use: a few tokens have most of the weight, some have none at all
        x = torch.exp(normal(*shape, std=2.0) - 3.0)
        return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.05, 0.0, x)

    if case["op"] == "select":
        s.update(sums=sums(case["layers"], batch + 1, kv, room), budgets=_ints(_budgets(case)), width=max(_budgets(case)))
        return s
    rows, slots = _table(case, lens, random.Random(int(seed) + 5))
    table = torch.zeros((batch + 1, room), dtype=torch.int32)
    for b, r in enumerate(rows):
        table[order[b], :len(r)] = torch.tensor(r, dtype=torch.int32)
    act, dim = _DTYPES[case["dtype"]], case["dim"]
    store = act if case["cache"] == "same" else _DTYPES[case["cache"]]
    s["table"] = table.cuda()
    if case["op"] == "evict":
        s["store"] = torch.empty((case["layers"], 2, kv, slots, dim), dtype=store, device="cuda")
        for layer in s["store"]:
            layer.copy_(normal(2, kv, slots, dim))
        s["sums"] = sums(case["layers"], batch + 1, kv, room)
        budgets = _budgets(case)
        s["counts"] = _ints(budgets)
        s["keep"] = torch.full((case["layers"], batch, kv, max(budgets)), -1, dtype=torch.int32, device="cuda")
        for b, (n, k) in enumerate(zip(lens, budgets)):     # the first tokens, the last ones, and others between
            rank = torch.rand((case["layers"], kv, n), generator=g, device="cuda")
            rank[..., :4], rank[..., max(0, n - 32):] = 2.0, 3.0
            s["keep"][:, b, :, :k] = rank.topk(k, dim=-1).indices.sort(dim=-1).values.to(torch.int32)
        return s
    # head-major storage seen as [slots, heads, features].  Some tokens are looked at far more than others: their keys lie along the
    # direction that queries share
    along = normal(kv, 1, dim)
    pull = torch.rand((kv, slots, 1), generator=g, device="cuda").clamp_(min=1e-6).log_().neg_().mul_(0.35)
    s["k_cache"] = normal(kv, slots, dim).addcmul_(along, pull).to(store).transpose(0, 1)
    total = batch if case["op"] == "decode" else sum(_new(case))
    s["q"] = (normal(total, kv, case["heads"] // kv, dim) + 0.5 * along).view(total, case["heads"], dim).to(act)
    s["sink"] = normal(case["heads"]) if case["sink"] else None
    s["scale"] = dim ** -0.5
    s["sums"] = sums(batch + 1, kv, room)
    if case["op"] == "decode":
        s["v_cache"] = normal(kv, slots, dim, dtype=store).transpose(0, 1)
        return s
    new = _new(case)
    s.update(prefix=_ints([n - m for n, m in zip(lens, new)]), start=_ints([sum(new[:i]) for i in range(batch)]), most=max(_observed(case)))
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"decode": _plain_decode, "prompt": _plain_prompt, "select": _plain_select, "evict": _plain_evict}[op](state)


def _own(op, s):
    from mllm_b200 import ops

    c = s["case"]
    if op == "decode":
        out = ops.attention_decode_weights(s["q"], s["k_cache"], s["v_cache"], s["table"], s["req"], s["seq"], s["scale"], s["sums"],
                                           decay=c["decay"], logit_cap=c["cap"], sink=s["sink"])
        return out, s["sums"]
    if op == "prompt":
        ops.attention_prefill_weights(s["q"], s["k_cache"], s["table"], s["req"], s["seq"], s["prefix"], s["start"], s["scale"], s["sums"],
                                      last=c["last"], add=c["add"], logit_cap=c["cap"], sink=s["sink"])
        return s["sums"]
    if op == "select":
        return ops.cache_select(s["sums"], s["req"], s["seq"], s["budgets"], s["width"], first=c["first"], recent=c["recent"], pool=c["pool"])
    ops.cache_evict(s["store"], s["sums"], s["table"], s["req"], s["keep"], s["counts"])
    return s["store"], s["sums"]


def _weights(scores, visible, s):
    """Softmax over the last axis of scaled scores [B, kv, group, .., L], with the soft cap and the sink."""
    if s["case"]["cap"]:
        scores = s["case"]["cap"] * torch.tanh(scores / s["case"]["cap"])
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, s["case"]["kv"], -1, *[1] * (scores.dim() - 3))
        top = torch.maximum(top, sink)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    den = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        den = den + torch.exp(sink - top)
    return torch.where(den > 0, e / den, 0.0)


def _cached(s, name):
    """[B, kv, L, D] in 32 bits."""
    slots = s["table"][s["req"].long()][:, :s["longest"]].long()
    return s[name][slots].float().transpose(1, 2)


def _plain_decode(s):
    c, req = s["case"], s["req"].long()
    at, seq = torch.arange(s["longest"], device="cuda"), s["seq"].long()
    q = s["q"].float().view(c["requests"], c["kv"], -1, c["dim"])
    visible = (at < seq[:, None])[:, None, None]
    w = _weights((q @ _cached(s, "k_cache").transpose(-1, -2)) * s["scale"], visible, s)
    old = s["sums"][req][:, :, :s["longest"]]
    grown = torch.where((at < seq[:, None] - 1)[:, None], c["decay"] * old, 0.0) + w.sum(2)
    s["sums"][req, :, :s["longest"]] = torch.where(visible[:, :, 0], grown, old)
    return (w @ _cached(s, "v_cache")).view(s["q"].shape).to(s["q"].dtype), s["sums"]


def _plain_prompt(s):
    c, req, most = s["case"], s["req"].long(), s["most"]
    at, seq = torch.arange(s["longest"], device="cuda"), s["seq"].long()
    new = seq - s["prefix"]
    look = torch.clamp(new, max=c["last"]) if c["last"] else new
    nth = torch.arange(most, device="cuda")
    row = torch.where(nth < look[:, None], s["start"][:, None] + (new - look)[:, None] + nth, 0)           # [B, most]
    q = s["q"][row].float().view(c["requests"], most, c["kv"], -1, c["dim"]).permute(0, 2, 3, 1, 4)        # [B, kv, group, most, D]
    scores = (q.reshape(c["requests"], c["kv"], -1, c["dim"]) @ _cached(s, "k_cache").transpose(-1, -2)) * s["scale"]
    place = (seq - look)[:, None] + nth                                                                    # of the queries among the tokens
    visible = (at <= place[:, :, None]) & (nth < look[:, None])[:, :, None]
    w = _weights(scores.view(c["requests"], c["kv"], -1, most, s["longest"]), visible[:, None, None], s).sum((2, 3))
    old = s["sums"][req][:, :, :s["longest"]]
    grown = w + torch.where((at < s["prefix"][:, None])[:, None], old, 0.0) if c["add"] else w
    s["sums"][req, :, :s["longest"]] = torch.where((at < seq[:, None])[:, None], grown, old)
    return s["sums"]


def _plain_select(s):
    c, at = s["case"], torch.arange(s["longest"], device="cuda")
    seq, counts = s["seq"].long()[:, None], torch.minimum(s["seq"], s["budgets"])
    score = torch.where((at < seq)[:, None], s["sums"][:, s["req"].long()][..., :s["longest"]], -math.inf)      # [layers, B, kv, L]
    half = c["pool"] // 2
    score = torch.nn.functional.pad(score, (half, half), value=-math.inf).unfold(-1, c["pool"], 1).amax(-1)
    count = counts.long()[:, None]
    last = count.clamp(max=c["recent"])
    first = (count - last).clamp(max=c["first"])
    always = (at >= seq - last) & (at < seq) | (at < first)
    # in the order of score, then those that stay in front, then those behind the request's last token at the end
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    kind = torch.where(at >= seq, 2, torch.where(always, 0, 1))[None, :, None].expand_as(order)
    order = order.gather(-1, torch.sort(kind.gather(-1, order), dim=-1, stable=True).indices)
    inside = torch.arange(s["width"], device="cuda") < count
    kept = torch.where(inside[:, None], order[..., :s["width"]], s["longest"]).sort(dim=-1).values
    return torch.where(inside[:, None], kept, -1).to(torch.int32), counts


def _plain_evict(s):
    batch, kv, width = s["keep"].shape[1:]
    req, at = s["req"].long()[:, None, None], torch.arange(width, device="cuda")
    table = s["table"].long()
    to = torch.where(at < s["counts"][:, None], at, 0)[:, None]                                            # behind the kept ones: the first again
    source = torch.where((at < s["counts"][:, None])[:, None], s["keep"], s["keep"][..., :1]).long()       # [layers, B, kv, width]
    head = torch.arange(kv, device="cuda")[:, None]
    to_slot = table[req, to]                                                                               # [B, 1, width]
    from_slot = table[req, source]
    layer = torch.arange(source.shape[0], device="cuda")[:, None, None, None]
    for_all = to_slot.expand(batch, kv, width)
    for tensor in (0, 1):
        s["store"][layer, tensor, head, for_all] = s["store"][layer, tensor, head, from_slot]
    s["sums"][layer, req, head, to] = s["sums"][layer, req, head, source]
    return s["store"], s["sums"]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    lens, kv = _lengths(case), case["kv"]
    total = sum(lens)
    if case["op"] == "select":
        lists = case["layers"] * kv
        return dict(bytes=4 * lists * (total + sum(_budgets(case))), flops=lists * total)
    item = 2 if case["cache"] == "same" else 1
    if case["op"] == "evict":
        moved = sum(max(1, k - 4) for k in _budgets(case))          # the first tokens stay where they are
        return dict(bytes=case["layers"] * kv * moved * (4 * case["dim"] * item + 12), flops=0)
    heads, dim = case["heads"], case["dim"]
    if case["op"] == "decode":
        return dict(bytes=total * kv * (2 * dim * item + 8) + 4 * case["requests"] * heads * dim, flops=4 * total * heads * dim)
    look = _observed(case)
    seen = sum(w * n - w * (w - 1) // 2 for w, n in zip(look, lens))
    return dict(bytes=total * kv * (dim * item + 4) + 2 * sum(look) * heads * dim, flops=2 * seen * heads * dim)


# ---------------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits, one request at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "select":
        return None                                     # token numbers only
    s = prepare(case, seed)
    table, lens, req = s["table"].cpu(), s["seq"].tolist(), s["req"].tolist()
    slots = [table[r, :n].long().cuda() for r, n in zip(req, lens)]
    total = s["sums"].double()
    if case["op"] == "evict":
        if s["store"].numel() > 2 ** 29:
            return None
        old, store = s["sums"].double(), s["store"].double()
        for b, count in enumerate(s["counts"].tolist()):
            for layer in range(case["layers"]):
                for head in range(case["kv"]):
                    kept = s["keep"][layer, b, head, :count].long()
                    for tensor in (0, 1):
                        store[layer, tensor, head, slots[b][:count]] = store[layer, tensor, head, slots[b][kept]]
                    total[layer, req[b], head, :count] = old[layer, req[b], head, kept]
        return store, total
    kv, dim, outs = case["kv"], case["dim"], []
    new = _new(case) if case["op"] == "prompt" else [1] * len(lens)
    look = _observed(case) if case["op"] == "prompt" else [1] * len(lens)
    for b, n in enumerate(lens):
        end = sum(new[:b + 1])
        q = s["q"][end - look[b]:end].double().view(look[b], kv, -1, dim)
        keys = s["k_cache"][slots[b]].double()
        values = s["v_cache"][slots[b]].double() if case["op"] == "decode" else None
        weights = torch.zeros((kv, n), dtype=torch.float64, device="cuda")
        for first in range(0, look[b], 256):            # some queries at a time
            part = q[first:first + 256]
            sc = torch.einsum("wkgd,lkd->kgwl", part, keys) * s["scale"]
            if case["cap"]:
                sc = torch.tanh(sc / case["cap"]) * case["cap"]
            place = n - look[b] + first + torch.arange(part.shape[0], device="cuda")
            sc = sc.masked_fill(torch.arange(n, device="cuda") > place[:, None], -math.inf)
            if s["sink"] is not None:
                sc = torch.cat([sc, s["sink"].double().view(kv, -1, 1, 1).expand(-1, -1, part.shape[0], 1)], dim=-1)
            p = torch.softmax(sc, dim=-1)[..., :n]
            weights += p.sum((1, 2))
            if values is not None:
                outs.append(torch.einsum("kgwl,lkd->wkgd", p, values).reshape(1, -1, dim))
        before = n - 1 if case["op"] == "decode" else n - new[b] if case["add"] else 0
        weights[:, :before] += case.get("decay", 1.0) * total[req[b], :, :before]
        total[req[b], :, :n] = weights
    return (torch.cat(outs), total) if case["op"] == "decode" else total
