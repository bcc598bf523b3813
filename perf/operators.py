"""One round of speculative decoding over the paged cache, operator by operator.

A draft is a tree of tokens per request: node 0 is the request's last token, every other node continues its parent.  The model
runs over all nodes at once.  Four operators do what a plain prompt pass cannot:

* ``prologue``   queries and keys of the nodes are normed per head and turned to the node's position (cached tokens + depth),
                 keys and values are appended to the request's slots;
* ``attention``  every node attends to the cached tokens, its ancestors and itself;
* ``verify``     walks each tree from its root with the target's filtered distribution: accepted nodes, and one more token;
* ``compact``    brings the cache rows of the accepted nodes together, in all layers.

A case is one call of one of them.  Head sizes, vocabularies and layer counts are those of the served models.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_EPS = 1e-6


def listed():
    return [
        # one user, a short chat and a small tree: the smallest call, latency alone
        _attention("attention-1x160-8", requests=1, context=160, nodes=8, heads=16, kv=8, dim=128, page=16),
        # a batch of the 8B model behind prompts of 2048 tokens, 32 nodes of 4 heads per kv head
        _attention("attention-8x2048-32", requests=8, context=2048, nodes=32, heads=32, kv=8, dim=128, page=16),
        # a serving batch of unlike lengths with slots given one at a time, odd trees
        _attention("attention-29x1900-17", requests=29, context=1900, spread=0.8, nodes=17, heads=32, kv=8, dim=128, page=1),
        # two long documents with wide heads (the hybrid's attention layers)
        _attention("attention-2x30000-48-d256", requests=2, context=30000, nodes=48, heads=8, kv=2, dim=256, page=16),
        # 8-bit cache, few kv heads
        _attention("attention-16x4096-24-e4m3", requests=16, context=4096, spread=0.3, nodes=24, heads=32, kv=4, dim=128, page=16,
                   cache="e4m3"),
        # the same round's prologue: one user; a full batch writing an 8-bit cache
        _prologue("prologue-1x8", requests=1, context=160, nodes=8, heads=16, kv=8, dim=128, page=16),
        _prologue("prologue-32x60-e4m3", requests=32, context=900, spread=0.5, nodes=60, heads=32, kv=8, dim=128, page=1, cache="e4m3"),
        # verification: one user, candidates that the draft ranked; a batch with the draft's own probabilities; a large batch
        _verify("verify-1x8", requests=1, nodes=8, vocab=151936, width=3, steps=5, draft=False),
        _verify("verify-8x16-sampled", requests=8, nodes=16, vocab=151936, width=3, steps=6, draft=True),
        _verify("verify-32x24", requests=32, nodes=24, vocab=128256, width=4, steps=6, draft=False),
        # the accepted rows of one user, and of a batch
        _compact("compact-1x8", requests=1, nodes=8, accepted=3, layers=28, kv=8, dim=128, page=16),
        _compact("compact-32x30", requests=32, nodes=30, accepted=6, layers=36, kv=8, dim=128, page=1),
    ]


def _named(name, case):
    return dict(case, name=name) if name else case


def _attention(name, *, requests, context, nodes, heads, kv, dim, page, spread=0.0, cache="same", dtype="bf16", window=0, cap=0.0, sink=False):
    return _named(name, dict(op="attention", requests=requests, context=context, spread=spread, nodes=nodes, heads=heads, kv=kv, dim=dim,
                             page=page, cache=cache, dtype=dtype, window=window, cap=cap, sink=sink))


def _prologue(name, *, requests, context, nodes, heads, kv, dim, page, spread=0.0, cache="same", dtype="bf16", rotated=None, norm=True):
    return _named(name, dict(op="prologue", requests=requests, context=context, spread=spread, nodes=nodes, heads=heads, kv=kv, dim=dim,
                             page=page, cache=cache, dtype=dtype, rotated=dim if rotated is None else rotated, norm=norm))


def _verify(name, *, requests, nodes, vocab, width, steps, draft, dtype="bf16"):
    return _named(name, dict(op="verify", requests=requests, nodes=nodes, vocab=vocab, width=width, steps=steps, draft=draft, dtype=dtype))


def _compact(name, *, requests, nodes, accepted, layers, kv, dim, page, cache="same", dtype="bf16"):
    return _named(name, dict(op="compact", requests=requests, nodes=nodes, accepted=accepted, layers=layers, kv=kv, dim=dim, page=page,
                             cache=cache, dtype=dtype))


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "prologue", "verify", "compact"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([1, 16])
    cache = rng.choice(["same", "same", "e4m3", "e5m2"])
    dim, kv, group = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    if op == "attention":
        requests, nodes = _log_int(rng, 1, 32), _log_int(rng, 1, 64)
        context = _log_int(rng, 1, min(30000, 60000 // requests, 60000 * 1024 // (requests * kv * dim * 2)))
        return _attention(None, requests=requests, context=context, spread=round(rng.uniform(0.0, 0.9), 2), nodes=nodes, heads=kv * group, kv=kv,
                          dim=dim, page=page, cache=cache, dtype=dtype, window=rng.choice([0, 0, 0, _log_int(rng, 2, 4000)]),
                          cap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.25)
    if op == "prologue":
        requests = _log_int(rng, 1, 32)
        return _prologue(None, requests=requests, context=_log_int(rng, 1, 1200), spread=round(rng.uniform(0.0, 0.9), 2),
                         nodes=_log_int(rng, 1, 60), heads=kv * group, kv=kv, dim=dim, page=page, cache=cache, dtype=dtype,
                         rotated=dim if dim < 256 else 64, norm=rng.random() < 0.6)
    if op == "verify":
        requests, nodes = _log_int(rng, 1, 32), _log_int(rng, 1, 24)
        return _verify(None, requests=requests, nodes=nodes, vocab=_log_int(rng, 1000, 151936), width=rng.randint(1, 4), steps=rng.randint(1, 7),
                       draft=requests * nodes <= 256 and rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    return _compact(None, requests=_log_int(rng, 1, 32), nodes=_log_int(rng, 2, 30), accepted=rng.randint(1, 6), layers=rng.randint(1, 36), kv=kv,
                    dim=dim, page=page, cache=cache, dtype=dtype)


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens and nodes of each request: spread evenly around the means, in an order that mixes them."""
    n, spread = case["requests"], case.get("spread", 0.0)
    at = [(((i * 7) % n if n % 7 else i) + 0.5) / n * 2 - 1 for i in range(n)]
    cached = [max(1, int(round(case.get("context", 40) * (1 + spread * a)))) for a in at]
    nodes = [max(1, case["nodes"] - (i % 3 if spread or case["op"] == "verify" else 0)) for i in range(n)]
    return cached, nodes


def _trees(nodes, seed, width=4, depth=8):
    """Parents of every request's nodes, -1 at the root: a node's parent is an earlier one with fewer than ``width`` children."""
    rng, out = random.Random(seed * 7919 + 11), []
    for n in nodes:
        parents, level, children = [-1], [0], [0]
        for _ in range(1, n):
            free = [j for j in range(len(parents)) if children[j] < width and level[j] + 1 < depth]
            p = rng.choice(free[:4]) if free else -1
            parents.append(p)
            level.append(level[p] + 1 if p >= 0 else 0)
            children.append(0)
            if p >= 0:
                children[p] += 1
        out.append(parents)
    return out


def _table(case, cached, nodes, rng):
    """(rows of the request table, number of slots): pages in the order that a used allocator gives them."""
    page, need = case["page"], [c + n for c, n in zip(cached, nodes)]
    pages = [-(-t // page) for t in need]
    order = list(range(1, sum(pages) + 1))
    if page == 1:
        rng.shuffle(order)
    else:       # runs of pages: what is freed together is given together
        runs = [order[i:i + 8] for i in range(0, len(order), 8)]
        rng.shuffle(runs)
        order = [p for r in runs for p in r]
    rows, at = [], 0
    for t, p in zip(need, pages):
        rows.append([order[at + i // page] * page + i % page for i in range(t)])
        at += p
    return rows, (sum(pages) + 1) * page


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1_000_003 + 17)
    cached, nodes = _lengths(case)
    total, batch = sum(nodes), case["requests"]
    starts = [sum(nodes[:i]) for i in range(batch)]
    trees = _trees(nodes, int(seed), case.get("width", 4), case.get("steps", 8))
    s = dict(case=case, parents=_ints([p for t in trees for p in t]), tree_lens=_ints(nodes), q_start=_ints(starts), most=max(nodes))
    act = torch.float32 if case["dtype"] == "fp32" else _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=act):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    if case["op"] == "verify":
        return _prepare_verify(case, s, trees, starts, normal, g)
    rows, slots = _table(case, cached, nodes, random.Random(int(seed) + 5))
    longest = max(len(r) for r in rows)
    order = list(range(batch))
    random.Random(int(seed) + 9).shuffle(order)        # the request table's rows are not the batch's
    table = torch.zeros((batch + 1, longest + 64), dtype=torch.int32)
    for b, r in enumerate(rows):
        table[order[b], :len(r)] = torch.tensor(r, dtype=torch.int32)
    store = act if case["cache"] == "same" else _DTYPES[case["cache"]]
    s.update(table=table.cuda(), req=_ints(order), prefix=_ints(cached), seq=_ints([c + n for c, n in zip(cached, nodes)]), longest=longest)
    kv, dim = case["kv"], case["dim"]
    if case["op"] == "compact":
        s["store"] = torch.stack([normal(2, kv, slots, dim, dtype=store) for _ in range(case["layers"])])
        picks, counts = _accepted(case, nodes, int(seed))
        s.update(path=_ints(picks), counts=_ints(counts))
        return s
    # head-major storage seen as [slots, heads, features]
    s["k_cache"] = normal(kv, slots, dim, dtype=store).transpose(0, 1)
    s["v_cache"] = normal(kv, slots, dim, dtype=store).transpose(0, 1)
    if case["op"] == "attention":
        s["q"] = normal(total, case["heads"], dim)
        s["sink"] = normal(case["heads"], dtype=torch.float32) if case["sink"] else None
        s["scale"] = dim ** -0.5
        return s
    s["qkv"] = normal(total, (case["heads"] + 2 * kv) * dim, std=1.5)
    s["gains"] = [(1 + normal(dim, std=0.2, dtype=torch.float32)).to(act) if case["norm"] else None for _ in range(2)]
    half = case["rotated"] // 2
    s["inv_freq"] = (1e6 ** -(torch.arange(half, dtype=torch.float64) / half)).float().cuda()
    return s


def _prepare_verify(case, s, trees, starts, normal, g):
    """Logits as a trained model's: a broad floor and some tokens far above it.  The draft is the target with noise; its tokens
    are drawn from its probabilities, or are its best ones in turn."""
    batch, vocab, total = case["requests"], case["vocab"], s["parents"].numel()
    logits = normal(total, vocab, std=1.5, dtype=torch.float32)
    peaks = torch.randint(0, vocab, (total, 24), generator=g, device="cuda")
    logits.scatter_(1, peaks, 11.0 + 2.5 * torch.randn((total, 24), generator=g, device="cuda"))
    parent_row, rank = [], []
    for t, at in zip(trees, starts):
        seen = {}
        for p in t:
            parent_row.append(at + max(0, p))
            rank.append(seen.get(p, 0) if p >= 0 else 0)
            seen[p] = seen.get(p, 0) + 1
    parent_row, rank = _ints(parent_row, torch.int64), _ints(rank, torch.int64)
    draft = (logits + 0.5 * torch.randn((total, vocab), generator=g, device="cuda")) / 0.8
    if case["draft"]:
        s["draft"] = torch.softmax(draft, dim=-1)
        s["tokens"] = torch.multinomial(s["draft"][parent_row], 1, generator=g)[:, 0]
    else:
        s["draft"] = None
        s["tokens"] = draft.topk(case["width"], dim=-1).indices[parent_row, rank.clamp(max=case["width"] - 1)]
    s["logits"] = logits.to(torch.float32 if case["dtype"] == "fp32" else _DTYPES[case["dtype"]])
    rng = random.Random(total * 31 + vocab)
    kinds = [dict(t=rng.choice([0.7, 0.8, 1.0]), k=rng.choice([0, 20, 50]), p=rng.choice([0.8, 0.95, 1.0]), m=rng.choice([0.0, 0.0, 0.05]))
             for _ in range(batch)]
    if batch > 3:
        kinds[2]["t"] = 0.0                             # one user wants the most likely tokens
    s.update(temperature=torch.tensor([k["t"] for k in kinds]).cuda(), top_k=_ints([k["k"] for k in kinds]),
             top_p=torch.tensor([k["p"] for k in kinds]).cuda(), min_p=torch.tensor([k["m"] for k in kinds]).cuda(),
             uniform=torch.rand((total,), generator=g, device="cuda"), uniform_final=torch.rand((batch,), generator=g, device="cuda"))
    return s


def _accepted(case, nodes, seed):
    """Accepted nodes of each request, the root first, and how many: later ones come from levels behind the first few nodes."""
    rng, picks, counts = random.Random(seed + 3), [], []
    for n in nodes:
        most = min(case["accepted"], n)
        behind = list(range(most, n))
        take = sorted(rng.sample(behind, min(len(behind), rng.randint(0, most - 1) if case["requests"] > 2 else most - 1)))
        path = [0] + take
        picks.append(path + [-1] * (case["accepted"] - len(path)))
        counts.append(len(path))
    return picks, counts


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"attention": _plain_attention, "prologue": _plain_prologue, "verify": _plain_verify, "compact": _plain_compact}[op](state)


def _own(op, s):
    from mllm_b200 import ops

    c = s["case"]
    if op == "attention":
        return ops.attention_tree(s["q"], s["k_cache"], s["v_cache"], s["table"], s["req"], s["seq"], s["prefix"], s["q_start"], s["parents"],
                                  s["scale"], window=c["window"] or None, logit_cap=c["cap"], sink=s["sink"])
    if op == "prologue":
        q = ops.tree_qk_norm_rope_kv_write(s["qkv"], *s["gains"], s["parents"], s["table"], s["req"], s["seq"], s["prefix"], s["q_start"],
                                           s["inv_freq"], s["k_cache"], s["v_cache"], c["heads"], c["kv"], c["dim"], _EPS)
        return q, s["k_cache"], s["v_cache"]
    if op == "verify":
        return ops.tree_speculative_sample(s["logits"], s["tokens"], s["parents"], s["tree_lens"], s["q_start"], s["temperature"], s["top_k"],
                                           s["top_p"], s["min_p"], s["uniform"], s["uniform_final"], c["steps"], draft_probs=s["draft"])
    ops.tree_kv_compact(s["store"], s["table"], s["req"], s["prefix"], s["path"], s["counts"])
    return s["store"]


def _row_of(s):
    """(request, node) of every row, [T] each."""
    t = torch.arange(s["parents"].numel(), device="cuda")
    b = (t[:, None] >= s["q_start"][None, :]).sum(1) - 1
    return b, t - s["q_start"].long()[b]


def _ancestors(s, b, j):
    """[requests, most, most] node i is on node j's way to the root, itself included, and the depths [requests, most]."""
    batch, most = s["tree_lens"].numel(), s["most"]
    step = torch.zeros((batch, most, most + 1), device="cuda")
    step[b, j, torch.where(s["parents"] < 0, most, s["parents"]).long()] = 1.0
    once = torch.eye(most, device="cuda") + step[:, :, :most]
    seen = torch.linalg.matrix_power(once, 8) > 0               # trees here have at most 8 levels
    return seen, seen.sum(-1) - 1


def _plain_attention(s):
    c, q, kv = s["case"], s["q"], s["case"]["kv"]
    b, j = _row_of(s)
    seen, depth = _ancestors(s, b, j)
    batch, most, longest = depth.shape[0], s["most"], s["longest"]
    qp = torch.zeros((batch, most, *q.shape[1:]), device="cuda")
    qp[b, j] = q.float()
    at = torch.arange(longest, device="cuda")
    slots = s["table"][s["req"].long()][:, :longest].long()
    keys, values = (t[slots].float().transpose(1, 2) for t in (s["k_cache"], s["v_cache"]))               # [B, kv, L, D]
    qp = qp.view(batch, most, kv, -1, c["dim"]).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, c["dim"])
    scores = (qp @ keys.transpose(-1, -2)) * s["scale"]
    scores = scores.view(batch, kv, -1, most, longest)
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    prefix = s["prefix"].long()
    node = at[None, :] - prefix[:, None]                                                                  # [B, L], negative: cached
    inside = (node >= 0) & (node < s["tree_lens"][:, None])
    node = node.clamp(0, most - 1)
    pos = torch.where(inside, prefix[:, None] + depth.gather(1, node), at[None, :])
    visible = torch.where(inside[:, None, :], seen.gather(2, node[:, None, :].expand(-1, most, -1)), (at[None, :] < prefix[:, None])[:, None, :])
    if c["window"]:
        visible = visible & (pos[:, None, :] > (prefix[:, None] + depth)[:, :, None] - c["window"])
    scores = torch.where(visible[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, kv, -1, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(scores - top)
    den = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        den = den + torch.exp(sink - top)
    out = (e.view(batch, kv, -1, longest) @ values).view(batch, kv, -1, most, c["dim"]) / den
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most, -1, c["dim"])[b, j].to(q.dtype)


def _plain_prologue(s):
    c, dtype = s["case"], s["qkv"].dtype
    b, j = _row_of(s)
    _, depth = _ancestors(s, b, j)
    pos = s["prefix"][b].double() + depth[b, j]
    heads = s["qkv"].float().view(-1, c["heads"] + 2 * c["kv"], c["dim"])
    q, k, v = heads.split([c["heads"], c["kv"], c["kv"]], dim=1)
    angle = pos[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, gain):
        if gain is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * gain.float()
        first, second, rest = x.split([c["rotated"] // 2, c["rotated"] // 2, c["dim"] - c["rotated"]], dim=-1)
        return torch.cat([first * cos - second * sin, second * cos + first * sin, rest], dim=-1)

    loc = s["table"][s["req"].long()[b], s["prefix"].long()[b] + j].long()
    s["k_cache"][loc] = turned(k, s["gains"][1]).to(s["k_cache"].dtype)
    s["v_cache"][loc] = v.to(s["v_cache"].dtype)
    return turned(q, s["gains"][0]).to(dtype), s["k_cache"], s["v_cache"]


def _filtered(logits, s):
    """The target's distribution in 64 bits (a token's border in the sum decides): the tokens that every filter keeps, ties included."""
    vocab = logits.shape[1]
    x, t = logits.double(), s["temperature"].double()[:, None]
    e = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(t <= 1e-6, 1.0, t))
    down = torch.sort(e, dim=-1, descending=True).values
    k, p = s["top_k"].long()[:, None], s["top_p"].double()[:, None]
    low = torch.where((k > 0) & (k < vocab), down.gather(1, (k - 1).clamp(0, vocab - 1)), 0.0)
    mass = torch.cumsum(down, -1)
    inside = (mass - down < p * mass[:, -1:]).sum(-1, keepdim=True).clamp(min=1)
    low = torch.maximum(low, torch.where(p < 1.0, down.gather(1, inside - 1), 0.0))
    low = torch.maximum(low, s["min_p"].double()[:, None])
    kept = torch.where(e >= low, e, 0.0)
    best = torch.zeros_like(e).scatter_(1, x.argmax(-1, keepdim=True), 1.0)
    kept = torch.where(t <= 1e-6, best, kept)
    return kept / kept.sum(-1, keepdim=True)


def _plain_verify(s):
    c, tokens, start = s["case"], s["tokens"].long(), s["q_start"].long()
    batch, most, steps = start.numel(), s["most"], c["steps"]
    b, j = _row_of(s)
    parent = torch.full((batch, most), -2, device="cuda")
    parent[b, j] = s["parents"].long()
    node, alive = torch.zeros_like(start), s["tree_lens"] > 0
    path, out = torch.full((batch, steps), -1, device="cuda", dtype=torch.int32), torch.full((batch, steps), -1, device="cuda")
    counts, all_rows = torch.zeros_like(s["tree_lens"]), torch.arange(batch, device="cuda")
    # a walk: what a step looks at is known when the step before is done
    for step in range(steps):
        row = start + node
        p = _filtered(s["logits"][row], s)
        path[:, step] = torch.where(alive, node, -1).to(torch.int32)
        counts += alive
        child_of = (parent == node[:, None]) & alive[:, None]
        rank = torch.cumsum(child_of, 1) * child_of
        taken = torch.full_like(node, -1)
        for turn in range(c["width"] if step + 1 < steps else 0):
            here = rank == turn + 1
            child = here.int().argmax(1)
            token = tokens[start + child][:, None]
            asked = here.any(1) & (taken < 0)
            q = torch.zeros_like(p).scatter_(1, token, 1.0) if s["draft"] is None else s["draft"][row].double()
            taken = torch.where(asked & ((s["uniform"][start + child].double()[:, None] * q.gather(1, token)) < p.gather(1, token))[:, 0], child, taken)
            left = (p - q).clamp(min=0.0)
            if s["draft"] is None:
                left = p * (q == 0)
            rest = left.sum(-1, keepdim=True)
            p = torch.where((asked & (taken < 0))[:, None] & (rest > 0), left / rest, p)
        sums = torch.cumsum(p, -1)
        drawn = (sums <= s["uniform_final"].double()[:, None] * sums[:, -1:]).sum(-1).clamp(max=c["vocab"] - 1)
        out[:, step] = torch.where(alive, torch.where(taken >= 0, tokens[start + taken.clamp(min=0)], drawn), -1)
        alive = alive & (taken >= 0)
        node = torch.where(alive, taken, node)
    return path, out, counts


def _plain_compact(s):
    path = s["path"].long()
    row = s["table"][s["req"].long()].long()
    first = s["prefix"].long()[:, None]
    column = torch.arange(path.shape[1], device="cuda")[None, :]
    column = torch.where(column < s["counts"][:, None], column, 0)
    source = torch.where(column > 0, path, path[:, :1])
    rows = s["store"][:, :, :, row.gather(1, first + source).flatten()]
    s["store"][:, :, :, row.gather(1, first + column).flatten()] = rows
    return s["store"]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    cached, nodes = _lengths(case)
    total, item = sum(nodes), 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "verify":
        # per request the root's row and one row behind it, with the draft's where there is one
        rows = 2 * case["requests"] if case["steps"] > 1 and case["nodes"] > 1 else case["requests"]
        return dict(bytes=rows * case["vocab"] * (item + 4 * case["draft"]), flops=rows * case["vocab"] * 8)
    kept = item if case["cache"] == "same" else 1
    width = case["kv"] * case["dim"]
    if case["op"] == "attention":
        seen = [min(c, case["window"]) if case["window"] else c for c in cached]
        keys = sum(s + n for s, n in zip(seen, nodes))
        return dict(bytes=keys * width * 2 * kept + 2 * total * case["heads"] * case["dim"] * item,
                    flops=sum(4 * n * (s + min(n, 4)) for s, n in zip(seen, nodes)) * case["heads"] * case["dim"])
    if case["op"] == "prologue":
        rows = total * case["dim"]
        return dict(bytes=rows * (2 * case["heads"] * item + 2 * case["kv"] * (item + kept)), flops=rows * (case["heads"] + case["kv"]) * 8)
    moved = sum(count - 1 for count in _accepted(case, nodes, 0)[1])
    return dict(bytes=max(1, moved) * case["layers"] * 4 * width * kept, flops=0)


# ---------------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits, one request at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    parents, first, count = s["parents"].tolist(), s["q_start"].tolist(), s["tree_lens"].tolist()
    if case["op"] == "verify":
        return None                                    # node and token numbers only
    table, prefix = s["table"].cpu(), s["prefix"].tolist()
    chains = []
    for b, n in enumerate(count):
        ways = []
        for i in range(n):
            up = parents[first[b] + i]
            ways.append(([] if up < 0 else ways[up]) + [i])
        chains.append(ways)
    slots = [table[r, :prefix[b] + count[b]].long().cuda() for b, r in enumerate(s["req"].tolist())]
    if case["op"] == "compact":
        store = s["store"].double() if s["store"].numel() < 2 ** 29 else None
        if store is None:
            return None
        for b, (nodes, n) in enumerate(zip(s["path"].tolist(), s["counts"].tolist())):
            for i in range(n):
                store[:, :, :, slots[b][prefix[b] + i]] = store[:, :, :, slots[b][prefix[b] + nodes[i]]]
        return store
    dim, kv = case["dim"], case["kv"]
    if case["op"] == "attention":
        outs = []
        for b, n in enumerate(count):
            k, v = (t[slots[b]].double() for t in (s["k_cache"], s["v_cache"]))
            q = s["q"][first[b]:first[b] + n].double().view(n, kv, -1, dim)
            sc = torch.einsum("nkgd,lkd->kgnl", q, k) * s["scale"]
            if case["cap"]:
                sc = torch.tanh(sc / case["cap"]) * case["cap"]
            seen = torch.zeros((n, prefix[b] + n), dtype=torch.bool)
            for i, way in enumerate(chains[b]):
                here = prefix[b] + len(way) - 1
                low = max(0, here - case["window"] + 1) if case["window"] else 0
                seen[i, low:prefix[b]] = True
                for up, node in enumerate(way):
                    seen[i, prefix[b] + node] = prefix[b] + up >= low
            sc = sc.masked_fill(~seen.cuda(), -math.inf)
            if s["sink"] is not None:
                sc = torch.cat([sc, s["sink"].double().view(kv, -1, 1, 1).expand(-1, -1, n, 1)], dim=-1)
            w = torch.softmax(sc, dim=-1)[..., :prefix[b] + n]
            outs.append(torch.einsum("kgnl,lkd->nkgd", w, v).reshape(n, -1, dim))
        return torch.cat(outs)
    rows = s["qkv"].double().view(-1, case["heads"] + 2 * kv, dim)
    half = case["rotated"] // 2
    pos = torch.tensor([prefix[b] + len(w) - 1 for b, ways in enumerate(chains) for w in ways], dtype=torch.float64).cuda()
    turn = torch.polar(torch.ones((pos.numel(), half), dtype=torch.float64, device="cuda"), torch.outer(pos, s["inv_freq"].double()))

    def one(x, gain):
        if gain is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / dim + _EPS).sqrt() * gain.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], dim=-1)

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    for b, n in enumerate(count):
        here, own_slots = slice(first[b], first[b] + n), slots[b][prefix[b]:]
        k_cache[own_slots] = one(rows[:, case["heads"]:case["heads"] + kv], s["gains"][1])[here]
        v_cache[own_slots] = rows[here, case["heads"] + kv:]
    return one(rows[:, :case["heads"]], s["gains"][0]), k_cache, v_cache
