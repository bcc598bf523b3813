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



class Round:
    """A tiny model that runs prompts and drafted trees, and the same tokens as plain prompts for comparison."""

    def __init__(self, preset, device, dtype, kv_cache_dtype="auto"):
        from mllm_b200.configs import ServerConfig
        from mllm_b200.executor import ModelRunner

        self.mr = ModelRunner(ServerConfig(model_path=f"preset:{preset}", dtype=dtype, max_running_requests=24, max_total_tokens=4096),
                              kv_cache_dtype=kv_cache_dtype, device=device)
        self.mr.initialize()
        self.dev = torch.device(device)

    def _alloc(self, n):
        return self.mr.token_to_kv_pool_allocator.alloc(n)

    def prompt(self, ids):
        """Runs a prompt; (request row, logits of its last token)."""
        mr = self.mr
        row = mr.req_to_token_pool.alloc(1)[0]
        loc = self._alloc(len(ids))
        mr.req_to_token_pool.req_to_token[row, :len(ids)] = loc.to(torch.int32)
        one = lambda x: torch.tensor([x], dtype=torch.int32, device=self.dev)  # noqa: E731
        fb = mr.prepare_forward_batch_extend(torch.tensor(ids, device=self.dev), one(row), one(len(ids)), one(len(ids)), one(0), loc, [len(ids)], [0])
        return row, mr.forward(fb).next_token_logits[0]

    def free(self, row):
        self.mr.req_to_token_pool.free(row)

    def plain(self, ids):
        """Logits behind `ids` as a prompt of its own."""
        row, logits = self.prompt(ids)
        self.free(row)
        return logits

    def tree(self, rows, lens, tokens, trees):
        """Runs a tree per request behind its cached tokens; the logits of all nodes."""
        mr = self.mr
        for row, n, t in zip(rows, lens, trees):
            mr.req_to_token_pool.req_to_token[row, n:n + len(t)] = self._alloc(len(t)).to(torch.int32)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        fb = mr.prepare_forward_batch_tree(torch.tensor([x for t in tokens for x in t], device=self.dev), ints([p for t in trees for p in t]),
                                           ints(rows), [len(t) for t in trees], list(lens))
        return fb, mr.forward(fb).next_token_logits

    def check(self, close):
        """A round of speculative decoding: logits of nodes, greedy verification, accepted rows, the next step."""
        from mllm_b200 import ops

        g = random.Random(5)
        vocab = self.mr.vocab_size
        prompts = [[g.randrange(vocab) for _ in range(n)] for n in (19, 70, 1)]
        rows, seen = [], []
        for p in prompts:
            row, logits = self.prompt(p)
            rows.append(row)
            seen.append(p + [int(logits.float().argmax())])             # the root: the request's last token
        for _ in range(2):                                              # two rounds in a row
            trees = [[-1, 0, 0, 1, 1, 3, 2], [-1, 0, 1, 2, 0, 4, 3, 3], [-1, 0, 0]]
            tokens = [[s[-1]] + [g.randrange(vocab) for _ in t[1:]] for s, t in zip(seen, trees)]
            # one way through each tree is what the model itself would say, for a while
            ways = [[2, 6], [1, 2, 3], []]
            for s, t, tok, way in zip(seen, trees, tokens, ways):
                said = list(s)
                for node in way:
                    said.append(int(self.plain(said).float().argmax()))
                    tok[node] = said[-1]
            lens = [len(s) - 1 for s in seen]
            fb, logits = self.tree(rows, lens, tokens, trees)
            at = 0
            for s, t, tok in zip(seen, trees, tokens):
                for j, way in enumerate(ways_of(t)):
                    close(logits[at + j], self.plain(s[:-1] + [tok[i] for i in way]))
                at += len(t)
            B, T = len(rows), logits.shape[0]
            f = lambda x, n: torch.full((n,), x, device=self.dev)  # noqa: E731
            path, out, counts = ops.tree_speculative_sample(
                logits, torch.tensor([x for t in tokens for x in t], device=self.dev), fb.tree_parents, fb.extend_seq_lens, fb.extend_start_loc,
                f(0.0, B), torch.zeros(B, dtype=torch.int32, device=self.dev), f(1.0, B), None, f(0.5, T), f(0.5, B), 5)
            self.mr.token_to_kv_pool.keep_accepted(self.mr.req_to_token_pool.req_to_token, fb.req_pool_indices, fb.extend_prefix_lens, path, counts)
            for b, way in enumerate(ways):
                n = int(counts[b])
                assert path[b, :len(way) + 1].tolist() == [0] + way[:n - 1] + [-1] * (len(way) + 1 - n) or n >= len(way) + 1
                assert out[b, :n - 1].tolist() == [tokens[b][i] for i in path[b, 1:n].tolist()]
                assert n >= len(way) + 1, "greedy verification takes what the model itself would say"
                seen[b] = seen[b] + out[b, :n].tolist()
        # behind it the requests go on as if they had been decoded token by token
        lens = [len(s) - 1 for s in seen]
        _, logits = self.tree(rows, lens, [[s[-1]] for s in seen], [[-1]] * len(seen))
        for b, s in enumerate(seen):
            close(logits[b], self.plain(s))
        ops.check_status()
