"""Batches of cached requests and what their weights, outputs and sums are in 64 bits, with bounds on the kernels' roundings."""
import random

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}      # half a step, relative


def cached_batch(lens, hq, hkv, D, dtype=torch.bfloat16, cache=None, page=1, seed=0, new=None, layers=0, room=None, extra_rows=1, device="cuda"):
    """Requests of ``lens`` cached tokens in a paged cache, table rows in another order than the batch.  ``new``: new rows per request (prompts);
    None: one query per request.  ``layers``: storage of that many layers instead of one pair of caches."""
    g = torch.Generator().manual_seed(seed + 1)
    rng = random.Random(seed)
    pages = [-(-n // page) for n in lens]
    order = list(range(1, sum(pages) + 1))
    rng.shuffle(order)
    rows = list(range(len(lens) + extra_rows))
    rng.shuffle(rows)
    room = room or max([1, *lens]) + 5
    table = torch.zeros((len(lens) + extra_rows, room), dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[rows[b], :n] = torch.tensor([order[at + i // page] * page + i % page for i in range(n)], dtype=torch.int32)
        at += pages[b]
    slots = (sum(pages) + 1) * page
    store = cache or dtype

    def ints(x):
        return torch.tensor(x, dtype=torch.int32).to(device)

    c = dict(table=table.to(device), req=ints(rows[:len(lens)]), seq=ints(list(lens)), scale=D ** -0.5, lens=list(lens), hkv=hkv)
    if layers:
        c["store"] = torch.randn((layers, 2, hkv, slots, D), generator=g).to(store).to(device)
        c["sums"] = torch.rand((layers, len(rows), hkv, room), generator=g).to(device)
        return c
    c["k"] = torch.randn((hkv, slots, D), generator=g).to(store).to(device).transpose(0, 1)
    c["v"] = torch.randn((hkv, slots, D), generator=g).to(store).to(device).transpose(0, 1)
    total = len(lens) if new is None else sum(new)
    c["q"] = (1.5 * torch.randn((total, hq, D), generator=g)).to(dtype).to(device)
    c["sink"] = torch.randn(hq, generator=g).to(device)
    c["sums"] = torch.rand((len(rows), hkv, room), generator=g).to(device)
    if new is not None:
        c.update(new=list(new), prefix=ints([n - m for n, m in zip(lens, new)]), start=ints([sum(new[:b]) for b in range(len(new))]))
    return c


def _weights(c, b, q, place, cap, sink, seen=None):
    """Softmax weights [W, kv, group, n] in 64 bits of queries at cache indices ``place``, and a bound on the relative error of each.

    A score is a sum of D products in fp32, 16 at a time: D / 16 + 4 additions, each off by at most a step (2^-23) of the sum of the
    products' sizes.  The scale, the step to base 2 and the difference from the maximum are off by half a step of the largest score each.  The
    exponential is off by 2^-22, the normaliser by that, by its scores' errors and by half a step for each of the additions in a row
    (at most n / 16 + 64).  Everything counts twice: in the weight and in its normaliser."""
    n = c["lens"][b]
    slots = c["table"][int(c["req"][b]), :n].long()
    inside = (slots >= 0) & (slots < c["k"].shape[0])
    slots = slots.clamp(0, c["k"].shape[0] - 1)
    keys = c["k"][slots].double()
    q = q.double().view(q.shape[0], c["hkv"], -1, q.shape[-1])
    s = torch.einsum("wkgd,lkd->wkgl", q, keys) * c["scale"]
    size = torch.einsum("wkgd,lkd->wkgl", q.abs(), keys.abs()) * c["scale"]
    if cap:
        s = cap * torch.tanh(s / cap)
    visible = (torch.arange(n, device=s.device) <= place[:, None]) & inside
    s = s.masked_fill(~visible[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.double().view(1, c["hkv"], -1, 1))
    top = top.masked_fill(top == float("-inf"), 0.0)
    e = torch.exp(s - top)
    den = e.sum(-1, keepdim=True)
    if sink is not None:
        den = den + torch.exp(sink.double().view(1, c["hkv"], -1, 1) - top) * (e.sum(-1, keepdim=True) > 0)
    w = torch.where(den > 0, e / den, 0.0)
    step = 2.0 ** -23
    off = (q.shape[-1] / 16 + 4) * step * size.masked_fill(~visible[:, None, None], 0.0).amax(-1, keepdim=True)
    large = torch.where(s.isfinite(), s.abs(), 0.0).amax(-1, keepdim=True) + top.abs()
    off = 2 * (off + 4 * step * large + (4 * step * cap if cap else 0.0)) + (n / 16 + 64) * step
    return w, off


def exact_decode(c, decay=1.0, cap=0.0, sink=None):
    """(out, its bound, sums, their bound).  The output's weights are rounded to 16 bits (fp16 over 8-bit caches), in the product and in the
    normaliser: 2 roundings of the weighted sizes of the values; then the result's own rounding."""
    sums, bound = c["sums"].double(), torch.zeros_like(c["sums"], dtype=torch.float64)
    out, tol = torch.zeros_like(c["q"], dtype=torch.float64), torch.zeros_like(c["q"], dtype=torch.float64)
    u = HALF[c["q"].dtype]
    uw = u if c["k"].dtype == c["q"].dtype else HALF[torch.float16]
    for b, n in enumerate(c["lens"]):
        if n == 0:
            continue
        w, off = _weights(c, b, c["q"][b:b + 1], torch.tensor([n - 1], device=c["q"].device), cap, sink)
        slots = c["table"][int(c["req"][b]), :n].long().clamp(0, c["k"].shape[0] - 1)
        values = c["v"][slots].double()
        values = torch.where(w.sum((0, 2)).T[..., None] > 0, values, 0.0)
        o = torch.einsum("wkgl,lkd->wkgd", w, values)
        mass = torch.einsum("wkgl,lkd->wkgd", w, values.abs())
        out[b] = o.reshape(out.shape[1:])
        # fp16 weights go below its smallest normal number: 2^-25 each, of weights whose largest is 2^-8 at least
        tol[b] = (1.01 * (u * o.abs() + (2 * uw + off) * mass) + n * 2.0 ** -16 * 2.0 ** -8 * values.abs().amax() * 2.0 ** -1 * (uw == 2.0 ** -11)
                  + 1e-30).reshape(out.shape[1:])
        add, slack = w.sum((0, 2)), (w * off).sum((0, 2))
        row = int(c["req"][b])
        old = sums[row, :, :n].clone()
        old[:, -1] = 0
        sums[row, :, :n] = (decay * old if decay else 0.0) + add
        bound[row, :, :n] = 1.01 * slack + 2.0 ** -22 * (old + 8 * add) + 1e-37
    return out, tol, sums, bound


def exact_prompt(c, last=0, add=False, cap=0.0, sink=None):
    """(sums, their bound): of the additions in a row, one for each observed row."""
    sums, bound = c["sums"].double(), torch.zeros_like(c["sums"], dtype=torch.float64)
    for b, n in enumerate(c["lens"]):
        new, row = c["new"][b], int(c["req"][b])
        if n == 0 or new == 0:
            continue
        look = min(last, new) if last else new
        end = sum(c["new"][:b + 1])
        w, off = _weights(c, b, c["q"][end - look:end], torch.arange(n - look, n, device=c["q"].device), cap, sink)
        total, slack = w.sum((0, 2)), (w * off).sum((0, 2))
        old = torch.zeros_like(total)
        if add:
            old[:, :n - new] = sums[row, :, :n - new]
        sums[row, :, :n] = old + total
        bound[row, :, :n] = 1.01 * slack + 2.0 ** -24 * (w.shape[0] * w.shape[2] + 8) * (old + total) + 1e-37
    return sums, bound


def plain_select(sums, req, lens, budgets, width, first, recent, pool):
    """One list at a time, one token at a time."""
    keep = torch.full((sums.shape[0], len(lens), sums.shape[2], width), -1, dtype=torch.int32)
    counts = []
    for b, n in enumerate(lens):
        count = max(0, min(n, budgets[b], width))
        counts.append(count)
        for layer in range(sums.shape[0]):
            for head in range(sums.shape[2]):
                x = [v if v == v else float("-inf") for v in sums[layer, req[b], head, :n].tolist()]
                score = [max(x[max(0, i - pool // 2):i + pool // 2 + 1]) for i in range(n)]
                end = min(recent, count)
                begin = min(first, count - end)
                stay = set(range(n - end, n)) | set(range(begin))
                for i in sorted(range(begin, n - end), key=lambda i: (-score[i], i)):
                    if len(stay) == count:
                        break
                    stay.add(i)
                keep[layer, b, head, :count] = torch.tensor(sorted(stay), dtype=torch.int32)
    return keep, torch.tensor(counts, dtype=torch.int32)


class Shortened:
    """A tiny model whose requests are shortened while they are decoded."""

    def __init__(self, preset, device, dtype, kv_cache_dtype="auto"):
        from mllm_b200.configs import ServerConfig
        from mllm_b200.executor import ModelRunner

        self.mr = ModelRunner(ServerConfig(model_path=f"preset:{preset}", dtype=dtype, max_running_requests=8, max_total_tokens=4096),
                              kv_cache_dtype=kv_cache_dtype, device=device)
        self.mr.initialize()
        self.dev = torch.device(device)

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def start(self, prompts, **kw):
        mr = self.mr
        rows = mr.req_to_token_pool.alloc(len(prompts))
        table, lens = mr.req_to_token_pool.req_to_token, [len(p) for p in prompts]
        locs = [mr.token_to_kv_pool_allocator.alloc(n) for n in lens]
        for r, loc in zip(rows, locs):
            table[r, :len(loc)] = loc.to(torch.int32)
        fb = mr.prepare_forward_batch_extend(torch.tensor([t for p in prompts for t in p], device=self.dev), self.ints(rows), self.ints(lens), self.ints(lens),
                                             self.ints([0] * len(rows)), torch.cat(locs), lens, [0] * len(rows), **kw)
        return rows, mr.forward(fb).next_token_logits.clone()

    def step(self, rows, lens, positions, tokens, **kw):
        """The next token of every request, whose cache has ``lens`` tokens."""
        mr = self.mr
        locs = torch.cat([mr.token_to_kv_pool_allocator.alloc(1) for _ in rows])
        table = mr.req_to_token_pool.req_to_token
        for r, n, loc in zip(rows, lens, locs.tolist()):
            table[r, n] = loc
        fb = mr.prepare_forward_batch_decode(torch.tensor(tokens, device=self.dev), self.ints(rows), self.ints([n + 1 for n in lens]), locs,
                                             max_seq_len=max(lens) + 1, positions=self.ints(positions), **kw)
        return mr.forward(fb).next_token_logits.clone()        # (a captured step has its logits in one place)

    def free(self, rows):
        for r in rows:
            self.mr.req_to_token_pool.free(r)

    def check(self, close):
        from mllm_b200 import ops

        g = random.Random(5)
        mr, prompts = self.mr, [[g.randrange(self.mr.vocab_size) for _ in range(n)] for n in (50, 23, 4)]
        tokens = [[g.randrange(mr.vocab_size) for _ in prompts] for _ in range(4)]
        table = mr.req_to_token_pool.req_to_token
        sums = mr.token_to_kv_pool.make_weight_sums(table.shape[0], 80)
        lens = [len(p) for p in prompts]
        # nothing is dropped: as if nothing had been asked for
        plain, want = self.start(prompts)
        want = [want] + [self.step(plain, [n + i for n in lens], [n + i for n in lens], tokens[i]) for i in range(2)]
        rows, got = self.start(prompts, weight_sums=sums, weight_last=8)
        close(got, want[0])
        heads = mr.model.model.layers[0].self_attn.attn.num_heads
        mass = sums[:, rows].sum((2, 3))
        torch.testing.assert_close(mass, torch.tensor([min(n, 8) * heads for n in lens], device=self.dev).float().expand_as(mass), rtol=1e-4, atol=1e-4)
        now = mr.evict_cache(sums, self.ints(rows), self.ints(lens), self.ints([80, 23, 4]), 80)
        assert now.tolist() == lens
        close(self.step(rows, lens, lens, tokens[0], weight_sums=sums), want[1])
        close(self.step(rows, [n + 1 for n in lens], [n + 1 for n in lens], tokens[1], weight_sums=sums, weight_decay=0.9), want[2])
        # and now it is: what is left is attended to as any cache is, at the positions that the tokens have in the text
        here = [n + 2 for n in lens]
        now = mr.evict_cache(sums, self.ints(rows), self.ints(here), self.ints([20, 12, 80]), 80, first=2, recent=5, pool=3)
        assert now.tolist() == [20, 12, 6]
        store, table_now = mr.token_to_kv_pool.store.clone(), table.clone()
        a = self.step(rows, now.tolist(), here, tokens[2], weight_sums=sums)
        mr.token_to_kv_pool.store.copy_(store)
        table.copy_(table_now)
        close(a, self.step(rows, now.tolist(), here, tokens[2]))
        # the dropped tokens matter to the requests that lost some, and to no other
        full = self.step(plain, here, here, tokens[2])
        assert (a[0].float() - full[0].float()).abs().max() > 1e-3 and (a[1].float() - full[1].float()).abs().max() > 1e-3
        close(a[2], full[2])
        # new text behind a shortened request
        n = [x + 1 for x in now.tolist()]
        locs = [mr.token_to_kv_pool_allocator.alloc(3) for _ in rows]
        for r, at, loc in zip(rows, n, locs):
            table[r, at:at + 3] = loc.to(torch.int32)
        fb = mr.prepare_forward_batch_extend(torch.tensor([1, 2, 3] * 3, device=self.dev), self.ints(rows), self.ints([x + 3 for x in n]), self.ints([3] * 3),
                                             self.ints(n), torch.cat(locs), [3] * 3, n, first_positions_cpu=[x + 1 for x in here], weight_sums=sums, weight_add=True)
        assert fb.positions.tolist() == [x + 1 + i for x in here for i in range(3)]
        before = sums.clone()
        assert torch.isfinite(mr.forward(fb).next_token_logits).all()
        added = (sums - before)[:, rows[0], :, :n[0]]
        assert (added >= 0).all() and (added.sum((1, 2)) > 0).all()
        ops.check_status()
        self.free(rows)
        self.free(plain)
