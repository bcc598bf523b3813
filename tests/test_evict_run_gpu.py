"""The four operators in a row, each against what the one before left: on a stream of its own, captured and replayed; and two prompts at once."""
import pytest
import torch

from evict_cases import cached_batch, exact_decode, exact_prompt, plain_select
from test_evict_gpu import i32, moved, prompt, within
from mllm_b200 import ops

pytestmark = pytest.mark.gpu
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


class Run:
    """A prompt's weights, selection, eviction and the next token, with what stood in the buffers between them."""

    def __init__(self, lens, new, hq, hkv, D, dtype, cache, page, budgets):
        self.p = p = cached_batch(lens, hq, hkv, D, dtype=dtype, cache=cache, seed=21, new=new, page=page)
        self.q = cached_batch([1] * len(lens), hq, hkv, D, dtype=dtype, seed=22)["q"]
        self.store = torch.stack([p["k"].transpose(0, 1), p["v"].transpose(0, 1)])[None].contiguous()
        p["k"], p["v"] = self.store[0, 0].transpose(0, 1), self.store[0, 1].transpose(0, 1)
        self.sums, self.budgets, self.width = p["sums"][None], i32(budgets), max(budgets)
        self.start = self.store.clone(), self.sums.clone()

    def reset(self):
        self.store.copy_(self.start[0])
        self.sums.copy_(self.start[1])

    def call(self):
        p = self.p
        ops.attention_prefill_weights(p["q"], p["k"], p["table"], p["req"], p["seq"], p["prefix"], p["start"], p["scale"], self.sums[0], last=8)
        seen = self.sums.clone()
        keep, counts = ops.cache_select(self.sums, p["req"], p["seq"], self.budgets, self.width, first=2, recent=8, pool=3)
        ops.cache_evict(self.store, self.sums, p["table"], p["req"], keep, counts)
        left, left_sums = self.store.clone(), self.sums.clone()
        out = ops.attention_decode_weights(self.q, p["k"], p["v"], p["table"], p["req"], counts, p["scale"], self.sums[0])
        return seen, keep, counts, left, left_sums, out

    def check(self, seen, keep, counts, left, left_sums, out):
        p = self.p
        k, v = (self.start[0][0, i].transpose(0, 1) for i in (0, 1))
        want, bound = exact_prompt(dict(p, k=k, sums=self.start[1][0]), last=8)
        within(seen[0], want, bound, "weights of the prompt")
        want, want_counts = plain_select(seen.cpu(), p["req"].tolist(), p["lens"], self.budgets.tolist(), self.width, 2, 8, 3)
        assert torch.equal(keep.cpu(), want) and torch.equal(counts.cpu(), want_counts)
        store, sums = moved(dict(p, store=self.start[0], sums=seen), keep, counts)
        assert torch.equal(left.view(torch.uint8), store.view(torch.uint8)) and torch.equal(left_sums, sums)
        k, v = (left[0, i].transpose(0, 1) for i in (0, 1))
        want, tol, sums, bound = exact_decode(dict(p, q=self.q, k=k, v=v, sums=left_sums[0], lens=counts.tolist()))
        within(out, want, tol, "out")
        within(self.sums[0], sums, bound, "sums")
        assert torch.equal(self.store.view(torch.uint8), left.view(torch.uint8))


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, None), (torch.float16, E5), (torch.bfloat16, E4)])
@pytest.mark.parametrize("lens,new,hq,hkv,D,page,budgets", [
    ([200, 77, 130], [200, 40, 130], 8, 2, 128, 1, [64, 77, 33]), ([3000, 1, 900], [700, 1, 900], 16, 2, 64, 16, [700, 1, 45]),
    ([600] * 6, [600, 10, 1, 64, 600, 300], 12, 3, 256, 16, [100, 200, 300, 400, 500, 600]),
])
def test_each_against_what_the_one_before_left(dtype, cache, lens, new, hq, hkv, D, page, budgets):
    r = Run(lens, new, hq, hkv, D, dtype, cache, page, budgets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = r.call()
    side.synchronize()
    r.check(*got)
    r.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = r.call()
    for turn in range(3):
        if turn:                             # other data, and then other budgets
            r.p["q"].copy_(r.p["q"].flip(0))
            r.q.copy_(r.q.flip(1))
            r.start[0][:, 0].copy_(r.start[0][:, 0].flip(-2))
        if turn == 2:
            r.budgets.sub_(1).clamp_(min=1)
        r.reset()
        graph.replay()
        torch.cuda.synchronize()
        r.check(*held)
    ops.check_status()


@pytest.mark.parametrize("D,cache", [(128, None), (64, None), (128, E4), (256, None)])
@pytest.mark.parametrize("last", [0, 64])
def test_two_prompts_at_once(D, cache, last):
    """Units are cut between blocks: partial results and notes are a call's own."""
    batches = [cached_batch([900, 300, 1100], 8, 2, D, cache=cache, seed=s, new=[900, 300, 700]) for s in (1, 2)]
    want = []
    for c in batches:
        sums = c["sums"].clone()
        prompt(dict(c, sums=sums), last=last)
        want.append(sums)
    exact, bound = exact_prompt(batches[0], last=last)
    within(want[0], exact, bound, "sums")
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, st in zip(batches, streams):
            with torch.cuda.stream(st):
                sums = c["sums"].clone()
                prompt(dict(c, sums=sums), last=last)
                got.append(sums)
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    ops.check_status()
