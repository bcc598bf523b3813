"""Shortened requests on the CPU: the statements against 64 bits and against a token at a time, and what is refused."""
import pytest
import torch

from evict_cases import Shortened, cached_batch, exact_decode, exact_prompt, plain_select
from mllm_b200 import ops


def index(c):
    return c["table"], c["req"], c["seq"]


@pytest.mark.parametrize("kw", [{}, dict(decay=0.5), dict(decay=0.0), dict(cap=3.0), dict(sink=True)])
def test_decode_statement(kw):
    c = cached_batch([1, 40, 0, 17], 4, 2, 16, dtype=torch.float32, seed=3, device="cpu")
    sink = c["sink"] if kw.pop("sink", False) else None
    want, tol, sums, bound = exact_decode(c, sink=sink, **kw)
    cap = kw.pop("cap", 0.0)
    got = ops.attention_decode_weights(c["q"], c["k"], c["v"], *index(c), c["scale"], c["sums"], logit_cap=cap, sink=sink, **kw)
    assert ((got.double() - want).abs() <= tol + 1e-5).all() and ((c["sums"].double() - sums).abs() <= bound + 1e-6).all()
    plain = ops.attention_decode(c["q"], c["k"], c["v"], *index(c), c["scale"], logit_cap=cap, sink=sink)
    torch.testing.assert_close(got[[0, 1, 3]], plain[[0, 1, 3]], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("last", [0, 1, 5, 100])
@pytest.mark.parametrize("add", [False, True])
def test_prompt_statement(last, add):
    c = cached_batch([9, 40, 3, 12], 4, 2, 16, dtype=torch.float32, seed=4, new=[9, 7, 0, 1], device="cpu")
    sums, bound = exact_prompt(c, last, add, sink=c["sink"])
    ops.attention_prefill_weights(c["q"], c["k"], *index(c), c["prefix"], c["start"], c["scale"], c["sums"], last=last, add=add, sink=c["sink"])
    assert ((c["sums"].double() - sums).abs() <= bound + 1e-6).all()


@pytest.mark.parametrize("first,recent,pool", [(0, 0, 1), (4, 8, 1), (3, 0, 5), (0, 6, 3), (50, 50, 1), (2, 100, 7)])
def test_select_statement(first, recent, pool):
    torch.manual_seed(first + recent + pool)
    lens, budgets = [1, 30, 0, 64, 11], [5, 12, 4, 0, 11]
    sums = torch.randint(0, 6, (2, 6, 3, 64)).float()          # many ties
    sums[0, :, :, 5] = float("nan")
    sums[1, :, 0, :20] = float("-inf")
    sums[1, :, 1, 3] = float("inf")
    sums[:, :, 2, 7] = -0.0
    req = [3, 0, 5, 1, 2]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    keep, counts = ops.cache_select(sums, i32(req), i32(lens), i32(budgets), 12, first=first, recent=recent, pool=pool)
    want, want_counts = plain_select(sums, req, lens, budgets, 12, first, recent, pool)
    assert torch.equal(keep, want) and torch.equal(counts, want_counts) and keep.dtype == counts.dtype == torch.int32


def test_evict_statement():
    c = cached_batch([20, 7, 30], 2, 2, 16, dtype=torch.bfloat16, seed=5, layers=2, page=4, device="cpu")
    budgets = torch.tensor([9, 7, 12], dtype=torch.int32)
    keep, counts = ops.cache_select(c["sums"], c["req"], c["seq"], budgets, 12, first=2, recent=3)
    store, sums = c["store"].clone(), c["sums"].clone()
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, counts)
    for b in range(3):
        row, n = int(c["req"][b]), int(counts[b])
        for layer in range(2):
            for head in range(2):
                for i in range(n):
                    k = int(keep[layer, b, head, i])
                    assert torch.equal(c["store"][layer, :, head, c["table"][row, i]], store[layer, :, head, c["table"][row, k]])
                    assert c["sums"][layer, row, head, i] == sums[layer, row, head, k]
    with pytest.raises(ValueError, match="smaller than its place"):
        ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep.flip(-1).contiguous().clamp(min=0), counts)


def refusals(device):
    """(call, what the message says) for arguments that no device takes."""
    c = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, device=device)
    p = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, new=[5, 6], device=device)
    s = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, layers=3, device=device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    budgets = i32([8, 8])

    def decode(**kw):
        a = dict(q=c["q"], k_cache=c["k"], v_cache=c["v"], req_to_token=c["table"], req_pool_indices=c["req"], seq_lens=c["seq"], scale=0.1,
                 sums=c["sums"])
        return lambda: ops.attention_decode_weights(**{**a, **kw})

    def prompt(**kw):
        a = dict(q=p["q"], k_cache=p["k"], req_to_token=p["table"], req_pool_indices=p["req"], seq_lens=p["seq"], prefix_lens=p["prefix"],
                 q_start_loc=p["start"], scale=0.1, sums=p["sums"])
        return lambda: ops.attention_prefill_weights(**{**a, **kw})

    def select(**kw):
        a = dict(sums=s["sums"], req_pool_indices=s["req"], seq_lens=s["seq"], budgets=budgets, max_budget=8)
        return lambda: ops.cache_select(**{**a, **kw})

    keep = torch.zeros((3, 2, 2, 8), dtype=torch.int32, device=device)

    def evict(**kw):
        a = dict(store=s["store"], sums=s["sums"], req_to_token=s["table"], req_pool_indices=s["req"], keep=keep, counts=i32([0, 0]))
        return lambda: ops.cache_evict(**{**a, **kw})

    return [
        (decode(q=c["q"][0]), "q must be"), (decode(q=c["q"].transpose(1, 2).contiguous().transpose(1, 2)), "q must be"),
        (decode(q=c["q"][:, :3]), "key heads|contiguous"), (decode(k_cache=c["k"].float()), "caches must be"), (decode(v_cache=c["v"][:-1]), "one layout"),
        (decode(v_cache=c["v"].to(torch.float8_e5m2)), "one layout"), (decode(scale=0.0), "scale"), (decode(scale=float("nan")), "scale"),
        (decode(scale=-1.0), "scale"), (decode(logit_cap=-2.0), "logit_cap"), (decode(logit_cap=float("inf")), "logit_cap"),
        (decode(decay=1.5), "decay"), (decode(decay=-0.1), "decay"), (decode(decay=float("nan")), "decay"), (decode(seq_lens=c["seq"].long()), "int32"),
        (decode(seq_lens=c["seq"][:1]), "vector of 2"), (decode(req_pool_indices=c["req"][:1]), "vector of|rows for"),
        (decode(req_to_token=c["table"].long()), "two-dimensional int32"), (decode(req_to_token=c["table"][0]), "two-dimensional int32"),
        (decode(sums=c["sums"].double()), "sums must be"), (decode(sums=c["sums"][:, :1]), "sums must be"), (decode(sums=c["sums"][..., ::2]), "sums must be"),
        (decode(sums=c["sums"][0]), "sums must be"), (decode(out=c["q"].float()), "out must be"), (decode(out=c["q"][:1]), "out must be"),
        (decode(sink=c["sink"][:3]), "sink must be"), (decode(sink=c["sink"].double()), "sink must be"),
        (prompt(q=p["q"][0]), "q must be"), (prompt(last=-1), "last"), (prompt(scale=float("inf")), "scale"), (prompt(prefix_lens=p["prefix"].long()), "int32"),
        (prompt(q_start_loc=p["start"][:1]), "vector of 2"), (prompt(sums=p["sums"][None]), "sums must be"), (prompt(sink=p["sink"][:1]), "sink must be"),
        (prompt(k_cache=p["k"][..., :32]), "caches must be"), (prompt(logit_cap=float("nan")), "logit_cap"),
        (select(sums=s["sums"][0]), "sums must be"), (select(sums=s["sums"].half()), "sums must be"), (select(max_budget=-1), "max_budget"),
        (select(max_budget=10 ** 6), "max_budget"), (select(first=-1), "first and recent"), (select(recent=-2), "first and recent"),
        (select(pool=0), "pool"), (select(pool=4), "pool"), (select(pool=65), "pool"), (select(budgets=budgets.long()), "int32"),
        (select(budgets=budgets[:1]), "vector of 2"), (select(seq_lens=s["seq"][:1]), "vector of 2"),
        (evict(store=s["store"][0]), "store must be"), (evict(store=s["store"][..., :32]), "store must be"),
        (evict(store=s["store"].reshape(3, 2, 2, -1, 4)), "store must be"), (evict(keep=keep[:2]), "keep must be"), (evict(keep=keep.long()), "keep must be"),
        (evict(keep=keep[..., ::2]), "keep must be"), (evict(counts=i32([0])), "vector of 2"), (evict(sums=s["sums"][:2]), "layers|sums"),
        (evict(sums=s["sums"].half()), "sums must be"), (evict(req_to_token=s["table"].long()), "two-dimensional int32"),
    ]


@pytest.mark.parametrize("i", range(len(refusals("cpu"))))
def test_refusals(i):
    call, message = refusals("cpu")[i]
    with pytest.raises(ValueError, match=message):
        call()


def test_kernels_cover():
    bf, fp = torch.bfloat16, torch.float16
    assert ops.cache_weights_cover(128, 32, bf, bf) and ops.cache_weights_cover(256, 16, torch.float8_e5m2, fp)
    assert not ops.cache_weights_cover(256, 17, bf, bf) and not ops.cache_weights_cover(96, 4, bf, bf) and not ops.cache_weights_cover(64, 4, fp, bf)
    assert not ops.cache_weights_cover(64, 4, torch.float32, torch.float32)


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen2-tiny", "qwen3-moe-tiny"])
def test_shortened_requests_of_a_model(preset):
    Shortened(preset, "cpu", "float32").check(lambda a, b: torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4))


def test_models_with_other_layers_keep_no_sums():
    s = Shortened("qwen3.5-tiny", "cpu", "float32")
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="attention weights"):
        s.mr.prepare_forward_batch_decode(one.long(), one, one + 1, one.long(), weight_sums=torch.zeros(1, 1, 1, 1))
    s = Shortened("qwen3-tiny", "cpu", "float32")
    with pytest.raises(ValueError, match="layers"):
        s.mr.prepare_forward_batch_decode(one.long(), one, one + 1, one.long(), weight_sums=torch.zeros(1, 1, 1, 1))
    with pytest.raises(ValueError, match="trees"):
        s.mr.prepare_forward_batch_tree(one.long(), one - 1, one, [1], [0], weight_sums=s.mr.token_to_kv_pool.make_weight_sums(2, 8))
    for m in s.mr.model.modules():
        if hasattr(m, "sliding_window"):
            m.sliding_window = 16
    with pytest.raises(ValueError, match="sliding window"):
        s.mr.prepare_forward_batch_decode(one.long(), one, one + 1, one.long(), weight_sums=s.mr.token_to_kv_pool.make_weight_sums(2, 8))
