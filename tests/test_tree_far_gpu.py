"""Operators of drafted token trees on tensors whose offsets pass 32 bits: caches, storages and logits of more than 2^31 elements."""
import pytest
import torch

from mllm_b200 import ops
from mllm_b200.ops import reference as ref
from tree_cases import exact_attention, exact_prologue, slots_of_rows, tree_batch

pytestmark = pytest.mark.gpu
FAR = 2_200_000         # slots: 8 heads of 128 features are 1024 elements each


def far_batch(cache):
    c = tree_batch([300, 5], [20, 7], 16, 8, 128, cache=cache)
    small = c["slots"]
    for name in ("k", "v"):
        big = torch.empty((FAR, 8, 128), dtype=c[name].dtype, device="cuda")
        big[-small:] = c[name]
        c[name] = big
    c["table"] += FAR - small
    return c


@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn])
def test_far_slots(cache):
    c = far_batch(cache)
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(27, 32 * 128, generator=g).cuda().to(torch.bfloat16)
    gains = [torch.ones(128, device="cuda", dtype=torch.bfloat16)] * 2
    inv = (1e4 ** -(torch.arange(64) / 64)).cuda()
    index = (c["table"], c["req"], c["seq"], c["prefix"], c["start"])
    q = ops.tree_qk_norm_rope_kv_write(qkv, *gains, c["parents"], *index, inv, c["k"], c["v"], 16, 8, 128, 1e-6)
    ops.check_status()
    loc = torch.tensor(slots_of_rows(c), device="cuda")
    for got, want in zip((q, c["k"][loc], c["v"][loc]), exact_prologue(c, qkv, gains, inv, 16, 8, 1e-6)):
        # one rounding, and 32-bit arithmetic of pairs; 8-bit caches: half a step of the smallest numbers too
        half = torch.finfo(got.dtype).eps / 2
        tiny = torch.finfo(got.dtype).smallest_normal * half
        assert ((got.double() - want).abs() <= half * want.abs() + want.abs().amax(-1, keepdim=True) * 2 ** -20 + tiny).all()
    got = ops.attention_tree(q, c["k"], c["v"], *index, c["parents"], c["scale"])
    ops.check_status()
    c["q"] = q
    want, bound = exact_attention(c, bounds=True)
    assert ((got.double() - want).abs() <= bound).all()


def test_far_rows_move():
    store = torch.empty((2, FAR // 2, 1024), dtype=torch.bfloat16, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    last = FAR // 2 - 8
    rows = torch.randn(2, 8, 1024, device="cuda").to(torch.bfloat16)
    store[:, last:] = rows
    ops.tree_kv_compact(store, ints([list(range(last, last + 8))]), ints([0]), ints([2]), ints([[0, 2, 5]]), ints([3]))
    ops.check_status()
    want = rows.clone()
    want[:, 3], want[:, 4] = rows[:, 4], rows[:, 7]
    assert torch.equal(store[:, last:], want)


def test_far_logits():
    T, V = 14_500, 151_936
    logits = torch.empty((T, V), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(4)
    near = torch.randn(6, V, generator=g)
    near[:, 7] = 9.0
    logits[-6:] = near.cuda().to(torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    one = lambda x: torch.tensor([x], device="cuda")  # noqa: E731
    tokens, parents, u = torch.full((T,), 7, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda"), torch.full((T,), 0.01, device="cuda")
    parents[-6:] = ints([-1, 0, 1, 2, 3, 4])
    rest = (one(0.7), ints([40]), one(0.95), one(0.0))
    got = ops.tree_speculative_sample(logits, tokens, parents, ints([6]), ints([T - 6]), *rest, u, one(0.3), 6)
    ops.check_status()
    want = ref.tree_speculative_sample(logits[-6:], tokens[-6:], parents[-6:], ints([6]), ints([0]), *rest, u[-6:], one(0.3), 6, None)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(got[2]) == 6
