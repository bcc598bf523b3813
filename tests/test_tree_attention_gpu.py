"""Attention of drafted token trees on the GPU against the formula in 64 bits: lengths around the tiles, odd trees and groups, slots in
any order, windows, chunks, caps, sinks, 8-bit caches, values that are no numbers, streams and captured graphs."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import exact_attention, tree_batch

pytestmark = pytest.mark.gpu


def check(case, **kw):
    c = tree_batch(**case)
    n0 = ops.launch_count()
    got = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], **kw)
    ops.check_status()
    assert ops.launch_count() > n0
    want, bound = exact_attention(c, bounds=True, **kw)
    over = (got.double() - want).abs() - bound
    assert not torch.isnan(got).any() and over.max().item() <= 0, ((got.double() - want).abs().max().item(), over.max().item())
    return c, got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("prefix,nodes", [
    ([0], [1]), ([0], [7]), ([1], [1]), ([63], [1]), ([64], [1]), ([60], [9]), ([127, 64, 1, 0], [1, 33, 64, 5]), ([700, 33], [65, 3]),
    ([1000], [130]), ([2500], [1]),
])
def test_lengths(D, prefix, nodes):
    check(dict(prefix=prefix, nodes=nodes, hq=8, hkv=2, D=D, seed=len(prefix) + D))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 1), (16, 1), (40, 8), (32, 4), (12, 3), (128, 1)])
def test_groups_of_heads(hq, hkv):
    check(dict(prefix=[300, 20], nodes=[17, 30], hq=hq, hkv=hkv, D=128, seed=hq))


@pytest.mark.parametrize("D,prefix,nodes,hq,hkv", [(128, [2048] * 8, [32] * 8, 32, 8), (64, [2048] * 8, [32] * 8, 32, 8), (256, [3000] * 4, [20] * 4, 8, 2)])
def test_long_runs_of_tiles(D, prefix, nodes, hq, hkv):
    """Several tiles in a row in every CTA, all CTAs at work: products and their waits overlap; twice, to the same bits."""
    c, got = check(dict(prefix=prefix, nodes=nodes, hq=hq, hkv=hkv, D=D, page=16))
    again = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"])
    assert torch.equal(got, again)
