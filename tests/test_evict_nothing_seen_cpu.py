"""Queries that see only scores of minus infinity: no weight, and a row of zeros, as on the GPU."""
import pytest
import torch

from evict_cases import cached_batch
from mllm_b200 import ops


def case(new):
    c = cached_batch([70, 5], 4, 1, 16, dtype=torch.float32, seed=13, new=new, device="cpu")
    c["q"][:] = c["q"].abs() + 0.1
    return c, c["table"][int(c["req"][0])].long()


@pytest.mark.parametrize("sink", [None, 0.5, float("-inf")])
def test_prompt(sink):
    c, slots = case([70, 5])
    c["k"][slots[:10]] = float("-inf")       # the first ten queries see nothing
    sinks = None if sink is None else torch.full((4,), sink)
    ops.attention_prefill_weights(c["q"], c["k"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["scale"], c["sums"], sink=sinks)
    got = c["sums"][int(c["req"][0]), 0, :70]
    assert not torch.isnan(got).any() and (got[:10] == 0).all()
    if sink != 0.5:
        assert abs(got.sum().item() - 60 * 4) < 1e-3
    c["k"][slots[30]] = float("nan")         # what is no number shows where it is seen
    ops.attention_prefill_weights(c["q"], c["k"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["scale"], c["sums"], last=1, sink=sinks)
    assert torch.isnan(c["sums"][int(c["req"][0]), 0, :70]).all() and not torch.isnan(c["sums"][int(c["req"][1])]).any()


@pytest.mark.parametrize("sink", [None, 0.5, float("-inf")])
def test_decode(sink):
    c, slots = case(None)
    c["k"][slots[:70]] = float("-inf")
    before, row = c["sums"].clone(), int(c["req"][0])
    out = ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["scale"], c["sums"],
                                       sink=None if sink is None else torch.full((4,), sink))
    assert (out[0] == 0).all() and torch.equal(c["sums"][row, :, :69], before[row, :, :69]) and (c["sums"][row, :, 69] == 0).all()
    assert not torch.isnan(out).any() and not torch.isnan(c["sums"]).any()
