"""Sums and outputs whose rows lie on each other are refused; other layouts are taken."""
import pytest
import torch

from evict_cases import cached_batch
from evict_refusals import overlapping, too_large
from mllm_b200 import ops


@pytest.mark.parametrize("i", range(len(overlapping("cpu"))))
def test_refusals(i):
    call, message = overlapping("cpu")[i]
    with pytest.raises(ValueError, match=message):
        call()


@pytest.mark.parametrize("i", range(len(too_large("cpu"))))
def test_scales_and_caps_that_are_too_large(i):
    call, message = too_large("cpu")[i]
    with pytest.raises(ValueError, match=message):
        call()


def test_layouts_that_are_taken():
    c = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, device="cpu")
    rows, heads, tokens = c["sums"].shape
    want = None
    flat = torch.zeros((heads, 2 * rows, tokens + 3))
    for sums in (c["sums"].clone(), c["sums"].transpose(0, 1).contiguous().transpose(0, 1), flat[:, ::2, 1:-2].transpose(0, 1).copy_(c["sums"])):
        ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], 0.1, sums)
        want = sums.clone() if want is None else want
        assert torch.equal(sums, want)
    # one row, one head: strides say nothing; and sums that are read only may be expanded
    one = cached_batch([9], 1, 1, 64, dtype=torch.bfloat16, seed=2, device="cpu", extra_rows=0)
    ops.attention_decode_weights(one["q"], one["k"], one["v"], one["table"], one["req"], one["seq"], 0.1, one["sums"].as_strided((1, 1, 14), (0, 0, 1)))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    keep, _ = ops.cache_select(c["sums"][None].expand(2, -1, -1, -1), c["req"], c["seq"], i32(8, 8), 8)
    assert torch.equal(keep[0], keep[1])
