"""What the bindings refuse before anything is launched."""
import pytest
import torch

from evict_cases import cached_batch
from evict_refusals import overlapping, too_large
from mllm_b200 import ops

pytestmark = pytest.mark.gpu


def test_what_lies_on_itself():
    before = ops.launch_count()
    for call, message in overlapping("cuda"):
        with pytest.raises(ValueError, match=message):
            call()
    assert ops.launch_count() == before


def test_scales_and_caps_that_are_too_large():
    for call, message in too_large("cuda"):
        with pytest.raises(ValueError, match=message):
            call()


def test_layouts_that_are_taken():
    c = cached_batch([40, 17], 4, 2, 64, seed=1)
    rows, heads, tokens = c["sums"].shape
    want, flat = None, torch.zeros((heads, 2 * rows, tokens + 3), device="cuda")
    for sums in (c["sums"].clone(), c["sums"].transpose(0, 1).contiguous().transpose(0, 1), flat[:, ::2, 1:-2].transpose(0, 1).copy_(c["sums"])):
        ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], 0.1, sums)
        want = sums.clone() if want is None else want
        assert torch.equal(sums, want)
    ops.check_status()
