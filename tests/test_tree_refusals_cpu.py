"""Calls of the operators for drafted token trees that are refused, on the CPU."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import tree_batch


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e-42, 1e39])
def test_refused_scales(scale):
    c = tree_batch([4, 2], [3, 2], 4, 2, 16, device="cpu", dtype=torch.float32)
    args = (c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"])
    ops.attention_tree(*args, 0.25)
    with pytest.raises(ValueError, match="scale"):
        ops.attention_tree(*args, scale)
