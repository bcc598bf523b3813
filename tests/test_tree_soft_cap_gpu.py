"""Soft caps far above the scores of drafted trees: the cap is the identity there."""
import pytest
import torch

from test_tree_attention_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [0.5, 50.0, 1e3, 1e6, 1e20])
@pytest.mark.parametrize("D,dtype,cache", [(128, torch.bfloat16, None), (64, torch.float16, None), (256, torch.bfloat16, None), (128, torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("prefix,nodes", [([0, 300, 129], [40, 9, 70]), ([200, 700], [65, 64])])
def test_caps(cap, D, dtype, cache, prefix, nodes):
    check(dict(prefix=prefix, nodes=nodes, hq=8, hkv=2, D=D, dtype=dtype, cache=cache, seed=D), logit_cap=cap)
