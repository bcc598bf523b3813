"""More tokens than a list of kept ones has: refused on the CPU."""
import pytest
import torch

from evict_cases import cached_batch
from mllm_b200 import ops


def test_more_tokens_stay_than_keep_has():
    c = cached_batch([20], 2, 2, 16, dtype=torch.bfloat16, seed=5, layers=2, device="cpu")
    keep = torch.arange(4, dtype=torch.int32).expand(2, 1, 2, 4).contiguous()
    with pytest.raises(ValueError, match="5 tokens stay and keep has 4"):
        ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, torch.tensor([5], dtype=torch.int32))
