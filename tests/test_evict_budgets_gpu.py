"""Budgets above the longest that a call provides for, or below 0, are cut, as documented: nothing is recorded."""
import pytest
import torch

from evict_cases import plain_select
from mllm_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("budgets", [[100, 40, 2 ** 31 - 1], [64, -1, 65], [-2 ** 31, 1000, 64]])
def test_budgets_are_cut(budgets):
    sums, lens = torch.rand((2, 3, 2, 200)), [150, 90, 200]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    keep, counts = ops.cache_select(sums.cuda(), i32([0, 1, 2]), i32(lens), i32(budgets), 64)
    ops.check_status()
    want, want_counts = plain_select(sums, [0, 1, 2], lens, budgets, 64, 4, 32, 1)
    assert torch.equal(keep.cpu(), want) and torch.equal(counts.cpu(), want_counts)
