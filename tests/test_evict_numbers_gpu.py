"""Numbers that the kernels of shortened requests cannot follow: recorded, and what they describe is left as it is."""
import pytest
import torch

from evict_cases import cached_batch
from mllm_b200 import ops

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def recorded():
    try:
        ops.check_status()
    except RuntimeError as e:
        assert "index out of range" in str(e)
        return True
    return False


@pytest.mark.parametrize("slot", [-2 ** 31, -2 ** 31 + 1, -1, 2 ** 31 - 1])
@pytest.mark.parametrize("end", ["from", "to"])
def test_moved_rows_whose_slots_are_none(slot, end):
    c = cached_batch([50], 2, 2, 64, seed=3, layers=2)
    slots = c["table"][int(c["req"][0])].long()
    c["table"][int(c["req"][0]), 24 if end == "from" else 4] = slot
    before = c["store"].clone()
    keep = torch.arange(20, 30, dtype=torch.int32, device="cuda").expand(2, 1, 2, 10).contiguous()
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, i32(10))
    assert recorded()
    moved = before.clone()
    others = [i for i in range(10) if i != 4]
    moved[:, :, :, slots[others]] = before[:, :, :, slots[[i + 20 for i in others]]]
    assert torch.equal(c["store"], moved)


@pytest.mark.parametrize("width", [0, 1, 10, 40])
def test_more_tokens_stay_than_keep_has(width):
    """One request's count says more than the list holds: that request stays as it is."""
    c = cached_batch([50, 45], 2, 2, 64, seed=3, layers=2)
    store, sums = c["store"].clone(), c["sums"].clone()
    keep = (torch.arange(width, dtype=torch.int32, device="cuda") + 2).expand(2, 2, 2, width).contiguous()
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, i32(width + 1, width))
    assert recorded()
    row = int(c["req"][1])
    slots = c["table"][row].long()
    want, total = store.clone(), sums.clone()
    want[:, :, :, slots[:width]] = store[:, :, :, slots[2:2 + width]]
    total[:, row, :, :width] = sums[:, row, :, 2:2 + width]
    assert torch.equal(c["store"], want) and torch.equal(c["sums"], total)
