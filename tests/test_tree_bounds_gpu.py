"""Drafted token trees on the GPU: operands that the binding refuses because the kernels could not read them."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import tree_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("shift", [1, 4, 7])
def test_weights_off_16_byte_boundaries_are_refused(D, which, shift):
    """The prologue reads weights 16 bytes at a time: a slice that begins elsewhere never reaches the kernel."""
    c = tree_batch([4, 2], [3, 2], 4, 2, D)
    qkv, inv = torch.randn(5, 8 * D, device="cuda").to(torch.bfloat16), torch.ones(D // 2, device="cuda")
    buffer = torch.ones(D + 8, device="cuda", dtype=torch.bfloat16)
    gains = [None, None]

    def call():
        return ops.tree_qk_norm_rope_kv_write(qkv, *gains, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], inv, c["k"], c["v"],
                                              4, 2, D, 1e-6)

    gains[which] = buffer[shift:shift + D]
    before = ops.launch_count()
    with pytest.raises(ValueError, match="16-byte"):
        call()
    assert ops.launch_count() == before
    gains[which] = buffer[8:]           # 16 bytes on
    call()
    ops.check_status()
