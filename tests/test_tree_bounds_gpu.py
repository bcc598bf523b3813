"""Drafted token trees on the GPU: operands that the binding refuses because the kernels could not read them,
and numbers that they are not made for."""
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


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e-42, 1e39])
def test_scales_that_are_not_positive_are_refused(scale):
    c = tree_batch([70, 2], [3, 2], 4, 2, 64)
    args = (c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"])
    before = ops.launch_count()
    with pytest.raises(ValueError, match="scale"):
        ops.attention_tree(*args, scale)
    assert ops.launch_count() == before
    # the smallest that is taken: all weights alike
    got = ops.attention_tree(*args, 2.0 ** -126)
    ops.check_status()
    slots = c["table"][int(c["req"][0]), :71].long()
    want = c["v"][slots].double().mean(0).repeat_interleave(2, dim=0)
    half = torch.finfo(torch.bfloat16).eps / 2       # weights are 1, sums of 71 in 32 bits, one rounding
    assert ((got[0].double() - want).abs() <= half * want.abs() + c["v"][slots].double().abs().mean(0).repeat_interleave(2, dim=0) * 71 * 2 ** -24).all()


def test_more_planes_than_the_kernel_counts_are_refused():
    """They were a negative number of planes, and nothing was moved.  (Memory that nobody touches.)"""
    store = torch.empty((2 ** 31, 1, 8), device="cuda", dtype=torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    before = ops.launch_count()
    with pytest.raises(ValueError, match="too many"):
        ops.tree_kv_compact(store, ints([[0, 0, 0]]), ints([0]), ints([0]), ints([[0, 2]]), ints([2]))
    assert ops.launch_count() == before
    del store
    torch.cuda.empty_cache()
