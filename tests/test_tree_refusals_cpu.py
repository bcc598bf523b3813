"""Calls of the operators for drafted token trees that are refused, on the CPU."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import Round, tree_batch


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e-42, 1e39])
def test_refused_scales(scale):
    c = tree_batch([4, 2], [3, 2], 4, 2, 16, device="cpu", dtype=torch.float32)
    args = (c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"])
    ops.attention_tree(*args, 0.25)
    with pytest.raises(ValueError, match="scale"):
        ops.attention_tree(*args, scale)


def test_models_without_kernels_for_trees_are_refused_when_the_batch_is_made(monkeypatch):
    """On the GPU, before anything runs; here the runner believes that it is on one."""
    mr = Round("qwen3-tiny", "cpu", "float32").mr

    def make():
        return mr.prepare_forward_batch_tree(torch.zeros(2, dtype=torch.int64), torch.tensor([-1, 0], dtype=torch.int32),
                                             torch.zeros(1, dtype=torch.int32), [2], [3])

    make()
    monkeypatch.setattr(ops, "use_kernels", lambda t: True)
    with pytest.raises(ValueError, match="float32"):
        make()
    for dtype, cache, dim, fine in ((torch.bfloat16, torch.bfloat16, 128, True), (torch.float16, torch.float8_e5m2, 64, True),
                                    (torch.bfloat16, torch.float8_e4m3fn, 256, True), (torch.bfloat16, torch.bfloat16, 96, False),
                                    (torch.bfloat16, torch.float16, 128, False)):
        mr.dtype, mr.kv_cache_dtype, mr.head_dim = dtype, cache, dim
        if fine:
            make()
        else:
            with pytest.raises(ValueError, match=str(dim)):
                make()


def test_batches_outside_the_request_table_are_refused():
    mr = Round("qwen3-tiny", "cpu", "float32").mr
    room = mr.req_to_token_pool.req_to_token.shape[1]
    ids, parents, one = torch.zeros(2, dtype=torch.int64), torch.tensor([-1, 0], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    mr.prepare_forward_batch_tree(ids, parents, one, [2], [room - 2])
    for rows, lens, prefix in ((one, [2], [room - 1]), (one, [2], [-1]), (one.repeat(2), [2], [3]), (one.repeat(2), [3, -1], [3, 3])):
        with pytest.raises(ValueError, match="table"):
            mr.prepare_forward_batch_tree(ids, parents, rows, lens, prefix)
