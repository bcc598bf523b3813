"""Rows behind the last drafted tree, and of requests whose numbers point outside: queries of zeros, caches as they were."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import tree_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (32, 8)])
@pytest.mark.parametrize("spare", [1, 7, 2000])        # few rows: several warps each
def test_queries_of_rows_without_a_request_are_zero(D, hq, hkv, spare):
    c = tree_batch([9, 0], [3, 4], hq, hkv, D, spare=spare)
    c["start"][1] = 10 ** 6             # the second request's rows belong to nobody
    g = torch.Generator().manual_seed(0)
    T = 7 + spare
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=g).cuda().to(torch.bfloat16)
    inv, k, v = torch.ones(D // 2, device="cuda"), c["k"].clone(), c["v"].clone()
    # what the result's memory held before: numbers that would show
    old = torch.full((T, hq, D), 7.0, device="cuda", dtype=torch.bfloat16)
    del old
    q = ops.tree_qk_norm_rope_kv_write(qkv, None, None, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], inv, c["k"], c["v"], hq,
                                       hkv, D, 1e-6)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert q[:3].abs().amax(-1).min() > 0 and (q[3:] == 0).all()
    mine = c["table"][int(c["req"][0]), 9:12].long()
    k[mine], v[mine] = c["k"][mine], c["v"][mine]
    assert torch.equal(k, c["k"]) and torch.equal(v, c["v"])
