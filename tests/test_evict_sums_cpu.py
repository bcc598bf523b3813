"""Sums of attention weights that a batch does not fit are refused when it is made."""
import pytest
import torch

from evict_cases import Shortened


@pytest.fixture(scope="module")
def tiny():
    return Shortened("qwen3-tiny", "cpu", "float32")


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def decode(mr, n, sums, **kw):
    return mr.prepare_forward_batch_decode(torch.tensor([1]), i32(0), i32(n), torch.tensor([1]), weight_sums=sums, **kw)


def extend(mr, prefix, new, sums):
    return mr.prepare_forward_batch_extend(torch.ones(new, dtype=torch.int64), i32(0), i32(prefix + new), i32(new), i32(prefix),
                                           torch.arange(1, new + 1), weight_sums=sums)


def test_requests_longer_than_the_sums(tiny):
    mr = tiny.mr
    rows = mr.req_to_token_pool.req_to_token.shape[0]
    sums = mr.token_to_kv_pool.make_weight_sums(rows, 24)
    decode(mr, 24, sums, max_seq_len=24)
    extend(mr, 14, 10, sums)
    for call in (lambda: decode(mr, 25, sums, max_seq_len=25), lambda: extend(mr, 15, 10, sums), lambda: decode(mr, 3, sums)):
        with pytest.raises(ValueError, match="for 24 tokens"):
            call()
    decode(mr, 3, mr.token_to_kv_pool.make_weight_sums(rows, mr.context_len))


def test_sums_of_fewer_rows_or_other_heads(tiny):
    mr = tiny.mr
    layers, heads, rows = mr.token_to_kv_pool.layer_num, mr.token_to_kv_pool.kv_heads, mr.req_to_token_pool.req_to_token.shape[0]
    for shape in ((layers, rows - 1, heads, 24), (layers, rows, heads + 1, 24), (layers, rows, heads - 1, 24), (layers, rows, 24), (layers + 1, rows, heads, 24)):
        for call in (lambda s: decode(mr, 3, s, max_seq_len=3), lambda s: extend(mr, 0, 3, s)):
            with pytest.raises(ValueError, match="rows of the request table"):
                call(torch.zeros(shape))


def test_modules_are_looked_up_once(tiny):
    mr = tiny.mr
    sums = mr.token_to_kv_pool.make_weight_sums(mr.req_to_token_pool.req_to_token.shape[0], 24)
    decode(mr, 3, sums, max_seq_len=3)
    walk = mr.model.modules
    mr.model.modules = lambda: pytest.fail("a batch walks through the model")
    try:
        decode(mr, 3, sums, max_seq_len=3)
    finally:
        mr.model.modules = walk


@pytest.mark.parametrize("preset", ["pebulix-tiny", "lufizen-tiny", "kesovik-tiny"])
def test_caches_that_cannot_be_shortened(preset):
    mr = Shortened(preset, "cpu", "float32").mr
    with pytest.raises(ValueError, match="cannot be shortened"):
        mr.evict_cache(torch.zeros((2, 3, 2, 24)), i32(0), i32(20), i32(10), 10)
