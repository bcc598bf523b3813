"""Slots of shortened requests go back to the pool by whole pages: none that holds a kept token."""
import random

import pytest
import torch

from mllm_b200.configs import ServerConfig
from mllm_b200.executor import ModelRunner
from mllm_b200.mem_cache.memory_pool import TokenToKVPoolAllocator


@pytest.mark.parametrize("page,old,kept,still", [(16, 50, 20, 32), (16, 50, 32, 32), (16, 50, 0, 0), (16, 50, 50, 50), (16, 50, 49, 50), (1, 50, 20, 20), (4, 3, 1, 3)])
def test_pages_behind(page, old, kept, still):
    a = TokenToKVPoolAllocator(64 * 16, page)
    slots = a.alloc(old)
    before = a.available_size()
    assert a.free_behind(slots, kept) == still
    assert a.available_size() - before == (-(-old // page) - -(-kept // page)) * page
    taken = a.alloc(a.available_size())
    assert not set(taken.tolist()) & set(slots[:kept].tolist())


def test_pages_that_are_not_in_the_order_of_tokens():
    a = TokenToKVPoolAllocator(160, 16)
    pages = a.alloc(160).view(10, 16)
    # a page a token behind the prompt's pages, and a page that holds a kept and a dropped token
    slots = torch.cat([pages[3], pages[1][:2], pages[7][:1], pages[1][2:3], pages[8][:1]])
    assert a.free_behind(slots, 17) == 18
    assert sorted(set((a.alloc(32) // 16).tolist())) == [8, 9] and a.alloc(1) is None       # pages 7 and 8 of the pool, which begins with 1


def test_what_cannot_be_kept():
    a = TokenToKVPoolAllocator(160, 16)
    for kept in (-1, 6):
        with pytest.raises(ValueError, match="cannot keep"):
            a.free_behind(a.alloc(5), kept)


@pytest.mark.parametrize("page", [1, 16])
def test_others_write_into_what_was_given_back(page):
    """A request is cut from 50 to 20 tokens, its pages go back, others take all that is free and write there; its next token is as before."""
    mr = ModelRunner(ServerConfig(model_path="preset:qwen3-tiny", dtype="float32", max_running_requests=4, max_total_tokens=256, radix_cache_page_size=page),
                     device="cpu")
    mr.initialize()
    g = random.Random(3)
    table, alloc = mr.req_to_token_pool.req_to_token, mr.token_to_kv_pool_allocator
    (row,) = mr.req_to_token_pool.alloc(1)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    slots = alloc.alloc(50)
    table[row, :50] = slots.to(torch.int32)
    sums = mr.token_to_kv_pool.make_weight_sums(table.shape[0], 64)
    ids = torch.tensor([g.randrange(mr.vocab_size) for _ in range(50)])
    mr.forward(mr.prepare_forward_batch_extend(ids, ints(row), ints(50), ints(50), ints(0), slots, [50], [0], weight_sums=sums, weight_last=8))
    kept = int(mr.evict_cache(sums, ints(row), ints(50), ints(20), 20, first=2, recent=4))
    assert kept == 20
    still = alloc.free_behind(table[row, :50], kept)
    assert still == (20 if page == 1 else 32)
    loc = table[row, kept:kept + 1].long() if still > kept else alloc.alloc(1)
    table[row, kept] = int(loc)

    def step():
        fb = mr.prepare_forward_batch_decode(torch.tensor([7]), ints(row), ints(kept + 1), loc, max_seq_len=kept + 1, positions=ints(50))
        return mr.forward(fb).next_token_logits.clone()

    want = step()
    others = alloc.alloc(alloc.available_size())
    assert others.numel() >= 256 - 50
    mr.token_to_kv_pool.store[:, :, :, others] = 100.0
    torch.testing.assert_close(step(), want, rtol=0, atol=0)
