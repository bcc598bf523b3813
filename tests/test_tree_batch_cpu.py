"""Batches of drafted token trees, as the model runner makes them."""
import torch

from tree_cases import Round


def test_new_tokens_have_the_slots_of_their_nodes():
    """Whatever a layer writes by ``out_cache_loc`` goes where the request table has the nodes."""
    r = Round("qwen3-tiny", "cpu", "float32")
    table = r.mr.req_to_token_pool.req_to_token
    rows = [r.mr.req_to_token_pool.alloc(1)[0] for _ in range(3)]
    lens, trees = [5, 0, 9], [[-1, 0, 0], [], [-1, 0]]
    for row, n, t in zip(rows, lens, trees):
        table[row, :n + len(t)] = r._alloc(n + len(t)).flip(0).to(torch.int32) if n + len(t) else 0
    fb = r.mr.prepare_forward_batch_tree(torch.zeros(5, dtype=torch.int64), torch.tensor([p for t in trees for p in t]),
                                         torch.tensor(rows, dtype=torch.int32), [len(t) for t in trees], lens)
    want = [int(table[row, n + j]) for row, n, t in zip(rows, lens, trees) for j in range(len(t))]
    assert fb.out_cache_loc.dtype == torch.int64 and fb.out_cache_loc.tolist() == want
