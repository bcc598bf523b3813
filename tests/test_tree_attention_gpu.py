"""Attention of drafted token trees on the GPU against the formula in 64 bits: lengths around the tiles, odd trees and groups, slots in
any order, windows, chunks, caps, sinks, 8-bit caches, values that are no numbers, streams and captured graphs."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import exact_attention, tree_batch

pytestmark = pytest.mark.gpu


def check(case, **kw):
    c = tree_batch(**case)
    n0 = ops.launch_count()
    got = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], **kw)
    ops.check_status()
    assert ops.launch_count() > n0
    want, bound = exact_attention(c, bounds=True, **kw)
    over = (got.double() - want).abs() - bound
    assert not torch.isnan(got).any() and over.max().item() <= 0, ((got.double() - want).abs().max().item(), over.max().item())
    return c, got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("prefix,nodes", [
    ([0], [1]), ([0], [7]), ([1], [1]), ([63], [1]), ([64], [1]), ([60], [9]), ([127, 64, 1, 0], [1, 33, 64, 5]), ([700, 33], [65, 3]),
    ([1000], [130]), ([2500], [1]),
])
def test_lengths(D, prefix, nodes):
    check(dict(prefix=prefix, nodes=nodes, hq=8, hkv=2, D=D, seed=len(prefix) + D))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 1), (16, 1), (40, 8), (32, 4), (12, 3), (128, 1)])
def test_groups_of_heads(hq, hkv):
    check(dict(prefix=[300, 20], nodes=[17, 30], hq=hq, hkv=hkv, D=128, seed=hq))


@pytest.mark.parametrize("D,prefix,nodes,hq,hkv", [(128, [2048] * 8, [32] * 8, 32, 8), (64, [2048] * 8, [32] * 8, 32, 8), (256, [3000] * 4, [20] * 4, 8, 2)])
def test_long_runs_of_tiles(D, prefix, nodes, hq, hkv):
    """Several tiles in a row in every CTA, all CTAs at work: products and their waits overlap; twice, to the same bits."""
    c, got = check(dict(prefix=prefix, nodes=nodes, hq=hq, hkv=hkv, D=D, page=16))
    again = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"])
    assert torch.equal(got, again)


@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("prefix,nodes,hq,hkv,kw", [
    ([500], [33], 4, 1, {}),                                  # one row over a tile
    ([0, 64], [43, 43], 3, 1, {}),                            # 42 nodes a tile: 126 rows
    ([700, 0, 100], [64, 64, 64], 8, 2, {}),                  # two full tiles
    ([200, 3000], [65, 64], 4, 1, {}),                        # a third tile of one node
    ([900, 10, 0, 77], [150, 1, 0, 9], 4, 2, {}),             # one tree above a tile, the others far below
    ([300, 129], [70, 40], 16, 2, dict(window=50)),
    ([300, 129], [70, 40], 16, 2, dict(chunk=64, logit_cap=4.0)),
    ([1000], [2], 128, 1, {}),                                # a node per tile
    ([2048] * 8, [48] * 8, 32, 8, {}),
])
def test_two_row_tiles_side_by_side(cache, prefix, nodes, hq, hkv, kw):
    """More rows of a kv head than a tile of 128 holds, on average: a CTA takes two of them through the same keys and values."""
    c, got = check(dict(prefix=prefix, nodes=nodes, hq=hq, hkv=hkv, D=128, cache=cache, seed=len(nodes)), **kw)
    again = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], **kw)
    assert torch.equal(got, again)


def test_two_row_tiles_with_values_that_are_no_numbers():
    c = tree_batch([100], [80], 4, 2, 128, trees=[[-1] + list(range(79))])
    slots = c["table"][int(c["req"][0])].long()
    c["v"][slots[170]] = float("nan")                        # node 70, seen by those from 70 on
    c["k"][slots[175]] = float("nan")
    got = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"])
    ops.check_status()
    assert torch.isnan(got[70:]).all()
    c["v"][slots[170]] = 0
    c["k"][slots[175]] = 0
    want, bound = exact_attention(c, bounds=True)
    assert ((got[:70].double() - want[:70]).abs() <= bound[:70]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=37), dict(window=130), dict(window=5000), dict(chunk=64), dict(chunk=100), dict(chunk=7),
                                dict(logit_cap=2.5), dict(window=70, logit_cap=30.0)])
def test_windows_chunks_caps(D, kw):
    check(dict(prefix=[0, 300, 129, 1000], nodes=[40, 9, 70, 1], hq=6, hkv=2, D=D, seed=D, roots=2), **kw)


@pytest.mark.parametrize("D,window", [(64, None), (128, 50), (256, None)])
def test_sinks(D, window):
    sink = torch.randn(8, generator=torch.Generator().manual_seed(1)).cuda() * 3
    check(dict(prefix=[3, 700, 0], nodes=[5, 30, 2], hq=8, hkv=4, D=D), sink=sink, window=window)


@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_8bit_caches(cache, D, dtype):
    check(dict(prefix=[200, 0, 1500], nodes=[20, 3, 33], hq=8, hkv=2, D=D, cache=cache, dtype=dtype))
    check(dict(prefix=[90, 600], nodes=[70, 1], hq=4, hkv=4, D=D, cache=cache, dtype=dtype, page=16), window=64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_major,page", [(True, 16), (False, 1), (False, 16)])
def test_layouts(dtype, head_major, page):
    check(dict(prefix=[500, 60, 17], nodes=[12, 64, 31], hq=16, hkv=4, D=128, dtype=dtype, head_major=head_major, page=page))


def test_rows_in_wider_tensors_and_behind_the_last_tree():
    c = tree_batch([70, 9], [11, 6], 8, 2, 128, spare=5)
    q = torch.randn(22, 12, 128, device="cuda").to(torch.bfloat16)
    q[:, 2:10] = c["q"]
    out = torch.full((22, 10, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    got = ops.attention_tree(q[:, 2:10], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"],
                             out=out[:, 1:9])
    ops.check_status()
    want, bound = exact_attention(c, bounds=True)
    assert got.data_ptr() == out[:, 1:9].data_ptr()
    assert ((got[:17].double() - want[:17]).abs() <= bound[:17]).all()
    assert (out[17:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 9] == 7).all()


def test_scores_that_grow():
    """Maxima that rise along the sequence: the rows of O are scaled down in place."""
    c = tree_batch([900], [30], 4, 2, 128)
    slots = c["table"][int(c["req"][0]), :930].long()
    c["k"][slots] = (c["k"][slots].float() * torch.linspace(0.1, 12.0, 930, device="cuda").view(-1, 1, 1)).to(torch.bfloat16)
    got = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"])
    want, bound = exact_attention(c, bounds=True)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("cache", [None, torch.float8_e5m2])
@pytest.mark.parametrize("window", [None, 40])
def test_values_that_are_no_numbers_reach_who_sees_them(cache, window):
    """NaN and infinities in the keys and values of a node, of a token outside the window and of slots of no request."""
    c = tree_batch([100], [12], 4, 2, 128, cache=cache, trees=[[-1, 0, 0, 1, 1, 2, 2, 3, 5, 5, 8, 0]])
    slots = c["table"][int(c["req"][0])].long()
    others = torch.ones(c["slots"], dtype=torch.bool)
    others[slots[:112].cpu()] = False
    bad = lambda t, i, x: t.index_put_((torch.as_tensor(i, device="cuda"),), torch.full_like(t[:1].float(), x).to(t.dtype))  # noqa: E731
    clean = [c["k"].clone(), c["v"].clone()]
    idle = torch.nonzero(others)[:, 0].cuda()
    c["v"][idle] = torch.full((len(idle), 2, 128), float("nan"), device="cuda").to(c["v"].dtype)
    c["k"][idle] = torch.full((len(idle), 2, 128), float("inf"), device="cuda").to(c["k"].dtype)
    bad(c["v"], slots[106:107], float("nan"))       # node 6 alone (a leaf)
    bad(c["v"], slots[103:104], float("inf"))       # node 3, seen by node 7
    bad(c["k"], slots[111:112], float("nan"))       # node 11, a leaf
    if window:
        bad(c["v"], slots[10:11], float("nan"))     # in front of every window
    got = ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], window=window)
    ops.check_status()
    c["k"], c["v"] = clean
    want, bound = exact_attention(c, bounds=True, window=window)
    fine = [0, 1, 2, 4, 5, 8, 9, 10]
    assert ((got[fine].double() - want[fine]).abs() <= bound[fine]).all()
    assert torch.isnan(got[6]).all() and torch.isnan(got[11]).all()
    assert torch.isinf(got[[3, 7]]).all()


def test_indexes_outside_the_tensors():
    """Slots, parents and requests that point outside: recorded, and left out."""
    def run(**change):
        c = tree_batch([50, 20], [6, 4], 4, 2, 64)
        for k, (i, x) in change.items():
            c[k].view(-1)[i] = x
        out = torch.full_like(c["q"], 3.0)
        ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], out=out)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status()
        return c, out

    c, out = run(table=(int(tree_batch([50, 20], [6, 4], 4, 2, 64)["req"][1]) * 61 + 3, 10 ** 6))
    c, out = run(parents=(2, 2))
    c, out = run(parents=(7, 100))
    for k, x in (("req", 9), ("req", -1), ("start", 7), ("start", -3), ("seq", 10 ** 6), ("prefix", -5)):
        c, out = run(**{k: (1, x)})
        assert (out[6:] == 3).all() and not (out[:6] == 3).any(), k


def test_empty_batches():
    c = tree_batch([4, 9], [3, 2], 4, 2, 64)
    c["seq"][0] = 4
    out = torch.full_like(c["q"], 3.0)
    args = (c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"])
    ops.attention_tree(c["q"], *args, c["parents"], c["scale"], out=out)
    assert (out[:3] == 3).all() and not (out[3:] == 3).any()
    got = ops.attention_tree(c["q"][:0], *args[:3], *(t[:0] for t in args[3:]), c["parents"][:0], c["scale"])
    ops.check_status()
    assert got.shape == (0, 4, 64)


def test_another_stream_and_two_graphs():
    """Captured calls on a side stream, replayed in turn with others' work in between: each graph has a workspace of its own."""
    cs = [tree_batch([1500] * 4, [16] * 4, 8, 2, 128, seed=s) for s in range(2)]
    run = lambda c: ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"])  # noqa: E731
    want = [run(c) for c in cs]
    side, graphs, outs = torch.cuda.Stream(), [], []
    side.wait_stream(torch.cuda.current_stream())
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(run(c))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    with torch.cuda.stream(side):
        got = run(cs[0])
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want[0]) and torch.equal(outs[1], want[1])
    # a replayed graph reads the lengths again
    cs[0]["seq"].sub_(1)
    outs[0].fill_(5)
    graphs[0].replay()
    torch.cuda.synchronize()
    ops.check_status()
    assert (outs[0].view(4, 16, 8, 128)[:, 15] == 5).all() and torch.equal(outs[0].view(4, 16, 8, 128)[:, :15], want[0].view(4, 16, 8, 128)[:, :15])
