"""Attention of drafted token trees over request tables that point outside the cache: such tokens are recorded, and seen by nobody."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import tree_batch, ways_of

pytestmark = pytest.mark.gpu


def exact(c, window=None, sink=None):
    """The definition in 64 bits without the tokens whose slots lie outside, and per element the largest error of a kernel that rounds weights and
    results to the activation type (half a step each) and forms scores in 32 bits (D roundings of the sum of |q k|, and 2^-21 of the
    exponential, twice)."""
    q = c["q"].double()
    want, bound = torch.zeros_like(q), torch.zeros_like(q)
    hkv, D = c["k"].shape[1], q.shape[2]
    half = torch.finfo(c["q"].dtype).eps / 2
    for b, parents in enumerate(c["trees"]):
        pl, qs = int(c["prefix"][b]), int(c["start"][b])
        slots = c["table"][int(c["req"][b])].tolist()
        for i, way in enumerate(ways_of(parents)):
            low = max(0, pl + len(way) - window) if window else 0
            see = list(range(low, pl)) + [pl + node for up, node in enumerate(way) if pl + up >= low]
            see = [s for s in (slots[x] for x in see) if 0 <= s < c["slots"]]
            if not see:
                continue
            kk, vv = c["k"][see].double(), c["v"][see].double()
            x = q[qs + i].view(hkv, -1, D)
            s = torch.einsum("kgd,lkd->kgl", x, kk) * c["scale"]
            span = torch.einsum("kgd,lkd->kgl", x.abs(), kk.abs()).amax().item() * c["scale"]
            if sink is not None:
                s = torch.cat([s, sink.double().view(hkv, -1, 1)], dim=-1)
            w = torch.softmax(s, dim=-1)[..., :len(see)]
            o, reach = (torch.einsum("kgl,lkd->kgd", w, t).reshape(-1, D) for t in (vv, vv.abs()))
            want[qs + i] = o
            bound[qs + i] = half * (o.abs() + reach) + reach * 2 * (D * 2 ** -24 * span + 2 ** -21)
    return want, bound


def run(c, **kw):
    out = torch.full_like(c["q"], 3.0)
    ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], out=out, **kw)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    want, bound = exact(c, kw.get("window"), kw.get("sink"))
    assert ((out.double() - want).abs() <= bound).all(), (out.double() - want).abs().max()


def spoil(c, b, places):
    """Slots in front of the cache, right behind it and far away."""
    for n, at in enumerate(places):
        c["table"][int(c["req"][b]), at] = (-1, c["slots"], 10 ** 6, 2 ** 31 - 1, -2 ** 31)[n % 5]


@pytest.mark.parametrize("hq,hkv,D,nodes", [(4, 2, 64, 9), (4, 2, 128, 9), (4, 2, 256, 9), (8, 1, 128, 33)])      # the last: two row tiles
@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("kw", [dict(), dict(window=50), dict(sink=True)])
def test_tokens_without_a_slot(hq, hkv, D, nodes, cache, kw):
    c = tree_batch([300, 20, 700], [nodes, 4, nodes - 2], hq, hkv, D, cache=cache, seed=D + nodes)
    if kw.get("sink"):
        kw = dict(sink=torch.linspace(-2, 2, hq, device="cuda"))
    spoil(c, 0, [0, 5, 64, 127, 128, 270, 271, 299, 300 + 2, 300 + nodes - 1])
    spoil(c, 1, [3])
    spoil(c, 2, list(range(128, 192)) + [699, 701])          # a whole tile
    run(c, **kw)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sink", [None, 0.5, float("-inf")])
def test_nodes_that_see_nothing(D, sink):
    trees = [[-1, 0, -1], [-1, 0], [-1, 0, 0]]
    c = tree_batch([0, 0, 200], [3, 2, 3], 4, 2, D, trees=trees)
    spoil(c, 0, [0, 1])             # node 2 sees itself
    spoil(c, 2, list(range(203)))
    run(c, sink=None if sink is None else torch.full((4,), sink, device="cuda"))


@pytest.mark.parametrize("slot", [-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 2, -2])
@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn])
def test_any_negative_slot(slot, cache):
    c = tree_batch([130], [5], 4, 2, 128, cache=cache)
    c["table"][int(c["req"][0]), [2, 40, 100, 132]] = slot
    run(c)
