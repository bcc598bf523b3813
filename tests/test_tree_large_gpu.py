"""Batches of drafted token trees beyond the usual: more requests than a warp has lanes, trees that do not fit the kernels' shared copies of the
parents, nodes with more children than are looked at, and rows whose mass lies in small weights."""
import random

import pytest
import torch

from mllm_b200 import ops
from mllm_b200.ops import reference as ref
from tree_cases import exact_attention, exact_prologue, slots_of_rows, tree_batch

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def attend(c, **kw):
    out = torch.full_like(c["q"], 3.0)
    ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], out=out, **kw)
    ops.check_status()
    want, bound = exact_attention(c, bounds=True, **kw)
    assert ((out.double() - want).abs() <= bound).all(), (out.double() - want).abs().max()


@pytest.mark.parametrize("requests", [33, 64, 75, 200])
@pytest.mark.parametrize("hq,hkv,D", [(4, 2, 64), (8, 2, 128), (2, 1, 256)])
def test_many_requests(requests, hq, hkv, D):
    rng = random.Random(requests + D)
    attend(tree_batch([rng.choice([0, 1, 63, 64, 200]) for _ in range(requests)], [1 + (5 * i) % 9 for i in range(requests)], hq, hkv, D, seed=requests))


def test_many_requests_with_two_row_tiles_and_a_window():
    attend(tree_batch([(37 * i) % 300 for i in range(70)], [20 + i % 5 for i in range(70)], 8, 1, 128, seed=1), window=33)


def test_many_requests_some_without_nodes():
    c = tree_batch([10 + i for i in range(100)], [3] * 100, 4, 2, 128)
    none = list(range(0, 100, 3)) + [97, 98]
    c["seq"][none] = c["prefix"][none]
    out = torch.full_like(c["q"], 3.0)
    ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], out=out)
    ops.check_status()
    want, bound = exact_attention(c, bounds=True)
    rows = torch.tensor([b in none for b in range(100)], device="cuda").repeat_interleave(3)
    assert (out[rows] == 3).all() and ((out.double() - want).abs() <= bound)[~rows].all()


def deep(n, seed):
    """A chain with side branches, and some nodes that continue the cached text."""
    rng = random.Random(seed)
    return [-1] + [-1 if rng.random() < 0.02 else i - 1 if rng.random() < 0.8 else rng.randrange(i) for i in range(1, n)]


@pytest.mark.parametrize("nodes", [255, 256, 257, 300, 700])
@pytest.mark.parametrize("kw", [dict(), dict(window=70), dict(chunk=100)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_trees(nodes, kw, D):
    attend(tree_batch([90, 5], [nodes, 40], 2, 1, D, trees=[deep(nodes, nodes), deep(40, 1)], seed=nodes), **kw)


def test_prologue_of_large_trees():
    trees = [deep(600, 3), deep(129, 4)]
    c = tree_batch([1000, 3], [600, 129], 2, 1, 128, trees=trees)
    g = torch.Generator().manual_seed(0)
    qkv, gains = torch.randn(729, 4 * 128, generator=g).cuda().to(torch.bfloat16), [torch.ones(128, device="cuda", dtype=torch.bfloat16)] * 2
    inv = (1e4 ** -(torch.arange(64) / 64)).cuda()
    q = ops.tree_qk_norm_rope_kv_write(qkv, *gains, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], inv, c["k"], c["v"], 2, 1,
                                       128, 1e-6)
    ops.check_status()
    loc, half = torch.tensor(slots_of_rows(c), device="cuda"), torch.finfo(torch.bfloat16).eps / 2
    for got, want in zip((q, c["k"][loc], c["v"][loc]), exact_prologue(c, qkv, gains, inv, 2, 1, 1e-6)):
        # one rounding, and 32-bit arithmetic of pairs
        assert ((got.double() - want).abs() <= half * want.abs() + want.abs().amax(-1, keepdim=True) * 2 ** -20).all()


def walk(logits, tokens, parents, lens, starts, u, uf, steps, draft=None, t=1.0):
    B = len(lens)
    ones = torch.ones(B, device="cuda")
    args = (logits, tokens, ints(parents), ints(lens), ints(starts), ones * t, ints([0] * B), ones, None, u, uf, steps, draft)
    got = ops.tree_speculative_sample(*args)
    ops.check_status()
    want = ref.tree_speculative_sample(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want)), (got, want)
    return got


@pytest.mark.parametrize("nodes", [511, 512, 513, 1500])
def test_walks_through_large_trees(nodes):
    """The accepted way leads to the last nodes."""
    V, g = 300, torch.Generator().manual_seed(nodes)
    parents = deep(nodes, 7)
    way = [nodes - 1]
    while parents[way[-1]] >= 0:
        way.append(parents[way[-1]])
    way = way[::-1]
    if way[0] != 0:             # a chain that begins at the root
        parents[way[0]] = 0
        way = [0] + way
    logits = torch.randn(nodes, V, generator=g)
    tokens = torch.randint(0, V, (nodes,), generator=g)
    for a, b in zip(way, way[1:]):
        tokens[b] = logits[a].argmax()
    steps = len(way) + 3
    # greedy: a sibling in front of the way's node with its token would be taken instead, so the others get another one
    for j, up in enumerate(parents):
        if up >= 0 and j not in way:
            tokens[j] = (int(logits[up].argmax()) + 1) % V
    got = walk(logits.cuda(), tokens.cuda(), parents, [nodes], [0], torch.full((nodes,), 0.5, device="cuda"), torch.tensor([0.5], device="cuda"), steps,
               t=0.0)
    assert got[0][0, :len(way)].tolist() == way


@pytest.mark.parametrize("draft", [False, True])
def test_more_children_than_are_looked_at(draft):
    """64 children are looked at, in order; the 65th is not, however likely."""
    n, V = 90, 200
    logits = torch.full((n, V), -30.0)
    logits[:, 7] = 9.0
    logits[:, 100:] = 0.0
    for place, taken in ((63, True), (64, True), (65, False), (89, False)):
        tokens = torch.full((n,), 3)
        tokens[place] = 7
        q = torch.full((n, V), 1.0 / V).cuda() if draft else None
        got = walk(logits.cuda(), tokens.cuda(), [-1] + [0] * (n - 1), [n], [0], torch.full((n,), 0.9, device="cuda"), torch.tensor([0.1], device="cuda"),
                   3, q)
        assert (int(got[2][0]) == 2) == taken
        if taken:
            assert got[0][0].tolist() == [0, place, -1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("p", [1.0, 0.97])
def test_mass_in_small_weights(dtype, p):
    """Rows most of whose mass is in weights below 2^-12, which are 32-bit.  Each is off by at most 2^-22 from the exponential and 2^-19 from its
    argument (of up to 32, in 24 bits, twice), sums of a thread by 12 roundings of 2^-24: together less than 2^-18 of the mass, for a running sum
    and for the whole; top-p's cut adds as much again."""
    B, V = 64, 151936
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(B, V, generator=g)
    logits[:, 1000] = 13.0
    logits = logits.cuda().to(dtype)
    uf = torch.rand(B, generator=g).cuda()
    ones = torch.ones(B, device="cuda")
    _, out, counts = ops.tree_speculative_sample(logits, torch.zeros(B, dtype=torch.int64, device="cuda"), ints([-1] * B), ints([1] * B), ints(list(range(B))),
                                                 ones, ints([0] * B), ones * p, None, uf, uf, 1)
    ops.check_status()
    assert (counts == 1).all()
    slack = (3 if p < 1 else 2) * 2 ** -18
    for b in range(B):
        w = ref._kept_distribution(logits[b], 1.0, 0, p, 0.0)
        assert (torch.softmax(logits[b].double(), -1) * (logits[b] < 13 - 12 * 0.6931)).sum() > 0.3     # the tail that this is about
        sums, x = torch.cumsum(w, 0), int(out[b, 0])
        assert sums[x] - w[x] - slack <= uf[b] <= sums[x] + slack
