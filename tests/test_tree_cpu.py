"""Drafted token trees on the CPU: the statements against the formulas, what is refused, and whole rounds of a tiny model."""
import pytest
import torch

from mllm_b200 import ops
from mllm_b200.layers.sampling import tree_speculative_sampling
from tree_cases import Round, exact_attention, exact_prologue, slots_of_rows, tree_batch


def attend(c, **kw):
    return ops.attention_tree(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["parents"], c["scale"], **kw)


@pytest.mark.parametrize("kw", [dict(), dict(window=5), dict(chunk=7), dict(logit_cap=3.0), dict(sink=torch.tensor([0.5, -1.0, 2.0, 0.0]))])
def test_attention_statement(kw):
    c = tree_batch([9, 0, 30], [7, 1, 12], 4, 2, 16, device="cpu", dtype=torch.float32, roots=2, spare=2)
    out = torch.full_like(c["q"], 9.0)
    attend(c, out=out, **kw)
    want = exact_attention(c, **kw)
    # sums of at most 42 fp32 products and weights
    assert (out[:20].double() - want[:20]).abs().max() <= 64 * 2 ** -23
    assert (out[20:] == 9).all()


def test_attention_statement_keeps_what_is_no_number_apart():
    c = tree_batch([3], [4], 2, 1, 8, device="cpu", dtype=torch.float32, trees=[[-1, 0, 0, 1]])
    slots = c["table"][int(c["req"][0])].long()
    c["v"][slots[5]] = float("nan")         # node 2, which nobody continues
    c["v"][slots[4]] = float("-inf")        # node 1, seen by node 3
    got = attend(c)
    assert torch.isfinite(got[0]).all() and torch.isnan(got[2]).all() and torch.isinf(got[[1, 3]]).all()


def test_prologue_statement():
    c = tree_batch([9, 0, 30], [7, 1, 12], 4, 2, 64, device="cpu", dtype=torch.float32, roots=2, spare=1)
    g = torch.Generator().manual_seed(0)
    qkv, gain = torch.randn(21, 8 * 64, generator=g), torch.randn(64, generator=g)
    inv = (1e4 ** -(torch.arange(16).double() / 16)).float()
    delta = torch.tensor([5, -9, 100000], dtype=torch.int32)
    q = ops.tree_qk_norm_rope_kv_write(qkv, gain, None, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], inv, c["k"], c["v"], 4,
                                       2, 64, 1e-6, delta)
    want = exact_prologue(c, qkv, (gain, None), inv, 4, 2, 1e-6, delta)
    loc = torch.tensor(slots_of_rows(c))
    for got, w in ((q[:20], want[0][:20]), (c["k"][loc], want[1][:20]), (c["v"][loc], want[2][:20])):
        assert (got.double() - w).abs().max() <= 2 ** -20 * w.abs().max()


def test_rows_statement_takes_them_in_order():
    store = torch.arange(2 * 10 * 4, dtype=torch.float32).view(2, 10, 4)
    want = store.clone()
    want[:, [4, 3]] = store[:, [3, 1]]      # node 1 <- node 2 (slot 3), node 2 <- node 4 (slot 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ops.tree_kv_compact(store, ints([[9, 5, 4, 3, 2, 1]]), ints([0]), ints([1]), ints([[0, 2, 4, 7]]), ints([3]))
    assert torch.equal(store, want)


def walk(probs, tokens, parents, u, u_final, draft=None, steps=4, **kw):
    n = len(tokens)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    args = dict(t=1.0, k=0, p=1.0, m=None)
    args.update(kw)
    path, out, count = ops.tree_speculative_sample(
        torch.log(torch.tensor(probs[:n])), torch.tensor(tokens), ints(parents), ints([n]), ints([0]), torch.tensor([args["t"]]), ints([args["k"]]),
        torch.tensor([args["p"]]), None if args["m"] is None else torch.tensor([args["m"]]), torch.tensor(u), torch.tensor([u_final]), steps,
        draft_probs=None if draft is None else torch.tensor(draft))
    c = int(count)
    assert (path[0, c:] == -1).all() and (out[0, c:] == -1).all()
    return path[0, :c].tolist(), out[0, :c].tolist()


def test_walks_by_hand():
    p = [[0.5, 0.3, 0.2]] * 4
    # candidates 1 and 0: 0.4 is not below p(1) = 0.3; without token 1, p(0) = 5 / 7.  At node 2 the candidate 2 falls to 0.9, which leaves
    # tokens 0 and 1
    assert walk(p, [0, 1, 0, 2], [-1, 0, 0, 2], [0, 0.4, 0.7, 0.9], 0.99) == ([0, 2], [0, 1])
    assert walk(p, [0, 1, 0, 2], [-1, 0, 0, 2], [0, 0.29, 0.7, 0.9], 0.0) == ([0, 1], [1, 0])
    assert walk(p, [0, 1, 0, 2], [-1, 0, 0, 2], [0, 0.4, 0.72, 0.9], 0.5) == ([0], [2])         # only token 2 is left
    # tokens drawn from q = (0.1, 0.8, 0.1): token 1 is taken below 0.3 / 0.8, and p - q leaves (0.4, 0, 0.1)
    q = [[0.1, 0.8, 0.1]] * 4
    assert walk(p, [0, 1, 1, 2], [-1, 0, 0, 2], [0, 0.37, 0.0, 0.9], 0.0, q)[0][:2] == [0, 1]
    # the second 1 has nothing left, and (0.8, 0, 0.2) - q, scaled, is (7/8, 0, 1/8)
    assert walk(p, [0, 1, 1, 2], [-1, 0, 0, 2], [0, 0.38, 0.0, 0.9], 0.87, q) == ([0], [0])
    assert walk(p, [0, 1, 1, 2], [-1, 0, 0, 2], [0, 0.38, 0.0, 0.9], 0.88, q) == ([0], [2])
    # filters: the two largest; no more than 0.45 of the mass in front; a tenth of the largest
    assert walk(p, [0], [-1], [0], 0.99, k=2) == ([0], [1])
    assert walk(p, [0], [-1], [0], 0.99, p=0.45) == ([0], [0])
    assert walk(p, [0], [-1], [0], 0.99, m=0.5) == ([0], [1])
    # greedy, and as many steps as are asked for
    assert walk(p, [0, 0, 0, 0], [-1, 0, 1, 2], [0.9] * 4, 0.9, t=0.0) == ([0, 1, 2, 3], [0, 0, 0, 0])
    assert walk(p, [0, 0, 0, 0], [-1, 0, 1, 2], [0.9] * 4, 0.9, t=0.0, steps=2) == ([0, 1], [0, 0])


def test_sampling_layer_draws_its_own_numbers():
    logits = torch.randn(6, 50, generator=torch.Generator().manual_seed(0))
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    args = (logits, torch.randint(0, 50, (6,)), ints([-1, 0, 0, -1, 0, 1]), ints([3, 3]), ints([0, 3]), 3)
    a, b = (tree_speculative_sampling(*args, temperature=0.7, top_k=10, top_p=0.9, seed=4) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and (a[2] >= 1).all()


def _case(name):
    c = tree_batch([4, 2], [3, 2], 4, 2, 16, device="cpu", dtype=torch.float32)
    inv = torch.ones(8)
    qkv = torch.randn(5, 8 * 16)
    calls = {
        "attention": lambda: attend(c, **kw),
        "prologue": lambda: ops.tree_qk_norm_rope_kv_write(qkv, None, None, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"],
                                                           inv, c["k"], c["v"], 4, 2, 16, 1e-6),
    }
    kw = {}
    return c, kw, calls[name]


@pytest.mark.parametrize("name", ["attention", "prologue"])
@pytest.mark.parametrize("key,change", [
    ("parents", lambda t: t.long()), ("parents", lambda t: t[:-1]), ("seq", lambda t: t[:1]), ("seq", lambda t: t.float()),
    ("prefix", lambda t: t.view(1, 2)), ("start", lambda t: t.long()), ("table", lambda t: t.long()), ("table", lambda t: t[0]),
    ("table", lambda t: t.t()), ("k", lambda t: t[..., :8]), ("k", lambda t: t.half()), ("v", lambda t: t[:-1]), ("k", lambda t: t.contiguous()),
])
def test_refused_indexes_and_caches(name, key, change):
    c, _, call = _case(name)
    call()
    c[key] = change(c[key])
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("change", [dict(window=-1), dict(chunk=-3), dict(window=4, chunk=4), dict(sink=torch.zeros(3)),
                                    dict(sink=torch.zeros(4).half()), dict(out=torch.zeros(5, 4, 8)), dict(out=torch.zeros(5, 4, 16).half())])
def test_refused_attention(change):
    c, kw, call = _case("attention")
    kw.update(change)
    with pytest.raises(ValueError):
        call()
    c, kw, call = _case("attention")
    c["q"] = c["q"][:, :3]
    with pytest.raises(ValueError):
        call()
    c["q"] = tree_batch([4, 2], [3, 2], 4, 2, 16, device="cpu", dtype=torch.float32)["q"].transpose(1, 2).contiguous().transpose(1, 2)
    with pytest.raises(ValueError):
        call()


def test_refused_prologue_rows_and_samples():
    c, _, _ = _case("prologue")
    ix = (c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"])
    good = dict(qkv=torch.randn(5, 128), gain=torch.ones(16), inv=torch.ones(8), delta=None)
    for change in (dict(qkv=torch.randn(5, 127)), dict(qkv=torch.randn(128, 5).t()), dict(gain=torch.ones(15)), dict(gain=torch.ones(16).half()),
                   dict(inv=torch.ones(9)), dict(inv=torch.ones(8).double()), dict(delta=torch.zeros(2)), dict(delta=torch.zeros(3, dtype=torch.int32))):
        a = {**good, **change}
        with pytest.raises(ValueError):
            ops.tree_qk_norm_rope_kv_write(a["qkv"], a["gain"], None, *ix, a["inv"], c["k"], c["v"], 4, 2, 16, 1e-6, a["delta"])
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    rows = dict(store=torch.zeros(2, 9, 4), table=ints([[1, 2, 3, 4]]), req=ints([0]), prefix=ints([0]), path=ints([[0, 2]]), counts=ints([2]))
    for change in (dict(store=torch.zeros(2, 9, 3)), dict(store=torch.zeros(9, 2, 4).transpose(0, 1)), dict(path=ints([0, 2])),
                   dict(path=ints([[0, 2]]).long()), dict(counts=ints([2, 2])), dict(prefix=ints([0, 0])), dict(path=ints([[0, 2], [0, 2]]))):
        with pytest.raises(ValueError):
            ops.tree_kv_compact(*{**rows, **change}.values())
    s = dict(logits=torch.randn(3, 8), tokens=torch.zeros(3, dtype=torch.int64), parents=ints([-1, 0, 0]), lens=ints([3]), start=ints([0]),
             t=torch.ones(1), k=ints([0]), p=torch.ones(1), m=None, u=torch.zeros(3), uf=torch.zeros(1), steps=3, draft=None)
    ops.tree_speculative_sample(*s.values())
    for change in (dict(logits=torch.randn(8, 3).t()), dict(logits=torch.randn(3, 8).double()), dict(tokens=torch.zeros(3)), dict(tokens=torch.zeros(2).long()),
                   dict(parents=ints([-1, 0])), dict(lens=ints([3, 1])), dict(t=torch.ones(2)), dict(u=torch.zeros(2)), dict(uf=torch.zeros(3)),
                   dict(steps=0), dict(draft=torch.zeros(3, 7)), dict(draft=torch.zeros(3, 8).double()), dict(m=torch.zeros(2))):
        with pytest.raises(ValueError):
            ops.tree_speculative_sample(*{**s, **change}.values())


def test_refused_numbers_of_heads():
    c, kw, call = _case("attention")
    c["q"] = c["q"][:, :0]
    with pytest.raises(ValueError):
        call()
    c, _, _ = _case("prologue")
    for hq, hkv in ((0, 4), (8, 0), (-4, 6)):       # the width of the rows fits
        with pytest.raises(ValueError):
            ops.tree_qk_norm_rope_kv_write(torch.randn(5, 128), None, None, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"],
                                           torch.ones(8), c["k"], c["v"], hq, hkv, 16, 1e-6)


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen2-tiny", "qwen3-moe-tiny"])
def test_rounds_of_a_model(preset):
    r = Round(preset, "cpu", "float32")
    # fp32 products of 256 to 512 terms through two layers, logits of some units
    r.check(lambda a, b: torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4))


def test_models_with_other_layers_refuse_trees():
    r = Round("qwen3.5-tiny", "cpu", "float32")
    with pytest.raises(ValueError, match="trees"):
        r.mr.prepare_forward_batch_tree(torch.zeros(2, dtype=torch.int64), torch.tensor([-1, 0]), torch.zeros(1, dtype=torch.int32), [2], [3])
    r = Round("qwen3-tiny", "cpu", "float32")
    with pytest.raises(ValueError, match="tree"):
        r.mr.prepare_forward_batch_tree(torch.zeros(2, dtype=torch.int64), torch.tensor([-1, 0]), torch.zeros(1, dtype=torch.int32), [3], [3])
