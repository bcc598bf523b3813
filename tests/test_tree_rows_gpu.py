"""Prologue and cache rows of drafted token trees on the GPU against the formulas in 64 bits."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import exact_prologue, slots_of_rows, tree_batch

pytestmark = pytest.mark.gpu


def prologue(c, hq, hkv, D, half, norm=True, delta=None, seed=0, dtype=torch.bfloat16, strided=False, theta=1e6):
    g = torch.Generator().manual_seed(seed)
    T = c["q"].shape[0]
    width = (hq + 2 * hkv) * D
    qkv = (torch.randn(T, width + (16 if strided else 0), generator=g) * 1.5).cuda().to(dtype)[:, :width]
    gains = [(1 + 0.2 * torch.randn(D, generator=g)).cuda().to(dtype) if norm else None for _ in range(2)]
    inv = (theta ** -(torch.arange(half, dtype=torch.float64) / max(1, half))).float().cuda()
    d = None if delta is None else torch.tensor(delta, dtype=torch.int32, device="cuda")
    k0, v0, before = c["k"].clone(), c["v"].clone(), qkv.clone()
    q = ops.tree_qk_norm_rope_kv_write(qkv, *gains, c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], inv, c["k"], c["v"], hq,
                                       hkv, D, 1e-6, d)
    ops.check_status()
    assert torch.equal(qkv, before)
    want = exact_prologue(c, qkv, gains, inv, hq, hkv, 1e-6, delta)
    rows = sum(len(t) for t in c["trees"])
    loc = torch.tensor(slots_of_rows(c), device="cuda")

    def near(got, want):
        # one rounding to the type of what it goes into, and 32-bit arithmetic: the norm (4 roundings), the turn (3) of pairs whose
        # length is at most sqrt 2 of the larger, angles off by half a step of an angle of pi
        half = torch.finfo(got.dtype).eps / 2
        top = want.abs().amax(-1, keepdim=True)
        tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
        assert ((got.double() - want).abs() <= half * want.abs() + top * 2 ** -20 + tiny).all(), (got.double() - want).abs().max()

    near(q[:rows], want[0][:rows])
    near(c["k"][loc], want[1][:rows])
    near(c["v"][loc], want[2][:rows])
    k0[loc], v0[loc] = c["k"][loc], c["v"][loc]
    assert torch.equal(k0.view(torch.uint8) if k0.element_size() == 1 else k0, c["k"].view(torch.uint8) if k0.element_size() == 1 else c["k"])
    return q


@pytest.mark.parametrize("D,half", [(64, 32), (64, 8), (128, 64), (128, 16), (256, 128), (256, 32), (128, 0)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (32, 8)])
def test_prologue_sizes(D, half, hq, hkv):
    c = tree_batch([0, 1, 700, 31], [1, 33, 7, 150], hq, hkv, D, seed=D + half, spare=3, roots=2)
    prologue(c, hq, hkv, D, half, seed=half)


@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prologue_8bit_cache(cache, D):
    c = tree_batch([40, 3], [20, 9], 8, 2, D, cache=cache, dtype=torch.float16)
    prologue(c, 8, 2, D, D // 2, dtype=torch.float16)


def test_prologue_without_norm_far_positions_slot_major_strided():
    c = tree_batch([200, 5], [12, 40], 6, 3, 128, head_major=False, page=16)
    prologue(c, 6, 3, 128, 64, norm=False, delta=[1_000_003, -2], strided=True, theta=1e4)


def test_prologue_many_requests():
    c = tree_batch([i % 7 for i in range(75)], [1 + i % 5 for i in range(75)], 4, 2, 64)
    prologue(c, 4, 2, 64, 32)


def move(planes, D, slots, table, req, prefix, path, counts, dtype):
    g = torch.Generator().manual_seed(D)
    store = torch.randn(*planes, slots, D, generator=g).cuda().to(dtype)
    want = store.clone().view(-1, slots, D)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    want = want.view(torch.uint8)
    for b, r in enumerate(req):
        rows = table[r][prefix[b]:]
        old = want.clone()
        for i in range(counts[b]):
            want[:, rows[i]] = old[:, rows[path[b][i]]]
    ops.tree_kv_compact(store, ints(table), ints(req), ints(prefix), ints(path), ints(counts))
    ops.check_status()
    assert torch.equal(store.view(-1, slots, D).view(torch.uint8), want)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float8_e4m3fn, 128), (torch.float32, 256), (torch.bfloat16, 576)])
@pytest.mark.parametrize("planes", [(1,), (3, 2, 5)])
def test_rows_move_together(dtype, D, planes):
    table = [[0] * 60, list(range(50, 110)), list(range(49, 0, -1)) + [110] * 11, [111 + (7 * i) % 60 for i in range(60)]]
    path = [[0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [0, 2, 3, 4, 9, 10, 11, 12, 13, 20, 21, 40], [0, 5, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1],
            [3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14]]
    move(planes, D, 171, table, [3, 1, 2, 1], [0, 0, 4, 48], path, [12, 12, 2, 0], dtype)


def test_rows_of_bad_paths_stay():
    store = torch.randn(2, 30, 64, device="cuda", dtype=torch.bfloat16)
    before = store.clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = ints([list(range(1, 21))])
    for path in ([0, 0, 0], [0, 19, 20], [0, -1, 5]):
        ops.tree_kv_compact(store, table, ints([0]), ints([1]), ints([path]), ints([2 if path[1] <= 0 else 3]))
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status()
    ops.tree_kv_compact(store, table, ints([1]), ints([1]), ints([[0, 4, 5]]), ints([3]))
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert torch.equal(store, before)


def test_refusals_of_device_tensors():
    """What the binding refuses before anything is launched."""
    c = tree_batch([4, 2], [3, 2], 4, 2, 64)
    ix = (c["parents"], c["table"], c["req"], c["seq"], c["prefix"], c["start"])
    inv, qkv, n0 = torch.ones(32, device="cuda"), torch.zeros(5, 512, device="cuda", dtype=torch.bfloat16), ops.launch_count()

    def prologue(qkv=qkv, ix=ix, inv=inv, k=c["k"], v=c["v"], hq=4, hkv=2, hd=64, gain=None, delta=None):
        ops.tree_qk_norm_rope_kv_write(qkv, gain, None, *ix, inv, k, v, hq, hkv, hd, 1e-6, delta)

    def attention(q=c["q"], k=c["k"], v=c["v"], ix=ix, **kw):
        ops.attention_tree(q, k, v, *ix[1:], ix[0], 1.0, **kw)

    changed = lambda i, x: ix[:i] + (x,) + ix[i + 1:]  # noqa: E731
    short = changed(3, c["seq"][:1]), changed(0, c["parents"].long()), changed(1, c["table"].t()), changed(2, c["req"].cpu())
    calls = [lambda x=x: prologue(ix=x) for x in short] + [lambda x=x: attention(ix=x) for x in short]
    calls += [lambda: prologue(qkv=qkv.float()), lambda: prologue(qkv=qkv[:, :448]), lambda: prologue(hq=0, hkv=4), lambda: prologue(hq=8, hkv=0),
              lambda: prologue(hd=32), lambda: prologue(inv=inv[:5]), lambda: prologue(inv=inv.double()), lambda: prologue(k=c["k"][:, :1]),
              lambda: prologue(k=c["k"].half()), lambda: prologue(gain=torch.ones(64, device="cuda")), lambda: prologue(delta=inv[:2]),
              lambda: attention(q=c["q"][:, :0]), lambda: attention(q=c["q"][:, :3]), lambda: attention(q=c["q"].float()),
              lambda: attention(q=c["q"][..., :32]), lambda: attention(k=c["k"].half()), lambda: attention(v=c["v"][:-1]),
              lambda: attention(window=-1), lambda: attention(window=3, chunk=3), lambda: attention(sink=inv[:3]),
              lambda: attention(out=torch.empty_like(c["q"]).half())]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = dict(store=torch.zeros(2, 9, 4, device="cuda"), table=ints([[1, 2, 3, 4]]), req=ints([0]), prefix=ints([0]), path=ints([[0, 2]]), counts=ints([2]))
    calls += [lambda x=x: ops.tree_kv_compact(*{**rows, **x}.values())
              for x in (dict(store=torch.zeros(2, 9, 3, device="cuda")), dict(path=ints([0, 2])), dict(path=ints([[0, 2]]).long()),
                        dict(counts=ints([2, 2])), dict(prefix=ints([0]).cpu()))]
    f = lambda *n: torch.zeros(n, device="cuda")  # noqa: E731
    s = dict(logits=f(3, 8), tokens=f(3).long(), parents=ints([-1, 0, 0]), lens=ints([3]), start=ints([0]), t=f(1), k=ints([0]), p=f(1), m=None, u=f(3),
             uf=f(1), steps=3, draft=None)
    calls += [lambda x=x: ops.tree_speculative_sample(*{**s, **x}.values())
              for x in (dict(logits=f(8, 3).t()), dict(logits=f(3, 8).double()), dict(logits=f(3, 0)), dict(tokens=f(3)), dict(parents=ints([-1, 0])),
                        dict(lens=ints([3, 1])), dict(t=f(2)), dict(u=f(2)), dict(uf=f(3)), dict(steps=0), dict(draft=f(3, 7)),
                        dict(draft=f(3, 8).double()), dict(m=f(2)), dict(u=f(3).cpu()))]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert ops.launch_count() == n0


def test_parameters_for_all_requests_at_once():
    """Expanded vectors, other types."""
    g = torch.Generator().manual_seed(1)
    logits, u = torch.randn(4, 50, generator=g).cuda(), torch.rand(4, generator=g).cuda()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    fixed = (logits, torch.tensor([1, 2, 3, 4], device="cuda"), ints([-1, 0, -1, 0]), ints([2, 2]), ints([0, 2]))
    one = lambda x, t=torch.float32: torch.tensor([x], dtype=t, device="cuda").expand(2)  # noqa: E731
    a = ops.tree_speculative_sample(*fixed, one(0.5, torch.float64), one(9, torch.int64), one(0.75), one(0.0), u, u[:2], 2)
    b = ops.tree_speculative_sample(*fixed, one(0.5).contiguous(), ints([9, 9]), one(0.75).contiguous(), None, u, u[:2], 2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
