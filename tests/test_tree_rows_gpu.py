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
