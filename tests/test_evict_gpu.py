"""Attention weights per cached token, selection and eviction on the GPU: against the formulas in 64 bits with derived bounds, whole numbers and
moved rows exactly; lengths around the tiles, odd groups, slots in any order, 8-bit caches, caps, sinks, empty requests, streams and graphs."""
import pytest
import torch

from evict_cases import Shortened, cached_batch, exact_decode, exact_prompt, plain_select
from mllm_b200 import ops
from mllm_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def decode(c, **kw):
    cap = kw.pop("cap", 0.0)
    return ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["scale"], c["sums"], logit_cap=cap, **kw)


def prompt(c, **kw):
    cap = kw.pop("cap", 0.0)
    ops.attention_prefill_weights(c["q"], c["k"], c["table"], c["req"], c["seq"], c["prefix"], c["start"], c["scale"], c["sums"], logit_cap=cap, **kw)


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    over = off - bound
    assert not torch.isnan(got).any() and over.max().item() <= 0, (what, off.max().item(), (off / bound.clamp(min=1e-300)).max().item())


def check_decode(c, sink=None, status=True, **kw):
    want, tol, sums, bound = exact_decode(c, kw.get("decay", 1.0), kw.get("cap", 0.0), sink)
    n0 = ops.launch_count()
    got = decode(c, sink=sink, **kw)
    if status:
        ops.check_status()
    assert ops.launch_count() > n0
    within(got, want, tol, "out")
    within(c["sums"], sums, bound, "sums")
    return got


def check_prompt(c, sink=None, status=True, **kw):
    sums, bound = exact_prompt(c, kw.get("last", 0), kw.get("add", False), kw.get("cap", 0.0), sink)
    prompt(c, sink=sink, **kw)
    if status:
        ops.check_status()
    within(c["sums"], sums, bound, "sums")


LENS = [[1], [2], [15], [16], [17], [63], [64], [65], [130], [1, 0, 64, 5, 0], [700, 33], [2500], [0]]


# ---------------------------------------------------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cache", [None, E4, E5])
@pytest.mark.parametrize("lens", LENS)
def test_decode_lengths(D, cache, lens):
    check_decode(cached_batch(lens, 8, 2, D, cache=cache, seed=len(lens) + D))


@pytest.mark.parametrize("hq,hkv,D", [(1, 1, 128), (3, 1, 128), (5, 1, 64), (7, 7, 128), (16, 2, 128), (9, 1, 128), (16, 1, 256), (18, 2, 128), (17, 1, 64),
                                      (32, 1, 128), (32, 1, 64), (40, 8, 128), (12, 3, 256)])
@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, E4), (torch.float16, E5)])
def test_decode_groups(hq, hkv, D, dtype, cache):
    check_decode(cached_batch([300, 20, 77], hq, hkv, D, dtype=dtype, cache=cache, seed=hq, page=16))


@pytest.mark.parametrize("kw", [dict(decay=0.9), dict(decay=0.0), dict(cap=5.0), dict(sink=True), dict(cap=2.0, sink=True, decay=0.5)])
@pytest.mark.parametrize("cache", [None, E4])
def test_decode_options(kw, cache):
    c = cached_batch([500, 64, 1, 4000], 8, 2, 128, cache=cache, seed=7)
    kw = dict(kw)
    check_decode(c, sink=c["sink"] if kw.pop("sink", False) else None, **kw)


@pytest.mark.parametrize("D,lens,hq,hkv", [(128, [2048] * 8, 32, 8), (64, [1900, 20, 3400, 700] * 7, 32, 8), (256, [20000, 3], 8, 2), (128, [100] * 200, 4, 1)])
def test_decode_many_tiles(D, lens, hq, hkv):
    """Several tiles in a row in every CTA, pairs cut between CTAs; twice, to the same bits."""
    c = cached_batch(lens, hq, hkv, D, page=16)
    first = c["sums"].clone()
    got = check_decode(c)
    once = c["sums"].clone()
    c["sums"].copy_(first)
    assert torch.equal(decode(c), got) and torch.equal(c["sums"], once)


def test_decode_weights_of_a_row_that_one_token_has():
    """One token carries nearly all of a row's weight: its sum is not off by the rounding to 16 bits, and neither are the others'."""
    c = cached_batch([400], 4, 1, 128, seed=2)
    slot = int(c["table"][int(c["req"][0]), 123])
    c["k"][slot] = (c["q"][0].float().sum(0) * 0.25).to(torch.bfloat16)
    check_decode(c)


def test_decode_strides_and_given_output():
    c = cached_batch([90, 300], 8, 2, 128, seed=9)
    row = torch.randn((2, 3 * 8 * 128), device="cuda").to(torch.bfloat16)
    row[:, 1024:2048] = c["q"].view(2, -1)
    c["q"] = row[:, 1024:2048].view(2, 8, 128)
    wide = torch.full((3, 3, 2, 400), 7.0, device="cuda")
    wide[:, 1, :, 3:3 + c["sums"].shape[2]] = c["sums"]
    c["sums"] = wide[:, 1, :, 3:3 + c["sums"].shape[2]]
    out = torch.full((2, 16, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    want, tol, sums, bound = exact_decode(c)
    decode(c, out=out[:, :8])
    ops.check_status()
    within(out[:, :8], want, tol, "out")
    within(c["sums"], sums, bound, "sums")
    assert (out[:, 8:] == 3).all() and (wide[:, 0] == 7).all() and (wide[:, 2] == 7).all() and (wide[:, 1, :, :3] == 7).all()
    assert (wide[:, 1, :, 3 + c["sums"].shape[2]:] == 7).all()


@pytest.mark.parametrize("where", ["slot", "negative slot", "row", "length"])
def test_decode_numbers_outside(where):
    c = cached_batch([200, 50], 4, 2, 128, seed=11)
    good = {k: v.clone() for k, v in c.items() if isinstance(v, torch.Tensor)}
    row = int(c["req"][0])
    if where == "slot":
        c["table"][row, 70] = c["k"].shape[0]
    elif where == "negative slot":
        c["table"][row, 199] = -0x7fffffff
    elif where == "row":
        c["req"][0] = 3
    else:
        c["seq"][0] = c["sums"].shape[2] + 1
    if where in ("slot", "negative slot"):
        check_decode(c, status=False)
    else:
        c["lens"] = [0, 50]
        check_decode(c, status=False)
        assert torch.equal(c["sums"][row], good["sums"][row])
    with pytest.raises(RuntimeError, match="index out of range"):
        ops.check_status()


def test_decode_values_that_are_no_numbers():
    c = cached_batch([100, 100, 64], 4, 2, 128, seed=12)
    # nobody's slots, and what stands behind the last token of a request
    c["k"][0] = float("nan")
    c["v"][0] = float("inf")
    want, tol, sums, bound = exact_decode(c)
    got = decode(c)
    within(got, want, tol, "out")
    slot = int(c["table"][int(c["req"][1]), 3])
    c["k"][slot, 1] = float("nan")           # one request, one kv head
    got = decode(c)
    ops.check_status()
    assert torch.isnan(got[1, 2:]).all() and not torch.isnan(got[1, :2]).any() and not torch.isnan(got[[0, 2]]).any()
    row = int(c["req"][1])
    assert torch.isnan(c["sums"][row, 1, :100]).all() and not torch.isnan(c["sums"][row, 0]).any() and not torch.isnan(c["sums"][row, 1, 100:]).any()


def test_decode_values_that_are_no_numbers_in_pairs_of_many_parts():
    c = cached_batch([9000, 50], 4, 2, 128, seed=15)
    slots = c["table"][int(c["req"][0])].long()
    c["k"][slots[:9000], 0] = float("nan")       # every part of the first kv head
    c["v"][slots[8000], 1] = float("inf")        # one part of the second
    got = decode(c, sink=c["sink"])
    ops.check_status()
    assert torch.isnan(got[0, :2]).all() and torch.isinf(got[0, 2:]).all() and not torch.isnan(got[1]).any()
    row = int(c["req"][0])
    assert torch.isnan(c["sums"][row, 0, :9000]).all() and not torch.isnan(c["sums"][row, 1]).any()


def test_decode_scores_of_minus_infinity():
    c = cached_batch([100], 4, 1, 128, seed=13, dtype=torch.float16)
    c["q"][:] = c["q"].abs() + 0.1
    slots = c["table"][int(c["req"][0])].long()
    c["k"][slots[5]] = float("-inf")
    before = c["sums"].clone()
    got = decode(c)
    ops.check_status()
    row = int(c["req"][0])
    assert not torch.isnan(got).any() and torch.equal(c["sums"][row, :, 5], before[row, :, 5])
    c["k"][slots[:100]] = float("-inf")      # nothing is left to see
    before = c["sums"].clone()
    got = decode(c)
    assert (got == 0).all() and torch.equal(c["sums"][row, :, :99], before[row, :, :99]) and (c["sums"][row, :, 99] == 0).all()


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_decode_queries_of_extreme_size_over_8_bit_caches(scale):
    """bf16 reaches further than fp16, in which the products over 8-bit rows run."""
    c = cached_batch([77], 4, 2, 64, cache=E4, seed=14)
    c["q"] = (c["q"].float() * scale).to(torch.bfloat16)
    c["q"][0, 1] = 0
    c["scale"] = c["scale"] / scale
    check_decode(c)


# ---------------------------------------------------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cache", [None, E4, E5])
@pytest.mark.parametrize("lens,new,last", [
    ([1], [1], 0), ([2], [1], 1), ([17], [17], 0), ([64], [64], 16), ([65], [65], 0), ([130], [2], 8), ([127, 128, 129], [127, 128, 129], 32),
    ([1, 0, 64, 5], [1, 0, 10, 0], 0), ([700, 33], [200, 33], 100), ([2500], [600], 64), ([300, 40], [300, 40], 0), ([1000, 257], [130, 257], 33),
])
def test_prompt_lengths(D, cache, lens, new, last):
    check_prompt(cached_batch(lens, 8, 2, D, cache=cache, seed=len(lens) + D, new=new), last=last)


@pytest.mark.parametrize("hq,hkv,D", [(1, 1, 128), (3, 1, 128), (5, 1, 64), (7, 7, 128), (16, 2, 128), (9, 1, 128), (16, 1, 256), (17, 1, 64), (32, 1, 128),
                                      (32, 1, 64), (40, 8, 128), (12, 3, 256)])
@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, E4), (torch.float16, E5)])
def test_prompt_groups(hq, hkv, D, dtype, cache):
    check_prompt(cached_batch([300, 20, 177], hq, hkv, D, dtype=dtype, cache=cache, seed=hq, page=16, new=[80, 20, 50]), last=40)


@pytest.mark.parametrize("kw", [dict(add=True), dict(cap=5.0), dict(sink=True), dict(cap=2.0, sink=True, add=True)])
@pytest.mark.parametrize("last", [0, 10])
def test_prompt_options(kw, last):
    c = cached_batch([500, 64, 1, 900], 8, 2, 128, seed=7, new=[100, 64, 1, 30])
    kw = dict(kw)
    check_prompt(c, sink=c["sink"] if kw.pop("sink", False) else None, last=last, **kw)


@pytest.mark.parametrize("D,lens,new,last,hq,hkv", [(128, [2048] * 8, [2048] * 8, 32, 32, 8), (128, [1400, 900], [1400, 900], 0, 16, 4),
                                                    (256, [9000, 3], [100, 3], 64, 8, 2), (64, [9000], [64], 64, 32, 8), (128, [50] * 100, [50] * 100, 7, 4, 1)])
def test_prompt_many_tiles(D, lens, new, last, hq, hkv):
    c = cached_batch(lens, hq, hkv, D, page=16, new=new)
    check_prompt(c, last=last)
    once = c["sums"].clone()
    prompt(c, last=last)
    assert torch.equal(c["sums"], once)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cache", [None, E4, E5])
@pytest.mark.parametrize("room", [256, 257])
@pytest.mark.parametrize("lens,new,last", [
    ([1], [1], 1), ([17], [17], 16), ([130], [2], 8), ([127, 128, 129], [127, 128, 129], 32), ([1, 0, 64, 5], [1, 0, 10, 0], 64), ([256, 33], [200, 33], 20),
    ([255, 31, 32, 33], [255, 31, 1, 30], 64), ([100] * 30, [100] * 30, 7),
])
def test_prompts_around_what_is_short(D, cache, room, lens, new, last):
    """Tables of 256 tokens and a few rows have a kernel of their own; the same requests in larger tables do not."""
    check_prompt(cached_batch(lens, 8, 2, D, cache=cache, seed=len(lens) + D, new=new, room=room), last=last)


@pytest.mark.parametrize("room", [250, 1000])
@pytest.mark.parametrize("hq,hkv,D,dtype,cache", [(1, 1, 128, torch.bfloat16, None), (5, 1, 64, torch.float16, None), (7, 7, 128, torch.bfloat16, E4),
                                                  (32, 1, 128, torch.float16, E5), (12, 3, 256, torch.bfloat16, None), (17, 1, 64, torch.bfloat16, E5)])
@pytest.mark.parametrize("kw", [dict(add=True), dict(cap=3.0), dict(sink=True), dict(cap=2.0, sink=True, add=True)])
def test_short_prompts_options(room, hq, hkv, D, dtype, cache, kw):
    c = cached_batch([200, 64, 1, 90], hq, hkv, D, dtype=dtype, cache=cache, seed=7, new=[100, 64, 1, 30], room=room)
    kw = dict(kw)
    check_prompt(c, sink=c["sink"] if kw.pop("sink", False) else None, last=8, **kw)


@pytest.mark.parametrize("scale", [1e-30, 1e30])
@pytest.mark.parametrize("room", [200, 300])
def test_prompt_queries_of_extreme_size_over_8_bit_caches(scale, room):
    c = cached_batch([77, 150], 4, 2, 64, cache=E4, seed=14, new=[20, 30], room=room)
    c["q"] = (c["q"].float() * scale).to(torch.bfloat16)
    c["q"][3, 1] = 0
    c["scale"] = c["scale"] / scale
    check_prompt(c, last=10)


@pytest.mark.parametrize("room", [None, 300])
@pytest.mark.parametrize("where", ["slot", "row", "length", "rows of q", "prefix", "lowest prefix"])
def test_prompt_numbers_outside(where, room):
    c = cached_batch([200, 50], 4, 2, 128, seed=11, new=[60, 20], room=room)
    row, before = int(c["req"][0]), c["sums"].clone()
    if where == "slot":
        c["table"][row, 70] = c["k"].shape[0]
    elif where == "row":
        c["req"][0] = -1
    elif where == "length":
        c["seq"][0] = c["sums"].shape[2] + 1
    elif where == "rows of q":
        c["start"][0] = 30
    else:
        c["prefix"][0] = -1 if where == "prefix" else -2 ** 31
    if where != "slot":
        c["new"][0] = 0
        q = c["q"]
        want, bound = exact_prompt(dict(c, q=q[60:]), 9)
        prompt(c, last=9)
        within(c["sums"], want, bound, "sums")
        assert torch.equal(c["sums"][row], before[row])
    else:
        check_prompt(c, last=9, status=False)
        assert (c["sums"][row, :, 70] == 0).all()
    with pytest.raises(RuntimeError, match="index out of range"):
        ops.check_status()


@pytest.mark.parametrize("room", [None, 300])
def test_prompt_values_that_are_no_numbers(room):
    c = cached_batch([100, 90, 64], 4, 2, 128, seed=12, new=[100, 20, 64], room=room)
    c["k"][0] = float("nan")                 # nobody's slot
    check_prompt(c, last=30)
    row = int(c["req"][0])
    slot = int(c["table"][row, 80])
    c["k"][slot, 1] = float("nan")           # seen by the queries from 80 on
    prompt(c, last=30)
    ops.check_status()
    assert torch.isnan(c["sums"][row, 1, :100]).all() and not torch.isnan(c["sums"][row, 0]).any()
    assert not torch.isnan(c["sums"][[int(r) for r in c["req"][1:]]]).any()
    prompt(c, last=0)
    assert torch.isnan(c["sums"][row, 1, :81]).all()
    c["k"][slot, 1] = 0
    c["q"][90, 2] = float("nan")             # a query: what stands behind it does not see it
    prompt(c, last=12)
    assert torch.isnan(c["sums"][row, 1, :91]).all() and not torch.isnan(c["sums"][row, 1, 91:]).any() and not torch.isnan(c["sums"][row, 0]).any()


@pytest.mark.parametrize("room", [None, 300])
def test_prompt_queries_without_a_visible_score(room):
    c = cached_batch([70], 4, 1, 64, seed=13, dtype=torch.float16, new=[70], room=room)
    c["q"][:] = c["q"].abs() + 0.1
    slots = c["table"][int(c["req"][0])].long()
    c["k"][slots[:10]] = float("-inf")       # the first ten queries see nothing
    prompt(c)
    ops.check_status()
    row = int(c["req"][0])
    got = c["sums"][row, 0, :70].double()
    assert not torch.isnan(got).any() and (got[:10] == 0).all() and abs(got.sum().item() - 60 * 4) < 1e-2


# ---------------------------------------------------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------------------------------------------------
def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("first,recent,pool", [(0, 0, 1), (4, 32, 1), (3, 0, 5), (0, 6, 3), (50, 50, 1), (2, 100, 7), (1, 1, 63)])
@pytest.mark.parametrize("kind", ["ties", "floats", "same", "special"])
def test_select(first, recent, pool, kind):
    g = torch.Generator().manual_seed(first + recent + pool)
    lens, budgets, req = [1, 300, 0, 1111, 64, 511, 513], [5, 120, 4, 333, 0, 511, 1], [3, 0, 7, 5, 1, 2, 6]
    shape = (2, 9, 3, 1200)
    sums = torch.randint(0, 6, shape, generator=g).float()
    if kind == "floats":
        sums = torch.exp(3 * torch.randn(shape, generator=g)) - 1.0
    elif kind == "same":
        sums.fill_(0.25)
    elif kind == "special":
        pick = torch.tensor([0.0, -0.0, float("nan"), float("inf"), float("-inf"), 1e-45, -1e-45, 3.0, -3.0, 3.4e38])
        sums = pick[torch.randint(0, len(pick), shape, generator=g)]
    keep, counts = ops.cache_select(sums.cuda(), i32(req), i32(lens), i32(budgets), 600, first=first, recent=recent, pool=pool)
    ops.check_status()
    want, want_counts = plain_select(sums, req, lens, budgets, 600, first, recent, pool)
    assert torch.equal(keep.cpu(), want) and torch.equal(counts.cpu(), want_counts)


@pytest.mark.parametrize("layers,lens,heads,keep_part,pool", [(1, [30001], 1, 0.1, 1), (1, [30000, 17, 9000], 2, 0.5, 7), (3, [8192, 8193], 8, 0.25, 7),
                                                             (1, [120000], 1, 0.02, 13), (36, [1200], 8, 0.4, 1), (2, [4095, 4096, 4097], 3, 0.9, 5)])
def test_select_long(layers, lens, heads, keep_part, pool):
    g = torch.Generator(device="cuda").manual_seed(5)
    sums = torch.exp(2 * torch.randn((layers, len(lens), heads, max(lens) + 3), generator=g, device="cuda"))
    sums = torch.where(torch.rand(sums.shape, generator=g, device="cuda") < 0.3, 0.125, sums)          # many equals
    budgets = [int(n * keep_part) for n in lens]
    args = (i32(list(range(len(lens)))), i32(lens), i32(budgets), max(budgets))
    keep, counts = ops.cache_select(sums, *args, pool=pool)
    want, want_counts = ref.cache_select(sums, *args, pool=pool)
    assert torch.equal(keep, want) and torch.equal(counts, want_counts)


def test_select_budgets_outside_and_strides():
    sums = torch.rand((4, 3, 5, 200), device="cuda")
    view = sums.transpose(0, 1)[1:, :, :, 7:]                # layers and rows change places
    args = (i32([2, 0]), i32([150, 90]), i32([-3, 40]), 64)
    keep, counts = ops.cache_select(view, *args)
    want, want_counts = ref.cache_select(view, *args)
    assert torch.equal(keep, want) and counts.tolist() == [0, 40] and torch.equal(counts, want_counts)
    ops.check_status()
    keep, counts = ops.cache_select(view, i32([1, 9]), i32([150, 90]), i32([100, 40]), 64)
    assert counts.tolist() == [64, 0] and (keep[:, 1] == -1).all()
    with pytest.raises(RuntimeError, match="index out of range"):
        ops.check_status()


# ---------------------------------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------------------------------
def moved(c, keep, counts):
    """What the call leaves, from the storage before it."""
    store, sums = c["store"].clone(), c["sums"].clone()
    for b, n in enumerate(counts.tolist()):
        if n <= 0:
            continue
        row = int(c["req"][b])
        slots = c["table"][row].long()
        for layer in range(store.shape[0]):
            for head in range(store.shape[2]):
                kept = keep[layer, b, head, :n].long()
                store.view(torch.uint8)[layer, :, head, slots[:n]] = c["store"].view(torch.uint8)[layer, :, head, slots[kept]]
                sums[layer, row, head, :n] = c["sums"][layer, row, head, kept]
    return store, sums


@pytest.mark.parametrize("lens,part", [([1], 1.0), ([2, 0, 9], 0.5), ([100, 1111, 64], 0.3), ([700], 0.99), ([5000, 3], 0.2), ([300] * 9, 0.6)])
@pytest.mark.parametrize("D,cache,page", [(128, None, 1), (64, E4, 16), (256, None, 16), (128, torch.float32, 1), (16, E5, 1)])
def test_evict(lens, part, D, cache, page):
    c = cached_batch(lens, 2, 2, D, cache=cache, page=page, seed=len(lens), layers=3)
    budgets = [max(1, int(n * part)) if n else 0 for n in lens]
    keep, counts = ops.cache_select(c["sums"], c["req"], c["seq"], i32(budgets), max(budgets), first=2, recent=5)
    store, sums = moved(c, keep, counts)
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, counts)
    ops.check_status()
    assert torch.equal(c["store"].view(torch.uint8), store.view(torch.uint8)) and torch.equal(c["sums"], sums)


@pytest.mark.parametrize("layers,D", [(20, 128), (40, 64), (40, 256), (120, 128)])
def test_evict_many_lists(layers, D):
    """With more lists rows are moved in larger pieces and shorter runs."""
    c = cached_batch([1, 70, 300, 129], 2, 2, D, seed=layers, layers=layers)
    keep, counts = ops.cache_select(c["sums"], c["req"], c["seq"], i32([1, 69, 170, 64]), 170, first=2, recent=5)
    store, sums = moved(c, keep, counts)
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, counts)
    ops.check_status()
    assert torch.equal(c["store"], store) and torch.equal(c["sums"], sums)


def test_evict_rows_that_are_read_where_others_are_written():
    """The token dropped stands in front: every row moves by one.  And rows that are kept more than once."""
    c = cached_batch([3000], 1, 1, 128, seed=1, layers=1)
    for keep in (torch.arange(1, 3000), torch.full((1500,), 2999), torch.arange(1500) * 2, torch.arange(1500).clamp(min=40) + 7):
        keep = keep.to(torch.int32).cuda().view(1, 1, 1, -1)
        counts = i32([keep.numel()])
        store, sums = moved(c, keep, counts)
        ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, counts)
        ops.check_status()
        assert torch.equal(c["store"], store) and torch.equal(c["sums"], sums)


def test_evict_without_sums_and_numbers_outside():
    c = cached_batch([50, 40], 2, 2, 64, seed=3, layers=2)
    keep, counts = ops.cache_select(c["sums"], c["req"], c["seq"], i32([20, 20]), 20)
    store, sums = moved(c, keep, counts)
    ops.cache_evict(c["store"], None, c["table"], c["req"], keep, counts)
    ops.check_status()
    assert torch.equal(c["store"], store)
    before = c["store"].clone()
    keep.fill_(0)                            # behind its place: left out
    keep[..., 0] = 10 ** 6
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, counts)
    assert torch.equal(c["store"], before)
    with pytest.raises(RuntimeError, match="index out of range"):
        ops.check_status()
    c["table"][int(c["req"][0]), 30] = -5    # a slot that is none: that row alone stays as it is
    keep, counts = torch.arange(20, 30, dtype=torch.int32, device="cuda").expand(2, 2, 2, 10).contiguous(), i32([10, 0])
    keep[..., 4] = 30
    ops.cache_evict(c["store"], c["sums"], c["table"], c["req"], keep, counts)
    slots = c["table"][int(c["req"][0])].long()
    assert torch.equal(c["store"][:, :, :, slots[4]], before[:, :, :, slots[4]]) and torch.equal(c["store"][:, :, :, slots[5]], before[:, :, :, slots[25]])
    with pytest.raises(RuntimeError, match="index out of range"):
        ops.check_status()


# ---------------------------------------------------------------------------------------------------------------------
# all of them
# ---------------------------------------------------------------------------------------------------------------------
def test_caches_behind_2_31_elements():
    """Slots whose rows lie more than 2^31 elements into the cache, and sums and storages of that size."""
    D, slots, heads = 128, 2 ** 24 + 4096, 1
    k = torch.zeros((heads, slots, D), dtype=torch.float16, device="cuda")
    c = cached_batch([400], 4, heads, D, dtype=torch.float16, seed=3, new=[50])
    far = torch.arange(slots - 400, slots, device="cuda")
    old = c["table"][int(c["req"][0]), :400].long()
    k[0, far] = c["k"][old, 0]
    one = torch.zeros((1, 2, heads, slots, D), dtype=torch.float16, device="cuda")
    one[0, 0] = k
    del k
    one[0, 1, 0, far] = c["v"][old, 0]
    c["k"], c["v"] = one[0, 0].transpose(0, 1), one[0, 1].transpose(0, 1)
    c["table"][int(c["req"][0]), :400] = far.to(torch.int32)
    check_prompt(c, last=20)
    c["q"] = c["q"][-1:].contiguous()
    check_decode(c)
    sums = c["sums"][None]
    keep, counts = ops.cache_select(sums, c["req"], c["seq"], i32([100]), 100)
    want = one[0, :, 0, far[keep[0, 0, 0].long()]].clone()
    ops.cache_evict(one, sums, c["table"], c["req"], keep, counts)
    ops.check_status()
    assert torch.equal(one[0, :, 0, far[:100]], want)


def test_sums_behind_2_31_elements():
    c = cached_batch([300], 4, 2, 64, seed=3, room=700)
    sums = torch.zeros((1, 2200, 2, 500000), device="cuda")
    sums[0, 2199, :, :700] = c["sums"][int(c["req"][0])]
    table = torch.zeros((2200, 700), dtype=torch.int32, device="cuda")
    table[2199] = c["table"][int(c["req"][0])]
    small = c["sums"].clone()
    got = ops.attention_decode_weights(c["q"], c["k"], c["v"], table, i32([2199]), c["seq"], c["scale"], sums[0])
    want = ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], c["scale"], small)
    assert torch.equal(got, want) and torch.equal(sums[0, 2199, :, :700], small[int(c["req"][0])])
    keep, counts = ops.cache_select(sums, i32([2199]), c["seq"], i32([90]), 90)
    again, _ = ops.cache_select(small[None], c["req"], c["seq"], i32([90]), 90)
    ops.check_status()
    assert torch.equal(keep, again) and int(counts) == 90


@pytest.mark.parametrize("room", [32, 300])
def test_the_most_requests(room):
    n, dev = 65535, "cuda"
    table = torch.zeros((n, room), dtype=torch.int32, device=dev)
    table[:, 0] = torch.arange(n, device=dev, dtype=torch.int32) % 999
    k = torch.randn((2, 999, 64), device=dev).to(torch.bfloat16).transpose(0, 1)
    q = torch.randn((n, 6, 64), device=dev).to(torch.bfloat16)
    ints = torch.arange(n, device=dev, dtype=torch.int32)
    one, none = torch.ones_like(ints), torch.zeros_like(ints)
    sums = torch.zeros((n, 2, room), device=dev)
    ops.attention_prefill_weights(q, k, table, ints.flip(0).contiguous(), one, none, ints, 0.125, sums, last=1)
    ops.check_status()
    assert (sums[:, :, 0] - 3).abs().max() < 1e-5 and (sums[:, :, 1:] == 0).all()
    ops.attention_decode_weights(q, k, k, table, ints, one, 0.125, sums)
    ops.check_status()
    assert (sums[:, :, 0] - 3).abs().max() < 1e-5 and (sums[:, :, 1:] == 0).all()
    more = torch.zeros(70000, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="too many"):
        ops.attention_prefill_weights(q, k, table, more, more, more, more, 0.125, sums, last=1)


def round_of(c, p, one, sums, budgets, width):
    """A prompt's weights, selection, eviction, and the next token over what is left."""
    ops.attention_prefill_weights(p["q"], p["k"], p["table"], p["req"], p["seq"], p["prefix"], p["start"], p["scale"], sums[0], last=8)
    keep, counts = ops.cache_select(sums, p["req"], p["seq"], budgets, width, first=2, recent=8, pool=3)
    ops.cache_evict(one, sums, p["table"], p["req"], keep, counts)
    out = ops.attention_decode_weights(c["q"], p["k"], p["v"], p["table"], p["req"], counts, p["scale"], sums[0])
    return keep, counts, out


@pytest.mark.parametrize("cache", [None, E4])
def test_a_run_of_them(cache):
    """All four in a row against the statements, on a stream of their own, and captured in a graph that is replayed on other data."""
    p = cached_batch([200, 77, 130], 8, 2, 128, cache=cache, seed=21, new=[200, 40, 130])
    c = cached_batch([1, 1, 1], 8, 2, 128, seed=22)
    one = torch.stack([p["k"].transpose(0, 1), p["v"].transpose(0, 1)])[None].contiguous()
    p["k"], p["v"] = one[0, 0].transpose(0, 1), one[0, 1].transpose(0, 1)
    sums, budgets = p["sums"][None].clone(), i32([64, 77, 33])
    start, start_sums = one.clone(), sums.clone()

    def statement():
        one.copy_(start)
        sums.copy_(start_sums)
        ops.force_torch(True)
        try:
            return [*round_of(c, p, one, sums, budgets, 80), one.clone(), sums.clone()]
        finally:
            ops.force_torch(False)

    def same(got, want):
        keep, counts, out, store, total = got
        assert torch.equal(counts, want[1])
        # a choice may turn where two scores differ in their last places only
        assert (keep != want[0]).float().mean() < 0.02
        if torch.equal(keep, want[0]):
            assert torch.equal(store.view(torch.uint8), want[3].view(torch.uint8))
            torch.testing.assert_close(total, want[4], rtol=2e-4, atol=1e-6)
        torch.testing.assert_close(out.float(), want[2].float(), rtol=0, atol=0.05)

    want = statement()
    one.copy_(start)
    sums.copy_(start_sums)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [*round_of(c, p, one, sums, budgets, 80), one.clone(), sums.clone()]
    side.synchronize()
    same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = round_of(c, p, one, sums, budgets, 80)
    for turn in range(2):
        if turn:
            p["q"].copy_(p["q"].flip(0))
            c["q"].copy_(c["q"].flip(1))
            want = statement()
        one.copy_(start)
        sums.copy_(start_sums)
        graph.replay()
        torch.cuda.synchronize()
        same([*held, one, sums], want)
    ops.check_status()


def test_two_calls_at_once():
    """Two streams, each with its own batch: workspaces are of a call alone."""
    batches = [cached_batch([900, 300], 8, 2, 128, seed=s, new=[100, 300]) for s in (1, 2)]
    for c in batches:
        c["rows"], c["q"] = c["q"], c["q"][:2].contiguous()
    want = []
    for c in batches:
        s = c["sums"].clone()
        want.append((decode(dict(c, sums=s)), s))
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, st in zip(batches, streams):
            with torch.cuda.stream(st):
                s = c["sums"].clone()
                got.append((decode(dict(c, sums=s)), s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_empty_batches():
    none = i32([])
    c = cached_batch([5], 4, 2, 64)
    p = cached_batch([5], 4, 2, 64, new=[5])
    before = c["sums"].clone()
    out = ops.attention_decode_weights(c["q"][:0], c["k"], c["v"], c["table"], none, none, 0.1, c["sums"])
    ops.attention_prefill_weights(p["q"][:0], p["k"], p["table"], none, none, none, none, 0.1, p["sums"])
    keep, counts = ops.cache_select(c["sums"][None], none, none, none, 3)
    one = torch.stack([c["k"].transpose(0, 1), c["v"].transpose(0, 1)])[None].contiguous()
    ops.cache_evict(one, c["sums"][None], c["table"], none, keep, counts)
    assert out.shape == (0, 4, 64) and keep.shape == (1, 0, 2, 3) and counts.numel() == 0 and torch.equal(before, c["sums"])
    keep, counts = ops.cache_select(c["sums"][None], c["req"], c["seq"], i32([0]), 0)
    assert keep.shape == (1, 1, 2, 0) and counts.tolist() == [0]


def test_refusals_on_the_device():
    from test_evict_cpu import refusals

    for call, message in refusals("cuda"):
        with pytest.raises(ValueError, match=message):
            call()
    c = cached_batch([40], 66, 2, 64)
    with pytest.raises(ValueError, match="groups of up to 32"):
        decode(c)
    with pytest.raises(ValueError, match="16-byte"):
        ops.attention_decode_weights(*(lambda c: (torch.randn(1, 4 * 64 + 4, device="cuda").to(torch.bfloat16)[:, 4:].view(1, 4, 64), c["k"], c["v"],
                                                  c["table"], c["req"], c["seq"], 0.1, c["sums"]))(cached_batch([40], 4, 2, 64)))
    with pytest.raises(ValueError, match="64, 128 or 256"):
        decode(cached_batch([40], 4, 2, 96))
    with pytest.raises(ValueError):
        decode(dict(cached_batch([40], 4, 2, 64), req=torch.zeros(1, dtype=torch.int32)))


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen3-moe-tiny"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_shortened_requests_of_a_model(preset, dtype):
    # both sides round some 12 tensors per layer to the activation type, half a step each, in two layers
    bound = 2 * 2 * 12 * torch.finfo(getattr(torch, dtype)).eps / 2
    before = ops.launch_count()

    def close(a, b):
        off = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert off <= bound, (off, bound)

    Shortened(preset, "cuda:0", dtype).check(close)
    assert ops.launch_count() > before
