"""Verification of drafted token trees where logits are infinite, absent or equal, and where most of the mass lies in small weights."""
import pytest
import torch

from mllm_b200 import ops
from mllm_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def both(logits, tokens, parents, u, u_final, draft=None, t=1.0, k=0, p=1.0, m=0.0, steps=3):
    """One tree; the kernel's answer, which has to be the statement's."""
    f = lambda x: torch.tensor(x, device="cuda", dtype=torch.float32)  # noqa: E731
    args = (logits, torch.tensor(tokens, device="cuda"), ints(parents), ints([len(tokens)]), ints([0]), f([t]), ints([k]), f([p]), f([m]), f(u),
            f([u_final]), steps, draft)
    got = ops.tree_speculative_sample(*args)
    ops.check_status()
    want = ref.tree_speculative_sample(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want)), (got, want)
    n = int(got[2])
    return got[0][0, :n].tolist(), got[1][0, :n].tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kw", [dict(), dict(m=0.5), dict(t=0.5), dict(k=5), dict(p=0.9), dict(k=1), dict(t=30.0)])
def test_two_infinite_logits_share_the_mass(dtype, kw):
    V = 20000
    logits = torch.randn(2, V, generator=torch.Generator().manual_seed(0)).cuda().to(dtype)
    logits[0, [70, 15000]] = INF
    logits[0, 71] = torch.finfo(dtype).max
    logits[1, 3] = 60.0
    # a picked candidate: taken below a half (what comes behind it is for the statement to say: a temperature of 30 leaves row 1 flat)
    path, out = both(logits, [0, 15000], [-1, 0], [0, 0.49], 0.2, **kw)
    assert path == [0, 1] and out[0] == 15000
    assert both(logits, [0, 15000], [-1, 0], [0, 0.51], 0.2, **kw) == ([0], [70])
    assert both(logits, [0, 71], [-1, 0], [0, 0.0], 0.6, **kw) == ([0], [15000])
    # a drawn one: taken below 0.5 / 0.8, and p - q leaves the other token
    q = torch.zeros(2, V, device="cuda")
    q[0, 70], q[0, 9] = 0.8, 0.2
    path, out = both(logits, [0, 70], [-1, 0], [0, 0.62], 0.2, q, **kw)
    assert path == [0, 1] and out[0] == 70
    assert both(logits, [0, 70], [-1, 0], [0, 0.63], 0.2, q, **kw) == ([0], [15000])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kw", [dict(), dict(p=0.7), dict(k=4500), dict(k=4500, p=0.7), dict(k=12, p=0.1)])
def test_more_infinite_logits_than_are_sorted(dtype, kw):
    V, n = 40000, 5000
    logits = torch.randn(2, V, generator=torch.Generator().manual_seed(1)).cuda().to(dtype)
    places = torch.randperm(V, generator=torch.Generator().manual_seed(2))[:n].sort().values
    logits[0, places.cuda()] = INF
    token = int(places[n // 2])
    assert both(logits, [0, token], [-1, 0], [0, 1.5 / n], 0.5, **kw)[0] == [0]
    assert both(logits, [0, token], [-1, 0], [0, 0.5 / n], 0.5, **kw)[1][0] == token
    assert both(logits[:1], [0], [-1], [0], 10.5 / n, steps=1, **kw) == ([0], [int(places[10])])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t", [0.0, 1.0])
def test_rows_without_a_finite_logit_give_their_first_token(dtype, t):
    V = 17000
    for fill, other, places in ((NAN, -INF, range(1, V)), (-INF, NAN, range(1, 9000)), (-INF, NAN, [0]), (NAN, NAN, [0]), (NAN, -INF, [V - 1])):
        logits = torch.full((2, V), fill, device="cuda", dtype=dtype)
        logits[:, list(places)] = other
        for kw in (dict(), dict(k=7), dict(p=0.5)):
            assert both(logits, [0, 0], [-1, 0], [0, 0.5], 0.9, t=t, **kw) == ([0, 1], [0, 0])
            assert both(logits, [0, 1], [-1, 0], [0, 0.5], 0.9, t=t, **kw) == ([0], [0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_zeros_of_both_signs_are_a_tie(dtype):
    V = 17000
    logits = torch.full((1, V), -1.0, device="cuda", dtype=dtype)
    logits[0, 9001], logits[0, 40] = 0.0, -0.0
    assert both(logits, [0], [-1], [0], 0.9, t=0.0) == ([0], [40])
    logits[0, 5] = 0.0
    assert both(logits, [0], [-1], [0], 0.9, t=0.0) == ([0], [5])
    # a cut at the zeros keeps all of them
    for kw in (dict(k=1), dict(k=2), dict(p=0.0), dict(m=1.0)):
        for u, token in ((0.3, 5), (0.5, 40), (0.9, 9001)):
            assert both(logits, [0], [-1], [0], u, t=0.2, **kw) == ([0], [token])
    # a flat row of zeros: more than are sorted
    logits[0, ::2] = -0.0
    logits[0, 1::2] = 0.0
    for kw in (dict(k=1), dict(k=6000), dict(p=0.5), dict(m=1.0)):
        assert both(logits, [0], [-1], [0], 0.25, **kw) == ([0], [V // 4])


def test_a_draft_that_is_the_target_up_to_rounding():
    """Every candidate refused, and what p - q leaves is rounding alone: whatever is emitted is a token that the filters keep."""
    n, V = 20000, 24
    g = torch.Generator().manual_seed(9)
    logits = torch.full((n, V), -INF)
    places = torch.stack([torch.randperm(V, generator=g)[:3] for _ in range(n)])
    values = torch.cat([torch.zeros(n, 1), -9.0 - 4.0 * torch.rand(n, 2, generator=g)], dim=1)
    logits.scatter_(1, places, values)
    q = torch.softmax(logits.double(), dim=-1).float()
    first = places[:, :1]
    q.scatter_(1, first, torch.nextafter(q.gather(1, first), torch.ones(n, 1)))        # refused by the largest random number below 1
    two = lambda t: t.repeat_interleave(2, dim=0).contiguous().cuda()  # noqa: E731
    ones = torch.ones(n, device="cuda")
    u = torch.full((2 * n,), 1 - 2 ** -24, device="cuda")
    path, out, counts = ops.tree_speculative_sample(
        two(logits), two(first[:, 0]), ints([-1, 0]).repeat(n), ints([2]).repeat(n), 2 * torch.arange(n, dtype=torch.int32, device="cuda"), ones,
        ints([0]).repeat(n), ones, None, u, torch.rand(n, generator=g).cuda(), 2, two(q))
    ops.check_status()
    emitted = out[:, 0].cpu()
    assert (emitted >= 0).all() and (emitted < V).all()
    assert torch.isfinite(logits.gather(1, emitted[:, None])).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lists_that_overflow_give_the_same_walk_every_time(dtype):
    """More tokens within reach of top-p's first guess than a list holds, mass in all of them; random numbers near borders."""
    B, V = 48, 60000
    g = torch.Generator().manual_seed(3)
    logits = (12 * torch.rand(B, V, generator=g)).cuda().to(dtype)
    logits[::3, :200] += 3
    f = lambda x: torch.tensor(x, device="cuda", dtype=torch.float32)  # noqa: E731
    args = (logits, torch.zeros(B, dtype=torch.int64, device="cuda"), ints([-1] * B), ints([1] * B), torch.arange(B, dtype=torch.int32, device="cuda"),
            f([1.0] * B), ints([(0, 9000)[i % 2] for i in range(B)]), f([0.3 + 0.69 * i / B for i in range(B)]), None, f([0.0] * B),
            torch.rand(B, generator=g).cuda(), 1)
    first = ops.tree_speculative_sample(*args)
    want = ref.tree_speculative_sample(*args)
    assert all(torch.equal(a, b) for a, b in zip(first, want))
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.tree_speculative_sample(*args)))
    ops.check_status()
