"""Verification of drafted token trees on the GPU against the walk in 64 bits, request by request.  Node and token numbers are compared as they
are: the kernel's sums are off by some 10^-9 of the whole, so a draw within that of a token's border would differ, and none of these is."""
import pytest
import torch

from mllm_b200 import ops
from mllm_b200.ops import reference as ref
from tree_cases import make_trees

pytestmark = pytest.mark.gpu


def batch(nodes, V, seed, dtype=torch.bfloat16, draft=False, floor=1.5, peak=11.0, width=3, spare=0, params=None):
    """Logits with some tokens far above the others; children's tokens are likely ones, or drawn from the draft's distribution."""
    g = torch.Generator().manual_seed(seed)
    trees = make_trees(nodes, seed, width)
    T, B = sum(nodes) + spare, len(nodes)
    logits = torch.randn(T, V, generator=g) * floor
    best = torch.randint(0, V, (T, min(V, 12)), generator=g)
    logits.scatter_(1, best, peak + 2.0 * torch.randn(best.shape, generator=g))
    noisy = logits + 0.5 * torch.randn(T, V, generator=g)
    probs = torch.softmax(noisy, dim=-1)
    starts = [sum(nodes[:i]) for i in range(B)]
    tokens = torch.zeros(T, dtype=torch.int64)
    for s, parents in zip(starts, trees):
        for j, up in enumerate(parents):
            row = s + max(up, 0)
            if draft:
                tokens[s + j] = torch.multinomial(probs[row], 1, generator=g)[0]
            else:
                rank = sum(1 for x in parents[:j] if x == up)
                tokens[s + j] = noisy[row].topk(min(V, rank + 1)).indices[-1]
    if params is None:
        params = [dict(t=(0.7, 1.0, 0.0, 1.3)[i % 4], k=(0, 20, 0, 50, 1)[i % 5], p=(1.0, 0.9, 0.5)[i % 3], m=(0.0, 0.0, 0.1)[(i // 2) % 3]) for i in range(B)]
    col = lambda k, dt: torch.tensor([x[k] for x in params], dtype=dt)  # noqa: E731
    parents = torch.tensor([p for t in trees for p in t] + [-1] * spare, dtype=torch.int32)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    args = [logits.to(dtype), tokens, parents, ints(nodes), ints(starts), col("t", torch.float32), col("k", torch.int32), col("p", torch.float32),
            col("m", torch.float32), torch.rand(T, generator=g), torch.rand(B, generator=g)]
    return [a.cuda() for a in args], probs.cuda() if draft else None


def compare(args, steps, draft=None):
    n0 = ops.launch_count()
    got = ops.tree_speculative_sample(*args, steps, draft_probs=draft)
    ops.check_status()
    assert ops.launch_count() > n0
    want = ref.tree_speculative_sample(*args, steps, draft)
    for a, b, name in zip(got, want, ("path", "tokens", "counts")):
        assert a.dtype == b.dtype and torch.equal(a, b), (name, a, b)
    return got


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 7, 33, 1000, 16385, 50257, 151936])
def test_walks(V, dtype, draft):
    args, probs = batch([1, 9, 16, 5, 12, 7, 20], V, seed=V + draft, dtype=dtype, draft=draft, spare=2)
    got = compare(args, 6, probs)
    assert got[2].max() > 1 or V < 50


@pytest.mark.parametrize("seed", range(6))
def test_draws_over_many_requests(seed):
    args, probs = batch([8] * 40, 2000, seed=seed, draft=bool(seed % 2), width=2)
    compare(args, 5, probs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [40000, 70001])
def test_more_requests_than_sms_for_them(V, dtype):
    """Requests of 8 CTAs each, more than SMs: two CTAs on an SM, and further ones behind them; flat rows among them."""
    params = [dict(t=1.0, k=(0, 40, 0)[i % 3], p=(0.95, 1.0, 0.8)[i % 3], m=0.0) for i in range(60)]
    args, _ = batch([3] * 60, V, seed=11, dtype=dtype, params=params)
    args[0][:9] *= 0.05
    compare(args, 3)


@pytest.mark.parametrize("steps", [1, 2, 9])
def test_steps(steps):
    args, _ = batch([10, 10, 10], 500, seed=3, width=1, params=[dict(t=0.0, k=0, p=1.0, m=0.0)] * 3)
    # the tokens that greedy decoding takes: the whole chain is accepted
    for b in range(3):
        for j in range(1, 10):
            row = b * 10 + j
            args[1][row] = args[0][b * 10 + int(args[2][row])].float().argmax()
    got = compare(args, steps)
    assert got[2].min() >= min(steps, 2)


@pytest.mark.parametrize("p", [0.3, 0.95, 0.9999])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_flat_rows(p, dtype):
    """Cuts with far more tokens above them than are sorted, and rows of one value."""
    params = [dict(t=1.0, k=k, p=p, m=0.0) for k in (0, 9000, 30000, 0)]
    args, _ = batch([3] * 4, 40000, seed=5, dtype=dtype, floor=0.3, peak=0.5, params=params)
    args[0][9:] = 0.25
    compare(args, 3)


def test_values_that_are_no_numbers():
    args, _ = batch([4] * 5, 3000, seed=8, params=[dict(t=1.0, k=5, p=0.9, m=0.0), dict(t=1.0, k=0, p=1.0, m=0.0), dict(t=0.0, k=0, p=1.0, m=0.0),
                                                   dict(t=1.0, k=0, p=0.9, m=0.1), dict(t=0.5, k=0, p=1.0, m=0.0)])
    nan, inf = float("nan"), float("inf")
    args[0][0, 5:40] = nan
    args[0][4, ::7] = -inf
    args[0][8:12, 100] = nan
    args[0][12:16] = -inf           # no finite logit: the first token
    args[0][16:20, 77] = inf        # all the mass
    got = compare(args, 4)
    assert int(got[1][3, 0]) == 0 and int(got[1][4, int(got[2][4]) - 1]) == 77


def test_same_tokens_twice_and_tokens_outside():
    args, probs = batch([6, 6], 300, seed=2, draft=True, params=[dict(t=1.0, k=0, p=1.0, m=0.0)] * 2)
    args[2][:] = torch.tensor([-1, 0, 0, 0, 0, 1, -1, 0, 0, 0, 0, 1], dtype=torch.int32)
    args[1][2] = args[1][1]
    args[1][8] = 300
    args[1][9] = -1
    args[9][:] = 0.999
    compare(args, 4, probs)
    compare(args, 4)


def test_distribution_of_the_first_token():
    """Whatever the draft, the first emitted token is distributed as the target's: 40000 walks over 6 tokens, three drawn candidates.
    Frequencies of n draws are off by at most 5 sqrt(p (1 - p) / n) once in some 10^6."""
    n, V = 40000, 6
    g = torch.Generator().manual_seed(1)
    target = torch.tensor([0.4, 0.25, 0.15, 0.1, 0.07, 0.03])
    q = torch.tensor([0.05, 0.5, 0.05, 0.2, 0.1, 0.1])
    logits = torch.log(target).expand(4 * n, V).contiguous().cuda()
    probs = q.expand(4 * n, V).contiguous().cuda()
    tokens = torch.multinomial(q, 4 * n, replacement=True, generator=g).cuda()
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32).repeat(n).cuda()
    ones = torch.ones(n, device="cuda")
    args = [logits, tokens, parents, torch.full((n,), 4, dtype=torch.int32, device="cuda"), 4 * torch.arange(n, dtype=torch.int32, device="cuda"),
            ones, torch.zeros(n, dtype=torch.int32, device="cuda"), ones, None, torch.rand(4 * n, generator=g).cuda(), torch.rand(n, generator=g).cuda()]
    # how often a candidate is taken: drawn ones, the first alone with probability sum min(p, q) = 0.55; picked ones, whenever the target's
    # own token is among them, sum p (1 - (1 - q)^3) = 0.3732
    picked = (target * (1 - (1 - q) ** 3)).sum().item()
    drawn = torch.minimum(target, q).sum().item()
    for draft in (probs, None):
        _, out, counts = ops.tree_speculative_sample(*args, 2, draft_probs=draft)
        ops.check_status()
        freq = torch.bincount(out[:, 0].cpu(), minlength=V).double() / n
        assert ((freq - target).abs() <= 5 * (target * (1 - target) / n).sqrt()).all(), freq
        taken, slack = counts.double().mean().item() - 1, 5 * 0.5 / n ** 0.5
        assert taken >= drawn - slack if draft is not None else abs(taken - picked) <= slack, taken


def test_requests_without_nodes_and_outside():
    args, _ = batch([3, 3, 3], 100, seed=4)
    args[3][1] = 0
    got = compare(args, 3)
    assert got[2][1] == 0 and (got[0][1] == -1).all()
    args[4][2] = 8
    path, out, counts = ops.tree_speculative_sample(*args, 3)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert counts[2] == 0 and (out[2] == -1).all()
