"""Soft caps far above the scores: the cap is the identity there, and a score keeps its places whatever the cap is."""
import pytest
import torch

import evict_cases
from evict_cases import cached_batch
from test_evict_gpu import decode, prompt, within
from mllm_b200 import ops

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn
STEP = 2.0 ** -23


def capped_sums(c, cap, queries, add):
    """(sums, their bound) in 64 bits; ``queries``: (first row of q, rows, their first cache index) per request.

    The bound is evict_cases.exact_prompt's, with the cap's part in terms of the score instead of the cap: three factors that are rounded on
    the host and four products, half a step each, and tanhf, two units in the last place: 5.5 steps of a score, which tanh's slope, at most
    1, does not enlarge; 8 are taken.  A score is in the weight and in the normaliser."""
    sums, bound = c["sums"].double(), torch.zeros_like(c["sums"], dtype=torch.float64)
    for b, (first, rows, place) in enumerate(queries):
        n, row = c["lens"][b], int(c["req"][b])
        q, at = c["q"][first:first + rows], torch.arange(place, place + rows, device=c["q"].device)
        w, _ = evict_cases._weights(c, b, q, at, cap, None)
        _, off = evict_cases._weights(c, b, q, at, 0.0, None)
        keys = c["k"][c["table"][row, :n].long()].double()
        s = torch.einsum("wkgd,lkd->wkgl", q.double().view(rows, c["hkv"], -1, q.shape[-1]), keys) * c["scale"]
        off = off + 2 * 8 * STEP * s.abs().amax(-1, keepdim=True)
        total, slack = w.sum((0, 2)), (w * off).sum((0, 2))
        old = sums[row, :, :n].clone()
        old[:, add[b]:] = 0
        sums[row, :, :n] = old + total
        bound[row, :, :n] = 1.01 * slack + STEP / 2 * (w.shape[0] * w.shape[2] + 8) * (old + total) + 1e-37
    return sums, bound


@pytest.mark.parametrize("cap", [2.0, 50.0, 1e3, 1e6, 1e20, 1e38])
@pytest.mark.parametrize("room", [256, 300])
@pytest.mark.parametrize("D,dtype,cache", [(128, torch.bfloat16, None), (64, torch.float16, None), (128, torch.bfloat16, E4), (256, torch.bfloat16, None)])
@pytest.mark.parametrize("last", [8, 0])
def test_prompt(cap, room, D, dtype, cache, last):
    c = cached_batch([200, 64, 1, 90], 8, 2, D, dtype=dtype, cache=cache, seed=7, new=[100, 64, 1, 30], room=room)
    queries = []
    for n, new, start in zip(c["lens"], c["new"], c["start"].tolist()):
        look = min(last, new) if last else new
        queries.append((start + new - look, look, n - look))
    want, bound = capped_sums(c, cap, queries, [0] * 4)
    prompt(c, last=last, cap=cap)
    ops.check_status()
    within(c["sums"], want, bound, "sums")


@pytest.mark.parametrize("cap", [2.0, 50.0, 1e3, 1e6, 1e20, 1e38])
@pytest.mark.parametrize("D,dtype,cache", [(128, torch.bfloat16, None), (64, torch.float16, None), (128, torch.bfloat16, E4)])
def test_decode(cap, D, dtype, cache):
    c = cached_batch([700, 64, 1, 90], 8, 2, D, dtype=dtype, cache=cache, seed=8)
    want, bound = capped_sums(c, cap, [(b, 1, n - 1) for b, n in enumerate(c["lens"])], [n - 1 for n in c["lens"]])
    decode(c, cap=cap)
    ops.check_status()
    within(c["sums"], want, bound, "sums")
