"""Many tokens of little weight behind one that has nearly all of a row's."""
import pytest
import torch

from mllm_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache", [(torch.float16, None), (torch.bfloat16, None), (torch.float16, torch.float8_e5m2), (torch.bfloat16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("below", [20.5, 25.5, 27.5])
@pytest.mark.parametrize("top", [0, 20000])
def test_weights_of_a_long_tail(dtype, cache, below, top):
    """Token ``top`` has the score below * ln 2, all others 0; values of the others are 1, of it 0: the result is the tail's share of the weight.

    A weight is off by half a step of 16 bits; in fp16 by half of 2^-24 at least, of weights whose largest is 2^7: 2^-32 for each of the n
    tokens.  The result is rounded once and its normaliser is what the product takes.  Of 64 tokens two are added to a lane's normaliser, one after
    the other: up to n / 32 = 1024 additions in a row, half a step each, which are 2^-14 of it; the products add 16 tokens at a time to a
    result, up to n / 64 = 512 additions cut off at a step: 2^-14."""
    n, D, batch = 32768, 128, 320                  # more requests than blocks that run at once: a warp has a quarter of a request's tokens
    store = cache or dtype
    q = torch.zeros((batch, 1, D), dtype=dtype, device="cuda")
    k = torch.zeros((1, n, D), dtype=store, device="cuda")
    v = torch.ones((1, n, D), dtype=store, device="cuda")
    q[:, :, 0], k[0, top, 0], v[0, top] = 1.0, 1.0, 0.0
    scale = below * 0.6931471805599453
    table = torch.arange(n, dtype=torch.int32, device="cuda").expand(batch, n)
    rows, lens = torch.arange(batch, dtype=torch.int32, device="cuda"), torch.full((batch,), n, dtype=torch.int32, device="cuda")
    sums = torch.zeros((batch, 1, n), device="cuda")
    out = ops.attention_decode_weights(q, k.transpose(0, 1), v.transpose(0, 1), table.contiguous(), rows, lens, scale, sums)
    ops.check_status()
    tail = (n - 1) * 2.0 ** -below
    want, half = tail / (1 + tail), torch.finfo(dtype).eps / 2
    weight = torch.finfo(torch.float16).eps / 2 if cache else half
    bound = (half + 2 * weight + 2.0 ** -13) * want + (n * 2.0 ** -32 if weight == 2.0 ** -11 else 0.0)
    off = (out.double() - want).abs().max().item()
    assert off <= bound, (off, bound, want)
    # the sums are of unrounded weights: a score's own roundings, twice, 64 steps for what joins the parts, and the normaliser's additions in a row
    each = 2.0 ** -below / (1 + tail)
    assert (sums[:, 0, 1:10].double() / each - 1).abs().max().item() <= (4 * below + 64 + n / 64) * 2.0 ** -23
