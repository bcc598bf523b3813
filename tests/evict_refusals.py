"""Calls that no device takes, beside those of test_evict_cpu.refusals."""
import torch

from evict_cases import cached_batch
from mllm_b200 import ops


def overlapping(device):
    """(call, what the message says): what is written lies on itself."""
    c = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, device=device)
    p = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, new=[5, 6], device=device)
    s = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, layers=3, device=device)
    rows, heads, tokens = c["sums"].shape
    keep, counts = torch.zeros((3, 2, 2, 8), dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device)
    flat = torch.zeros(4 * rows * heads * tokens, device=device)

    def decode(sums=None, out=None):
        return lambda: ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], 0.1, c["sums"] if sums is None else sums, out=out)

    def prompt(sums):
        return lambda: ops.attention_prefill_weights(p["q"], p["k"], p["table"], p["req"], p["seq"], p["prefix"], p["start"], 0.1, sums)

    def evict(sums):
        return lambda: ops.cache_evict(s["store"], sums, s["table"], s["req"], keep, counts)

    calls = []
    for bad in (c["sums"][:1].expand(rows, -1, -1), c["sums"][:, :1].expand(-1, heads, -1), flat.as_strided((rows, heads, tokens), (heads * tokens, tokens - 1, 1)),
                flat.as_strided((rows, heads, tokens), (tokens, tokens, 1))):
        calls += [(decode(sums=bad), "must not overlap"), (prompt(bad), "must not overlap"), (evict(bad[None].expand(3, -1, -1, -1)), "must not overlap")]
    calls += [(evict(s["sums"][:1].expand(3, -1, -1, -1)), "must not overlap"), (decode(out=c["q"][:1].expand(2, -1, -1)), "out must be")]
    return calls


def too_large(device):
    """Scales and caps that are finite, but not in units of log2."""
    c = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, device=device)
    p = cached_batch([40, 17], 4, 2, 64, dtype=torch.bfloat16, seed=1, new=[5, 6], device=device)

    def decode(scale=0.1, cap=0.0):
        return lambda: ops.attention_decode_weights(c["q"], c["k"], c["v"], c["table"], c["req"], c["seq"], scale, c["sums"], logit_cap=cap)

    def prompt(scale=0.1, cap=0.0):
        return lambda: ops.attention_prefill_weights(p["q"], p["k"], p["table"], p["req"], p["seq"], p["prefix"], p["start"], scale, p["sums"], logit_cap=cap)

    return [(f(**kw), name) for f in (decode, prompt) for kw, name in ((dict(scale=3e38), "scale"), (dict(cap=3e38), "logit_cap"))]
