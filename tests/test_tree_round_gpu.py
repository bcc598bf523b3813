"""Whole rounds of speculative decoding of tiny models on the GPU: prologue, attention, verification and accepted rows, as they are used
together, against the same tokens run as plain prompts; and a round captured in a CUDA graph."""
import pytest
import torch

from mllm_b200 import ops
from tree_cases import Round, tree_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen3-moe-tiny"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_rounds_of_a_model(preset, dtype):
    r = Round(preset, "cuda:0", dtype)
    # Both sides round some 12 tensors per layer and direction to the activation type, half a step each, in two layers; errors of the
    # 2-norm add up at most linearly.
    bound = 2 * 2 * 12 * torch.finfo(getattr(torch, dtype)).eps / 2
    before = ops.launch_count()
    r.check(lambda a, b: (lambda x, y: pytest.fail(f"{x} over {y}") if not x <= y else None)(
        ((a.double() - b.double()).norm() / b.double().norm()).item(), bound))
    assert ops.launch_count() > before


def test_rounds_over_an_8bit_cache():
    r = Round("qwen3-tiny", "cuda:0", "bfloat16", kv_cache_dtype="fp8_e4m3")
    # keys and values rounded once more, to 4 bits: 2^-4 of each; both sides, two layers
    bound = 2 * 2 * (12 * 2 ** -8 + 2 * 2 ** -4)
    r.check(lambda a, b: (lambda x, y: pytest.fail(f"{x} over {y}") if not x <= y else None)(
        ((a.double() - b.double()).norm() / b.double().norm()).item(), bound))


def test_a_round_in_a_graph():
    """All four operators captured together and replayed with other random numbers, lengths and slots."""
    hq, hkv, D, V, steps = 8, 2, 128, 4000, 4
    trees = [[-1, 0, 0, 1, 2], [-1, 0, 1, 0]]
    c = tree_batch([300, 40], [5, 4], hq, hkv, D, trees=trees)
    g = torch.Generator().manual_seed(0)
    store = torch.randn(2, 2, hkv, c["slots"], D, generator=g).cuda().to(torch.bfloat16)
    qkv = torch.randn(9, (hq + 2 * hkv) * D, generator=g).cuda().to(torch.bfloat16)
    head = torch.randn(hq * D, V, generator=g).cuda().to(torch.bfloat16)
    inv = (1e4 ** -(torch.arange(D // 2).double() / (D // 2))).float().cuda()
    tokens = torch.randint(0, V, (9,), generator=g).cuda()
    f = lambda x: torch.tensor(x, device="cuda")  # noqa: E731
    u, uf = torch.rand(9, generator=g).cuda(), torch.rand(2, generator=g).cuda()
    lens = c["seq"] - c["prefix"]
    knobs = (f([0.8, 1.0]), f([50, 0]).int(), f([0.95, 1.0]), f([0.0, 0.05]))

    def step():
        s = store.clone()
        k, v = s[1, 0].transpose(0, 1), s[1, 1].transpose(0, 1)
        ix = (c["table"], c["req"], c["seq"], c["prefix"], c["start"])
        q = ops.tree_qk_norm_rope_kv_write(qkv, None, None, c["parents"], *ix, inv, k, v, hq, hkv, D, 1e-6)
        o = ops.attention_tree(q, k, v, *ix, c["parents"], D ** -0.5)
        logits = torch.nn.functional.linear(o.view(9, -1), head.t()) * 0.2
        path, out, counts = ops.tree_speculative_sample(logits, tokens, c["parents"], lens, c["start"], *knobs, u, uf, steps)
        ops.tree_kv_compact(s, c["table"], c["req"], c["prefix"], path, counts)
        return s, q, o, path, out, counts

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for seed in range(3):
        n = torch.Generator().manual_seed(seed + 7)
        u.copy_(torch.rand(9, generator=n))
        uf.copy_(torch.rand(2, generator=n))
        qkv.copy_(torch.randn(qkv.shape, generator=n))
        if seed == 2:
            c["prefix"].sub_(7)
            c["seq"].sub_(7)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        ops.check_status()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
