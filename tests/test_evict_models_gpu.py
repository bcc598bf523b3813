"""Shortened requests of models with an 8-bit cache and with a soft cap, on the GPU."""
import pytest
import torch

from evict_cases import Shortened
from test_evict_models_cpu import capped
from mllm_b200 import ops
from mllm_b200.layers.attention import RadixAttention

pytestmark = pytest.mark.gpu


def run(preset, dtype, cache="auto"):
    # as in test_evict_gpu: both sides round some 12 tensors per layer to the activation type, half a step each, in two layers
    bound = 2 * 2 * 12 * torch.finfo(getattr(torch, dtype)).eps / 2

    def close(a, b):
        off = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert off <= bound, (off, bound)

    s = Shortened(preset, "cuda:0", dtype, cache)
    s.check(close)
    return s


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("cache", ["fp8_e4m3", "fp8_e5m2"])
def test_8_bit_cache(dtype, cache):
    before = ops.launch_count()
    run("qwen3-tiny", dtype, cache)
    assert ops.launch_count() > before


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny"])
def test_soft_cap(preset, monkeypatch):
    capped(monkeypatch, 0.25)
    s = run(preset, "bfloat16")
    assert {m.logit_cap for m in s.mr.model.modules() if isinstance(m, RadixAttention)} == {0.25}
