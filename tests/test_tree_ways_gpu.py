"""Rounds of tiny models on the GPU: the accepted way, and that a wrong tree shows."""
import pytest

from tree_ways import accepted_way, errors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen2-tiny", "qwen3-moe-tiny"])
@pytest.mark.parametrize("kw", [dict(), dict(kv_cache_dtype="fp8_e4m3")])
def test_the_accepted_way_is_the_planned_one(preset, kw):
    accepted_way(preset, "cuda:0", "float16", **kw)


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen2-tiny", "qwen3-moe-tiny"])
def test_a_wrong_parent_shows(preset):
    right, wrong = errors(preset, "cuda:0", "float16")
    # both sides round some 12 tensors per layer to fp16, half a step each, in two layers; errors of the 2-norm add up at most linearly
    bound = 2 * 2 * 12 * 2 ** -11
    assert max(right) <= bound < min(wrong)
