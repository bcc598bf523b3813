"""Rounds of tiny models on the CPU: the accepted way, and that a wrong tree shows."""
import pytest

from tree_ways import accepted_way, errors


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen2-tiny", "qwen3-moe-tiny"])
def test_the_accepted_way_is_the_planned_one(preset):
    accepted_way(preset, "cpu", "float32")


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny", "qwen2-tiny", "qwen3-moe-tiny"])
def test_a_wrong_parent_shows(preset):
    right, wrong = errors(preset, "cpu", "float32")
    # fp32 products of 256 to 512 terms through two layers; the bound that the same models are held to in fp16
    assert max(right) <= 2 * 2 * 512 * 2 ** -24 * 8 and min(wrong) > 2 * 2 * 12 * 2 ** -11
