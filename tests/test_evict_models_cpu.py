"""Shortened requests of models with an 8-bit cache and with a soft cap."""
import pytest
import torch

from evict_cases import Shortened
from mllm_b200.layers.attention import RadixAttention


def capped(monkeypatch, cap):
    plain = RadixAttention.__init__

    def init(self, *args, **kw):
        plain(self, *args, **kw)
        self.logit_cap = cap

    monkeypatch.setattr(RadixAttention, "__init__", init)


def close(a, b):
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("cache", ["fp8_e4m3", "fp8_e5m2"])
def test_8_bit_cache(cache):
    Shortened("qwen3-tiny", "cpu", "float32", cache).check(close)


@pytest.mark.parametrize("preset", ["qwen3-tiny", "llama-tiny"])
def test_soft_cap(preset, monkeypatch):
    capped(monkeypatch, 0.25)
    s = Shortened(preset, "cpu", "float32")
    assert {m.logit_cap for m in s.mr.model.modules() if isinstance(m, RadixAttention)} == {0.25}
    s.check(close)
