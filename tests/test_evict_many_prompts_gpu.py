"""Attention weights of many short prompts: a CTA has several requests' blocks of rows in a row, some of one step each."""
import pytest
import torch

from evict_cases import cached_batch
from test_evict_gpu import check_prompt

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn


@pytest.mark.parametrize("D,dtype,cache", [(64, torch.bfloat16, None), (64, torch.float16, None), (64, torch.bfloat16, E4), (128, torch.bfloat16, None),
                                           (256, torch.float16, None)])
@pytest.mark.parametrize("lens", [[100] * 64, [100, 200] * 40, [300, 90, 128, 129, 1] * 20, [40] * 150, [1000] + [100] * 40])
@pytest.mark.parametrize("last", [0, 64])
def test_blocks_of_few_steps(D, dtype, cache, lens, last):
    check_prompt(cached_batch(lens, 32, 8, D, dtype=dtype, cache=cache, seed=len(lens) + D, new=lens, room=1100), last=last)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (12, 3), (32, 1)])
@pytest.mark.parametrize("last", [0, 64])
def test_blocks_of_few_steps_of_other_groups(hq, hkv, last):
    lens = [129, 260, 130] * 30
    check_prompt(cached_batch(lens, hq, hkv, 64, seed=hq, new=lens, page=16), last=last)
