"""CPU tests of what flash_attention_cached takes as its output."""

import pytest
import torch

from flash_attention_amd._impl import kv_cache


@pytest.mark.parametrize("overlap,shape,strides", [
    (False, (5, 4, 64), (256, 64, 1)), (False, (5, 4, 64), (64, 320, 1)), (False, (5, 4, 64), (1024, 128, 1)), (False, (1, 4, 64), (0, 64, 1)), (False, (5, 1, 64), (64, 0, 1)),
    (False, (0, 4, 64), (0, 64, 1)), (False, (5, 4, 64), (256 + 8, 64, 1)),
    (True, (5, 4, 64), (0, 64, 1)), (True, (5, 4, 64), (256, 0, 1)), (True, (5, 4, 64), (128, 64, 1)), (True, (5, 4, 64), (256, 32, 1)), (True, (5, 4, 64), (64, 64, 1)),
    (True, (5, 4, 64), (248, 64, 1))])
def test_rows_that_share_memory(overlap, shape, strides):
    t = torch.empty(8192).as_strided(shape, strides)
    assert kv_cache._rows_overlap(t) is overlap
