"""GPU tests of flash_attention_cached at the borders inside a call: units, parts, waves and requests that one workgroup takes one after the other."""

import numpy as np
import pytest
import torch

from test_gpu_kv_cache import check_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    import flash_attention_amd.kv_cache as kv

    return kv


BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


@BOTH
@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("max_q_len", [2, 100])
def test_nan_marks_of_one_request_after_the_other(kv, dtype, P, D, max_q_len):
    """every request has a NaN of its own that its last row alone sees: other columns, heads and requests of the same workgroup stay clean"""
    rng = np.random.default_rng(P + D)
    held = rng.integers(0, 200, 400).tolist()

    def poke(k, v, tables, lens):
        codes = v.view(torch.uint8)
        for b, n in enumerate(lens):
            if b % 3 != 2:
                codes[int(tables[b, (n - 1) // P]), b % 2, (37 * b) % D, (n - 1) % P] = 0x7F

    out = check_attention(kv, held, [2] * 400, 2, 2, D, P, dtype, seed=31, max_q_len=max_q_len, poke=poke)
    assert not bool(torch.isnan(out[0::2]).any()) and int(torch.isnan(out[1::2]).sum()) == 2 * sum(b % 3 != 2 for b in range(400))
