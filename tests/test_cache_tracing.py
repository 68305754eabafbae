"""CPU tests: the cache and rotation operators under forward-mode levels (no kernel runs)."""

import pytest
import torch
from torch.autograd import forward_ad

import flash_attention_amd.kv_cache as kv
import flash_attention_amd.rotary as rot


def test_tangents_are_refused():
    table = torch.zeros(8, 64)
    x = torch.zeros(4, 2, 64)
    ones, ints = torch.ones(4, 2), torch.zeros(4, dtype=torch.int32)
    codes = [torch.zeros(4, 2, *s, dtype=torch.uint8).view(torch.float8_e4m3fn) for s in ((16, 64), (64, 16))]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        weight = forward_ad.make_dual(torch.ones(64), torch.ones(64))
        scale = forward_ad.make_dual(ones, torch.ones(4, 2))
        for args in ((dual, x, None, None, table), (x, dual, None, None, table), (x, x, weight, None, table), (x, x, None, weight, table),
                     (x, x, None, None, forward_ad.make_dual(table, torch.ones_like(table)))):
            with pytest.raises(ValueError, match="forward-mode"):
                rot.qk_norm_rope(*args)
        for args in ((dual, x, ints, *codes, ones, ones), (x, dual, ints, *codes, ones, ones), (x, x, ints, *codes, scale, ones)):
            with pytest.raises(ValueError, match="forward-mode"):
                kv.cache_append(*args)
        for args in ((dual, *codes, ones, ones), (x, *codes, ones, scale)):
            with pytest.raises(ValueError, match="forward-mode"):
                kv.flash_attention_cached(*args, torch.zeros(1, 1, dtype=torch.int32), ints[:1], ints[:2])
        with pytest.raises((ValueError, TypeError), match="GPU"):          # (no tangent: the other checks)
            rot.qk_norm_rope(x, x, None, None, table)
