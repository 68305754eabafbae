"""CPU test of the softmax scales that the attention over the cache takes: the check stands in front of every launch."""

import ctypes

import pytest

BAD_SCALE = -11


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan"), 3.0e38])
def test_scales_that_are_refused(scale):
    """3e38 is finite, but not times log2 e: every score would become an infinity or NaN"""
    from flash_attention_amd._impl import _native

    lib = _native.load_native_library()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    tokens, blocks = (ctypes.c_int64 * 4)(64, 64, 64, 64), (ctypes.c_int64 * 4)(1024, 1024, 1, 1)
    rc = lib.fa_cache_attn(at, at, at, at, at, at, at, at, at, None, 0, 1, 1, 1, 1, 64, 64, 1, 16, 1, 1, 1, tokens, blocks, 0, scale, None)
    assert rc == BAD_SCALE and b"softmax_scale" in lib.fa_last_error()
