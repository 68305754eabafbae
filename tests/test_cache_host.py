"""CPU tests of the cache and rotation operators: the C entry points' checks under sanitizers, the Python layer's refusals, the tests' own references."""

import pathlib
import subprocess

import numpy as np
import pytest
import torch

from kv_cache_reference import e4m3_values, nearest_e4m3, tables_reference

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_entry_points_under_address_and_ub_sanitizers(tmp_path):
    """fa_cache_capi.cpp built host-only with -fsanitize=address,undefined, the kernels replaced by launchers that check what they get"""
    exe = tmp_path / "test_cache_capi_host_asan"
    res = subprocess.run(["make", "-C", str(ROOT / "flash-attention-ipu_amd"), "sanitize-cache", f"SAN_CACHE_OUT={exe}"], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "PASSED" in res.stdout, res.stdout[-3000:] + res.stderr[-3000:]
    assert "runtime error" not in res.stderr and "AddressSanitizer" not in res.stderr


def test_c_entry_points_refuse_before_they_launch():
    from flash_attention_amd._impl import _native

    lib = _native.load_native_library()
    assert lib.fa_cache_attn_workspace(1, 1, 8, 3, 128, 64, 4, 1) == -2 and b"multiple of heads_kv" in lib.fa_last_error()
    assert lib.fa_cache_attn_workspace(1, 1, 8, 2, 128, 64, 400, 1) > 0 and lib.fa_cache_attn_workspace(1, 1, 8, 2, 128, 64, 4, 1) == 0
    assert lib.fa_cache_append(None, None, None, None, None, None, None, 1, 1, 64, 64, 1, 16, None, None, 1, None) == -1
    assert lib.fa_error_string(-16) == b"workspace too small"


def test_cpu_tensors_are_refused():
    import flash_attention_amd.kv_cache as kv
    import flash_attention_amd.rotary as rot

    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    k, v = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 2, 64, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s, t = torch.ones(4, 2), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        rot.qk_norm_rope(x, x, None, None, rot.rotary_table(4, 64))
    with pytest.raises(ValueError):
        kv.cache_append(x, x, i, k, v, s, s)
    with pytest.raises(ValueError):
        kv.cache_tables(i, i, t, i, i[:1], 2, 16)
    with pytest.raises(ValueError):
        kv.flash_attention_cached(x, k, v, s, s, t, i, torch.zeros(3, dtype=torch.int32))


def test_rotary_table():
    import flash_attention_amd.rotary as rot

    t = rot.rotary_table(100000, 128, theta=5e5)
    pos = np.array([0, 1, 7, 99999])
    angle = pos[:, None].astype(np.longdouble) * np.longdouble(5e5) ** (-2 * np.arange(64, dtype=np.longdouble) / 128)
    want = np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float64)
    # formed in 64 bits: an angle of 10^5 is off by some 2^-36, a value by that and half a step of 32 bits
    assert np.abs(t[pos].double().numpy() - want).max() <= 2.0 ** -25 + 2.0 ** -33


def test_reference_codes():
    v = e4m3_values()
    torch_values = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(v, torch_values)
    x = torch.linspace(-448, 448, 4097, dtype=torch.float64).mul(torch.exp2(torch.arange(4097).remainder(17).double() * -1)).float()
    np.testing.assert_array_equal(nearest_e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())


def test_reference_tables():
    r = tables_reference([3, 16, 0], [1, -1, 17], [[5, -1], [6, -1], [-1, -1]], [1, 2, 3, 0], 3, 18, 16)
    assert r["seq_lens"] == [4, 0, 17] and r["pool"] == [1, 2, 3, 6] and r["free"] == 2 and r["tables"][2] == [6, 3]
    assert r["slots"][0] == 5 * 16 + 3 and r["slots"][1] == 96 and r["slots"][17] == 48 and r["positions"][:2] == [3, 0]
