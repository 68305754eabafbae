"""GPU tests of flash_attention_cached at the borders inside a call: units, parts, waves and requests that one workgroup takes one after the other."""

import numpy as np
import pytest
import torch

from kv_cache_reference import attention_reference
from test_gpu_kv_cache import DEV, check_attention, code_values, ints, tolerance

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


@BOTH
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hint", [1, 1000])
@pytest.mark.parametrize("why", ["pool", "table", "tokens", "long"])
def test_refused_requests_between_served_ones(kv, dtype, D, hint, why):
    """rows whose tokens found no place: zeros; the others' attention, the cache and a later step are as if they had not been there"""
    Hkv, H, P, g = 2, 4, 16, torch.Generator().manual_seed(41)
    blocks, most, held, new, served, room = {
        "pool": (10, 128, [40, 30, 20, 0], [1, 60, 5, 2], [1, 0, 5, 0], 70),
        "table": (60, 64, [40, 30, 20, 0], [1, 60, 5, 2], [1, 0, 5, 2], 68),
        "tokens": (60, 128, [40, 30, 20, 0], [1, 60, 5, 20], [1, 60, 5, 0], 76),
        "long": (700, 5040, [4900, 5000, 100], [2, 90, 1], [2, 0, 1], 95)}[why]
    cache = kv.KVCache(1, blocks, Hkv, D, requests=len(held), max_tokens=most, block_size=P)
    draw = lambda n: [torch.randn(n, h, D, generator=g).to(dtype) for h in (H, Hkv, Hkv)]  # noqa: E731
    q, k, v = draw(sum(held))
    cache.append(0, k.to(DEV), v.to(DEV), cache.step(ints(held), sum(held)))
    q, k, v = draw(room)
    step = cache.step(ints(new), room)
    out = torch.full((room, H, D), 7.0, dtype=dtype, device=DEV)
    cache.attend(0, q.to(DEV), k.to(DEV), v.to(DEV), step, max_q_len=hint, out=out)
    assert step.granted.tolist() == served and cache.seq_lens.tolist() == [h + s for h, s in zip(held, served)]
    cu = np.minimum(np.concatenate([[0], np.cumsum(new)]), room).tolist()
    lens = [h + s if s else 0 for h, s in zip(held, served)]
    k_cache, v_cache, ks, vs = cache._layer[0]
    ref, mag = attention_reference(q.double(), code_values(k_cache), code_values(v_cache).transpose(2, 3), ks.cpu().double(), vs.cpu().double(), cache.block_tables.tolist(), lens, cu,
                                   D ** -0.5)
    assert bool((out[cu[-1]:] == 7.0).all())
    out, ref, mag = out[: cu[-1]].cpu().double(), ref[: cu[-1]], mag[: cu[-1]]
    assert bool(((out - ref).abs() <= tolerance(dtype, ref, mag, 448 * float(vs.max()), max(lens))).all())
    for b, s in enumerate(served):
        rows = out[cu[b]:cu[b + 1]]
        assert bool((rows == 0).all()) if s == 0 else float(rows.abs().min()) >= 0 and float(rows.abs().max()) > 0
    with pytest.raises((ValueError, TypeError)):
        kv.flash_attention_cached(q.to(DEV), k_cache, v_cache, ks, vs, cache.block_tables, step.seq_lens, step.cu_new, granted=step.granted.long())
    with pytest.raises((ValueError, TypeError)):
        kv.flash_attention_cached(q.to(DEV), k_cache, v_cache, ks, vs, cache.block_tables, step.seq_lens, step.cu_new, granted=step.granted[1:])


@BOTH
@pytest.mark.parametrize("D", [64, 128, 256])
def test_one_prompt_beside_idle_rows(kv, dtype, D):
    """the default hint says one token each, and one request has them all"""
    new = [0] * 40 + [37] + [0] * 9
    check_attention(kv, [5] * 40 + [300] + [70] * 9, new, 2, 2, D, 16, dtype, seed=51)
    check_attention(kv, [5] * 40 + [3000] + [70] * 9, new, 2, 2, D, 64, dtype, seed=52)


def test_outputs_whose_rows_share_memory_are_refused(kv):
    c = kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=16)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV)
    args = (*c._layer[0], c.block_tables, ints([1, 1]), ints([0, 1, 2]))
    room = torch.zeros(1024, dtype=torch.float16, device=DEV)
    for strides in ((0, 64, 1), (256, 0, 1), (128, 64, 1)):
        with pytest.raises(ValueError, match="share memory"):
            kv.flash_attention_cached(q, *args, out=room.as_strided((2, 4, 64), strides))
    kv.flash_attention_cached(q, *args, out=room.as_strided((2, 4, 64), (64, 128, 1)))


@BOTH
@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("new", [1, 70])
def test_blocks_of_a_larger_allocation(kv, dtype, P, new):
    """a layer's blocks and scales as slices of tensors that hold more: strides between blocks of their own, codes and scales around them NaN"""
    g = torch.Generator().manual_seed(61)
    N, H, D = 24, 2, 128
    plain = [torch.randint(0, 120, s, generator=g, dtype=torch.uint8).to(DEV) for s in ((N, H, P, D), (N, H, D, P))]
    scales = [torch.exp2(torch.randint(-8, -4, (N, H), generator=g).float()).to(DEV) for _ in "kv"]
    wide = [torch.full((N, 3, *t.shape[1:]), 0x7F, dtype=torch.uint8, device=DEV) for t in plain]
    wide_scales = [torch.full((N, 3, H), float("nan"), device=DEV) for _ in "kv"]
    for w, t in zip(wide + wide_scales, plain + scales):
        w[:, 1] = t
    tables, lens, cu = ints(np.random.default_rng(0).permutation(N).reshape(2, 12)), ints([12 * P - 3, 7 * P + 1]), ints([0, new, 2 * new])
    q = torch.randn(2 * new, 4, D, generator=g).to(dtype).to(DEV)
    fp8 = lambda ts: [t.view(torch.float8_e4m3fn) for t in ts]  # noqa: E731
    want = kv.flash_attention_cached(q, *fp8(plain), *scales, tables, lens, cu, max_q_len=new)
    got = kv.flash_attention_cached(q, *[t[:, 1] for t in fp8(wide)], *[t[:, 1] for t in wide_scales], tables, lens, cu, max_q_len=new)
    assert torch.equal(got, want) and bool(torch.isfinite(want).all())
