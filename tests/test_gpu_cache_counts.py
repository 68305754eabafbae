"""GPU tests that every key is counted once: queries of zeros give all keys of a row the same weight, and every column of the values has one key alone, so that a key
(or a unit, part or block) that is skipped, taken twice or seen by the wrong row changes its column by all that it holds."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def kv():
    import flash_attention_amd.kv_cache as kv

    return kv


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def check_counts(kv, lens, new, Hkv, group, D, P, dtype, told=None, seed=0):
    rng = np.random.default_rng(seed)
    W, B, H = kv.cache_width(D), len(lens), Hkv * group
    need = [-(-n // P) for n in lens]
    N = sum(need) + 2
    ids, width = rng.permutation(N), max(need + [1]) + 1
    tables = np.full((B, width), -1)
    for b, n in enumerate(need):
        tables[b, :n] = ids[sum(need[:b]):sum(need[:b]) + n]
    cu = np.concatenate([[0], np.cumsum(new)])
    # the first and the last key of every unit of 64, the keys round the rows' limits, and some others
    wanted = []
    for n, m in zip(lens, new):
        keys = [k for u in range(0, n, 64) for k in (u, u + 63)] + [k for i in range(m) for k in (n - m + i - 1, n - m + i, n - m + i + 1)] + rng.integers(0, max(n, 1), 40).tolist()
        wanted.append(sorted({k for k in keys if 0 <= k < n}))
    g = torch.Generator().manual_seed(seed)
    k_cache = (60 * torch.randn(N, Hkv, P, W, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV)
    scales = [torch.exp2(torch.randint(-3, 3, (N, Hkv), generator=g).float()).to(DEV) for _ in "kv"]
    q = torch.zeros(int(cu[-1]), H, D, dtype=dtype, device=DEV)
    u, columns = torch.finfo(dtype).eps / 2, Hkv * D
    for at in range(0, max(len(w) for w in wanted), columns):
        v_cache = torch.zeros(N, Hkv, W, P, dtype=torch.uint8)
        want = np.zeros((int(cu[-1]), Hkv, D))
        vs = scales[1].cpu().numpy()
        for b, keys in enumerate(wanted):
            keys = np.array(keys[at:at + columns], dtype=np.int64)
            place = rng.permutation(columns)[: len(keys)]
            block = tables[b, keys // P]
            v_cache[block, place // D, place % D, keys % P] = 0x78                      # 256
            for i in range(new[b]):
                limit = lens[b] - new[b] + i + 1
                if limit > 0:
                    want[cu[b] + i, place // D, place % D] = np.where(keys < limit, 256.0 * vs[block, place // D] / limit, 0.0)
        out = kv.flash_attention_cached(q, k_cache, v_cache.view(torch.float8_e4m3fn).to(DEV), *scales, ints(tables), ints(lens), ints(cu), max_q_len=told)
        got = out.cpu().double().unflatten(1, (Hkv, group)).numpy()
        want = want[:, :, None]
        # Weights and scales are powers of two and meet one value: nothing is rounded but the sum of the weights (32 bits, a rounding for each of up to 700 units and parts)
        # and the result.
        bad = np.abs(got - want) > (u + 2.0 ** -14) * want
        assert not bad.any(), f"{bad.sum()} of {got.size}, first at (row, head, group, column) {tuple(np.argwhere(bad)[0])}"


BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
BLOCKS = pytest.mark.parametrize("P", [16, 32, 64, 128])


@BOTH
@BLOCKS
@pytest.mark.parametrize("D,Hkv,group", [(64, 4, 1), (128, 2, 4), (256, 1, 3), (192, 2, 1), (80, 1, 16)])
def test_single_tokens(kv, dtype, P, D, Hkv, group):
    check_counts(kv, [9001, 4, 1, 65, 2048, 701, 64, 0, 63], [1] * 9, Hkv, group, D, P, dtype, seed=1)
    check_counts(kv, [1, P, P + 1, 500, 1024, 1000], [1] * 6, Hkv, group, D, P, dtype, seed=2)       # (short caches: no row tile is cut)


@BOTH
@BLOCKS
def test_one_long_request(kv, dtype, P):
    check_counts(kv, [20001], [1], 2, 2, 128, P, dtype, seed=3)
    check_counts(kv, [12345, 2], [1, 1], 4, 1, 64, P, dtype, seed=4)


@BOTH
@BLOCKS
@pytest.mark.parametrize("D", [64, 128, 256])
def test_drafts(kv, dtype, P, D):
    check_counts(kv, [3000, 70, 131, 8], [8, 3, 5, 8], 2, 4, D, P, dtype, told=8, seed=5)
    check_counts(kv, [3000, 10, 701], [40, 3, 1], 1, 4, D, P, dtype, told=1, seed=6)                    # (more rows than the call was told of)


@BOTH
@BLOCKS
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_prompts(kv, dtype, P, D):
    check_counts(kv, [3064, 100], [200, 100], 1, 2, D, P, dtype, seed=7)                                # few row tiles: keys in parts
    check_counts(kv, [300, 37, 129, 64, 0], [150, 37, 1, 64, 3], 2, 4, D, P, dtype, seed=8)
    check_counts(kv, [190, 260], [190, 131], 8, 4, D, P, dtype, seed=9)
    check_counts(kv, [9012], [12], 2, 2, D, P, dtype, told=500, seed=10)


@BOTH
def test_many_requests(kv, dtype):
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 90, 700).tolist()
    check_counts(kv, lens, [1] * 700, 1, 2, 64, 16, dtype, seed=11)
    check_counts(kv, lens, rng.integers(0, 3, 700).tolist(), 1, 2, 64, 64, dtype, told=2, seed=12)
    check_counts(kv, lens, rng.integers(0, 3, 700).tolist(), 1, 2, 64, 64, dtype, told=100, seed=13)
