"""GPU tests of the block cache: tables, append, attention, alone and together, against plain 64-bit forms."""

import numpy as np
import pytest
import torch

from kv_cache_reference import append_reference, attention_reference, e4m3_values, tables_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
VALUES = e4m3_values()


@pytest.fixture(scope="module")
def kv():
    import flash_attention_amd.kv_cache as kv

    return kv


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def code_values(cache):
    """code values as float64 on the CPU, from the bytes"""
    return torch.from_numpy(VALUES)[cache.view(torch.uint8).cpu().long()]


# ---- tables --------------------------------------------------------------------------------------------------------------------------
def make_tables(rng, held, P, width, spare, total=None):
    need = sum(-(-h // P) for h in held)
    total = need + spare if total is None else total
    ids = rng.permutation(total)
    tables = np.full((len(held), width), -1, np.int64)
    at = 0
    for b, h in enumerate(held):
        n = -(-h // P)
        tables[b, :n] = ids[at:at + n]
        at += n
    pool = np.full(total, -7, np.int64)
    pool[:spare] = ids[at:at + spare]
    return tables, pool


TABLE_CASES = [
    # requests, P, width, spare blocks, num_tokens - sum, chance of an end, most new tokens
    (1, 16, 4, 3, 0, 0.0, 1),
    (64, 64, 8, 100, 3, 0.1, 1),
    (7, 16, 3, 4, 0, 0.2, 40),         # not enough blocks, some rows too narrow
    (33, 32, 5, 1000, -9, 0.2, 50),    # the batch's rows do not hold all tokens
    (300, 128, 6, 50, 11, 0.3, 200),
    (1500, 16, 4, 700, 5, 0.3, 9),     # more requests than a workgroup has threads, two kernels
    (2600, 16, 3, 4000, 0, 0.2, 17),
    (40, 16, 64, 3000, 8, 0.0, 900),
    (5, 64, 4, 0, 2, 0.5, 3),          # an empty pool
]


@pytest.mark.parametrize("B,P,width,spare,slack,end,most", TABLE_CASES)
@pytest.mark.parametrize("inplace", [False, True])
def test_tables(kv, B, P, width, spare, slack, end, most, inplace):
    rng = np.random.default_rng(B * 131 + P)
    held = rng.integers(0, width * P - most if width * P > most else 1, B)
    held[rng.random(B) < 0.15] = 0
    new = rng.integers(0, most + 1, B)
    new[rng.random(B) < end] = -1
    tables, pool = make_tables(rng, held, P, width, spare)
    tokens = max(1, int(np.maximum(new, 0).sum()) + slack)
    ref = tables_reference(held.tolist(), new.tolist(), tables.tolist(), pool.tolist(), spare, tokens, P)
    t, f, s, c = ints(tables), ints(pool), ints(held), ints([spare])
    step = kv.cache_tables(s, ints(new), t, f, c, tokens, P, inplace=inplace)
    assert (step.seq_lens is s) == inplace and (step.free_count is c) == inplace
    if not inplace:
        assert s.tolist() == held.tolist() and c.item() == spare
    assert step.seq_lens.tolist() == ref["seq_lens"]
    assert step.free_count.tolist() == [ref["free"]]
    assert step.cu_new.tolist() == ref["cu"]
    assert step.granted.tolist() == ref["granted"]
    assert step.positions.tolist() == ref["positions"]
    assert step.slots.tolist() == ref["slots"]
    assert t.tolist() == ref["tables"] and f.tolist() == ref["pool"]


def test_tables_no_tokens_and_strided_rows(kv):
    big = ints(np.full((4, 9), -1))
    t = big[:, 2:6]                                     # rows inside a wider table
    step = kv.cache_tables(ints([0, 0, 0, 0]), ints([0, 0, 0, 0]), t, ints([1, 2, 3]), ints([3]), 0, 16)
    assert step.slots.numel() == 0 and step.free_count.item() == 3
    step = kv.cache_tables(ints([0, 0, 0, 0]), ints([0, 17, 0, 1]), t, ints([1, 2, 3]), ints([3]), 18, 16)
    assert big.tolist() == [[-1] * 9, [-1, -1, 3, 2] + [-1] * 5, [-1] * 9, [-1, -1, 1] + [-1] * 6]
    assert step.slots.tolist() == [48 + i for i in range(16)] + [32, 16]


def test_tables_saturates(kv):
    """lengths whose sum passes 2^31 are refused, not wrapped"""
    t = ints(np.full((3, 2), -1))
    step = kv.cache_tables(ints([0, 0, 5]), ints([2 ** 31 - 1, 2 ** 31 - 1, 1]), t, ints([4, 5, 6]), ints([3]), 8, 16)
    assert step.granted.tolist() == [0, 0, 0] and step.seq_lens.tolist() == [0, 0, 5] and step.free_count.item() == 3
    assert step.slots.tolist() == [-1] * 8 and min(step.cu_new.tolist()) >= 0


# ---- append --------------------------------------------------------------------------------------------------------------------------
def empty_cache(kv, N, H, P, D, fill=0x5A):
    W = kv.cache_width(D)
    k = torch.full((N, H, P, W), fill, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.full((N, H, W, P), fill, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    return k, v, torch.full((N, H), 0.5, device=DEV), torch.full((N, H), 0.25, device=DEV)


def check_append(kv, runs, N, H, P, D, dtype, seed, k=None, v=None, edge=None, cache=None):
    """runs: [(first slot, tokens)] in order; negative first slots are padding"""
    g = torch.Generator().manual_seed(seed)
    slots = [s + i if s >= 0 else s for s, n in runs for i in range(n)]
    T = len(slots)
    k, v = (torch.randn(T, H, D, generator=g).mul(torch.exp2(torch.randint(-6, 6, (T, 1, 1), generator=g).float())).to(dtype) for _ in "kv")
    if edge is not None:
        edge(k, v)
    cache = empty_cache(kv, N, H, P, D) if cache is None else cache
    kc, vc, ks, vs = cache
    want = []
    for x, c, s, keys in ((k, kc, ks, True), (v, vc, vs, False)):
        values, scale = code_values(c).numpy(), s.cpu().double().numpy().copy()
        values = values.copy() if keys else np.ascontiguousarray(values.transpose(0, 1, 3, 2))
        append_reference(x.double().numpy(), slots, values, scale, P)
        want.append((values, scale))
    kv.cache_append(k.to(DEV), v.to(DEV), ints(slots), kc, vc, ks, vs)
    got_k, got_v = code_values(kc).numpy(), code_values(vc).numpy().transpose(0, 1, 3, 2)
    np.testing.assert_array_equal(ks.cpu().double().numpy(), want[0][1])
    np.testing.assert_array_equal(vs.cpu().double().numpy(), want[1][1])
    np.testing.assert_array_equal(got_k, want[0][0])
    np.testing.assert_array_equal(got_v, want[1][0])
    return cache


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("D,H", [(64, 3), (128, 2), (80, 5), (256, 1), (8, 12), (192, 2)])
def test_append_runs(kv, dtype, P, D, H):
    """single tokens, a run over three blocks that begins inside one, odd ends, padding between"""
    runs = [(3 * P, 1), (-1, 2), (5, 1), (P + 7, 9), (4 * P + 3, P - 3), (6 * P, P), (2 * P, 5), (-5, 1), (7 * P + P - 1, 1)]
    cache = check_append(kv, runs, 9, H, P, D, dtype, 1)
    check_append(kv, [(3 * P + 1, 1), (6, 3), (P + 16 - 0, 0), (2 * P + 5, 1)], 9, H, P, D, dtype, 2, cache=cache)


def test_append_many_windows(kv):
    """more tokens than a window of the kernel holds: runs that begin in one and end in another, single tokens in between"""
    P, runs, at = 64, [], 0
    rng = np.random.default_rng(5)
    for b in rng.permutation(400)[:300]:
        off = int(rng.integers(0, P)) if rng.random() < 0.5 else 0
        n = 1 if rng.random() < 0.4 else int(rng.integers(1, P - off + 1))
        runs.append((int(b) * P + off, n))
    check_append(kv, runs, 400, 8, P, 64, torch.bfloat16, 3)
    check_append(kv, [(int(b) * P + 7, 1) for b in rng.permutation(400)], 400, 8, P, 64, torch.float16, 4)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_scale_grows_and_codes_follow(kv, dtype):
    cache = check_append(kv, [(0, 4), (64, 1)], 3, 2, 64, 128, dtype, 1, edge=lambda k, v: (k.mul_(2.0 ** -8), v.mul_(2.0 ** -8)))
    for i, f in enumerate((1.0, 2.0 ** 5, 2.0 ** -3)):
        check_append(kv, [(4 + i, 1), (65 + i, 1)], 3, 2, 64, 128, dtype, 10 + i, edge=lambda k, v: (k.mul_(f), v.mul_(f)), cache=cache)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_borders(kv, dtype):
    """zeros, the exact border of a scale, subnormals, the type's largest value, inf and NaN"""
    def edge(k, v):
        k[0], v[0] = 0, 0
        k[1, 0], k[1, 0, 0] = 1.0, 448.0
        k[2, 0], k[2, 0, 0] = 1.0, 450.0 if dtype == torch.bfloat16 else 448.25
        k[3] = torch.finfo(dtype).tiny / 4
        k[4, 1, 3] = torch.finfo(dtype).max
        v[4, 1, 3] = -torch.finfo(dtype).max
        v[5, 0, 1], v[5, 0, 2], v[5, 1, 3] = float("inf"), float("nan"), float("-inf")
        k[6] = float("nan")
        v[6, 0] = float("inf")
    check_append(kv, [(0, 1), (16, 1), (32, 1), (48, 1), (64, 1), (80, 1), (96, 1)], 8, 2, 16, 64, dtype, 9, edge=edge)


def test_append_skips_what_is_outside(kv):
    cache = empty_cache(kv, 3, 2, 16, 64)
    before = [t.clone() for t in cache]
    x = torch.ones(6, 2, 64, dtype=torch.float16, device=DEV)
    kv.cache_append(x, x, ints([-1, 48, 2 ** 31 - 1, -2 ** 31, 1000, 49]), *cache)
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
    kv.cache_append(x[:0], x[:0], ints([]), *cache)


def test_append_strided_operands_and_layers(kv):
    """keys and values as slices of one projection, the cache a layer of a larger tensor; unaligned rows are copied"""
    H, D, P, N = 4, 64, 32, 6
    fused = torch.randn(9, 3 * H * D + 8, device=DEV).bfloat16()
    k, v = (fused[:, i * H * D:(i + 1) * H * D].view(9, H, D) if False else fused[:, i * H * D:(i + 1) * H * D].unflatten(1, (H, D)) for i in (1, 2))
    layers = [torch.zeros((N, 2, H, P, 64), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros((N, 2, H, 64, P), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)]
    scales = [torch.ones(N, 2, H, device=DEV) for _ in "kv"]
    slots = ints([33, 34, 35, 64, 0, 1, 2, 3, -1])
    kv.cache_append(k, v, slots, layers[0][:, 1], layers[1][:, 1], scales[0][:, 1], scales[1][:, 1])
    plain = [torch.zeros((N, H, P, 64), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros((N, H, 64, P), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
             torch.ones(N, H, device=DEV), torch.ones(N, H, device=DEV)]
    kv.cache_append(k.contiguous(), v.contiguous(), slots, *plain)
    assert torch.equal(layers[0][:, 1].contiguous().view(torch.uint8), plain[0].view(torch.uint8)) and torch.equal(scales[1][:, 1], plain[3])
    assert torch.equal(layers[1][:, 1].contiguous().view(torch.uint8), plain[1].view(torch.uint8))
    assert int(layers[0][:, 0].contiguous().view(torch.uint8).sum()) == 0 and int(layers[1][:, 0].contiguous().view(torch.uint8).sum()) == 0
    odd = torch.randn(9, H, D + 1, device=DEV).bfloat16()[..., 1:]           # rows that start at odd elements
    again = [t.clone() for t in plain]
    kv.cache_append(odd, odd, slots, *plain)
    kv.cache_append(odd.contiguous(), odd.contiguous(), slots, *again)
    assert torch.equal(plain[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(plain[1].view(torch.uint8), again[1].view(torch.uint8))


# ---- attention -----------------------------------------------------------------------------------------------------------------------
def random_cache(kv, g, N, H, P, D):
    W = kv.cache_width(D)
    codes = lambda *s: (60 * torch.randn(*s, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    k, v = codes(N, H, P, W), codes(N, H, W, P)
    if W != D:
        k.view(torch.uint8)[..., D:] = 0
    scale = lambda: torch.exp2(torch.randint(-8, -4, (N, H), generator=g).float()) * (1 + torch.rand(N, H, generator=g))  # noqa: E731  (any positive scale)
    return [t.to(DEV) for t in (k, v, scale(), scale())]


def tolerance(dtype, out, mag, vmax, keys):
    """u: half a step.  The output is rounded once, every weight once: u |o| + u sum p |v|.  Half weights are added up before they are rounded, bf16 ones after:
    sum w (1 + d) v / sum w (1 + d) with |d| <= u is off by at most u sum p |v - o| <= u (sum p |v| + |o|).  32-bit products, maximum and exponentials: a score of
    magnitude s is off by some s 2^-22 and its weight by as much; 2^-12 sum p |v| covers |s| up to 2^10.  A weight below the smallest normal half is off by at most
    2^-25 (the sum of the weights is at least 1)."""
    u = torch.finfo(dtype).eps / 2
    return (u if dtype == torch.float16 else 2 * u) * out.abs() + (u + 2.0 ** -12) * mag + (keys * 2.0 ** -25 * vmax if dtype == torch.float16 else 1e-30)


def check_attention(kv, held, new, Hkv, group, D, P, dtype, seed=0, max_q_len=None, bad=(), poke=None, pad=0, cache=None):
    """held: tokens in front; new: queries (the last tokens)"""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed + 17)
    lens = [h + n for h, n in zip(held, new)]
    width = max(1, max(-(-x // P) for x in lens)) + 1
    need = sum(-(-x // P) for x in lens)
    N = need + 3
    ids = rng.permutation(N)
    tables = np.full((len(lens), width), -1, np.int64)
    at = 0
    for b, x in enumerate(lens):
        n = -(-x // P)
        tables[b, :n] = ids[at:at + n]
        at += n
    for b, j, value in bad:
        tables[b, j] = value
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    T = cu[-1] + pad
    q = (torch.randn(T, Hkv * group, D, generator=g) * 1.5).to(dtype)
    k, v, ks, vs = random_cache(kv, g, N, Hkv, P, D)
    # whatever lies behind a request's last token must not matter: NaN codes there
    for b, x in enumerate(lens):
        if x % P and tables[b, x // P] >= 0 and tables[b, x // P] < N:
            k.view(torch.uint8)[tables[b, x // P], :, x % P:] = 0x7F
            v.view(torch.uint8)[tables[b, x // P], :, :, x % P:] = 0xFF
    if poke is not None:
        poke(k, v, tables, lens)
    out = torch.full((T, Hkv * group, D), 7.0, dtype=dtype, device=DEV)
    got = kv.flash_attention_cached(q.to(DEV), k, v, ks, vs, ints(tables), ints(lens), ints(cu), max_q_len=max_q_len, out=out)
    assert got is out
    kval, vval = code_values(k), code_values(v).transpose(2, 3)
    ref, mag = attention_reference(q.double(), kval, vval, ks.cpu().double(), vs.cpu().double(), tables.tolist(), lens, cu, D ** -0.5)
    if pad:
        assert bool((out[cu[-1]:] == 7.0).all())           # rows behind the last request: left as they were
    out, ref, mag = out[: cu[-1]].cpu().double(), ref[: cu[-1]], mag[: cu[-1]]
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    vmax = 448 * float(vs.max())
    err, tol = (out - ref).abs(), tolerance(dtype, ref, mag, vmax, max(lens + [1]))
    fine = ~torch.isnan(ref)
    assert bool((err[fine] <= tol[fine]).all()), f"max |delta| {err[fine].max():.3e}, over by {(err - tol)[fine].max():.3e}"
    return out


BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])


@BOTH
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("D,Hkv,group", [(64, 3, 1), (128, 2, 4), (128, 1, 16), (256, 1, 3), (192, 2, 2), (80, 2, 3), (8, 1, 1)])
def test_single_tokens(kv, dtype, P, D, Hkv, group):
    held = [0, 1, P - 1, P, 62, 63, 64, 300, 129]
    check_attention(kv, held, [1] * len(held), Hkv, group, D, P, dtype)


@BOTH
@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("D,Hkv,group", [(64, 2, 1), (128, 2, 8), (128, 1, 32), (256, 1, 2), (192, 1, 6)])
def test_drafts(kv, dtype, P, D, Hkv, group):
    """several tokens per request through the row kernel: up to 32 rows of a key/value head, and more than it was told of"""
    check_attention(kv, [0, 70, 5, 200, 31], [4, 3, 1, 2, 4], Hkv, group, D, P, dtype, max_q_len=4 if group <= 8 else 1)
    check_attention(kv, [3, 500], [9, 1], Hkv, group, D, P, dtype, max_q_len=1)


@BOTH
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("D,Hkv,group", [(64, 2, 3), (128, 2, 4), (256, 1, 2), (192, 1, 1), (96, 1, 5)])
def test_prompts(kv, dtype, P, D, Hkv, group):
    check_attention(kv, [0, 37, 200, 0, 64], [70, 45, 1, 130, 64], Hkv, group, D, P, dtype)


def test_prompts_without_split(kv):
    """enough row tiles that none is split"""
    check_attention(kv, [100, 0, 3], [150, 171, 160], 16, 8, 64, 64, torch.bfloat16)


@BOTH
def test_lengths_that_cross_ranges(kv, dtype):
    """one long request beside short ones: split over many workgroups, every border somewhere else"""
    check_attention(kv, [9000, 3, 0, 64, 2047, 700], [1] * 6, 2, 4, 128, 64, dtype, seed=3)
    check_attention(kv, [20000], [1], 1, 2, 64, 16, dtype, seed=4)
    check_attention(kv, [5000, 100], [2, 2], 1, 16, 128, 128, dtype, seed=5)


@BOTH
def test_many_requests(kv, dtype):
    rng = np.random.default_rng(8)
    held = rng.integers(0, 40, 700).tolist()
    check_attention(kv, held, [1] * 700, 1, 2, 64, 16, dtype, seed=6)
    new = rng.integers(0, 3, 700).tolist()
    check_attention(kv, held, new, 1, 2, 64, 32, dtype, seed=7, max_q_len=2)


@BOTH
@pytest.mark.parametrize("max_q_len", [1, 40])
def test_empty_requests_and_rows_without_keys(kv, dtype, max_q_len):
    """no queries, no tokens at all (zeros), fewer tokens than queries (the first see nothing), padding behind"""
    check_attention(kv, [50, 0, 20, -2, 0], [0, 1, 0, 5, 2], 2, 2, 64, 16, dtype, max_q_len=max_q_len, pad=3)
    out = check_attention(kv, [-1, 60], [1, 1], 2, 2, 128, 64, dtype, max_q_len=max_q_len)
    assert bool((out[0] == 0).all())


@BOTH
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("max_q_len", [1, 40])
def test_blocks_that_do_not_exist(kv, dtype, P, max_q_len):
    """table entries outside the cache: their keys are not seen"""
    bad = [(0, 0, -1), (1, 1, 10 ** 6), (2, 0, -(2 ** 31)), (2, 1, 2 ** 31 - 1)]
    check_attention(kv, [3 * P, 3 * P + 5, P + 3], [1, 2, 2], 2, 2, 64, P, dtype, bad=bad, max_q_len=max_q_len)
    check_attention(kv, [P - 1], [1], 1, 1, 64, P, dtype, bad=[(0, 0, -1)], max_q_len=max_q_len)


@BOTH
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("max_q_len", [2, 60])
def test_nan_reaches_only_the_rows_that_see_it(kv, dtype, P, max_q_len):
    """a NaN value of a later token must not reach the tokens in front of it in the same unit"""
    def poke(k, v, tables, lens):
        for b, t, col in ((0, 70, 3), (1, 9, 60), (1, 10, 0)):
            v.view(torch.uint8)[int(tables[b, t // P]), 0, col, t % P] = 0x7F
        k.view(torch.uint8)[int(tables[2, 20 // P]), 1, 20 % P, 5] = 0xFF
    out = check_attention(kv, [60, 0, 0], [30, 20, 40], 2, 2, 64, P, dtype, poke=poke, max_q_len=max_q_len)
    assert bool(torch.isnan(out[10:30, :2, 3]).all()) and not bool(torch.isnan(out[:10]).any())


@BOTH
def test_large_scores_and_scales(kv, dtype):
    """one key far above the others, key scales that differ by 2^16 between blocks of one unit, value scales of zero"""
    g = torch.Generator().manual_seed(0)
    N, P, D = 8, 16, 64
    k, v, ks, vs = random_cache(kv, g, N, 1, P, D)
    ks[:, 0] = torch.tensor([2.0 ** e for e in (-14, 0, -3, -8, 2, -20, -6, -1)])
    vs[:, 0] = torch.tensor([0.0, 2.0 ** -20, 1.0, 2.0 ** 10, 0.0, 0.0, 2.0 ** -6, 3.0])
    q = torch.randn(3, 2, D, generator=g).to(dtype).to(DEV)
    tables, lens, cu = ints([[0, 1, 2, 3, 4, 5, 6, 7], [0, 4, 5, 0, 0, 0, 0, 0], [3, 2, 1, 0, 7, 0, 0, 0]]), [128, 40, 70], [0, 1, 2, 3]
    out = kv.flash_attention_cached(q, k, v, ks, vs, tables, ints(lens), ints(cu)).cpu().double()
    ref, mag = attention_reference(q.cpu().double(), code_values(k), code_values(v).transpose(2, 3), ks.cpu().double(), vs.cpu().double(), tables.tolist(), lens, cu, D ** -0.5)
    # (scores reach 2^13 here: 2^-9 in the place of 2^-12)
    assert bool(((out - ref).abs() <= tolerance(dtype, ref, mag, 448 * 1024, 128) + 2.0 ** -9 * mag).all())
    assert bool((out[1] == 0).all())


@BOTH
@pytest.mark.parametrize("D", [64, 128, 256])
def test_more_rows_than_the_call_was_told_of(kv, dtype, D):
    """parts of many row tiles that are joined although max_q_len said one row, and one tile although it said many"""
    check_attention(kv, [3000, 10, 700], [40, 3, 1], 1, 4, D, 64, dtype, seed=21, max_q_len=1)
    check_attention(kv, [9000], [12], 2, 2, D, 16, dtype, seed=22, max_q_len=1)
    check_attention(kv, [5000, 0], [1, 2], 1, 2, D, 128, dtype, seed=23, max_q_len=500)


@BOTH
@pytest.mark.parametrize("D,group,new", [(64, 8, 8), (64, 16, 3), (128, 8, 4), (256, 4, 4)])
def test_as_many_rows_as_the_row_kernel_takes(kv, dtype, D, group, new):
    check_attention(kv, [6000, 5], [new, new], 1, group, D, 64, dtype, seed=24)
    check_attention(kv, [6000, 5], [new + 1, new], 1, group, D, 64, dtype, seed=25)


@BOTH
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("held,new", [([3000], [64]), ([2900, 0], [200, 30]), ([100], [300]), ([1500] * 3 + [0], [70, 1, 33, 129])])
def test_prompts_in_parts(kv, dtype, D, held, new):
    """few row tiles: their keys are cut into parts, more of them than a short request has units"""
    check_attention(kv, held, new, 1, 2, D, 64, dtype, seed=26)


def test_a_layout_is_looked_at_in_every_call(kv):
    """the same shapes with other strides, after a call that passed"""
    layer = kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=16)._layer[0]
    k = torch.zeros(4, 2, 64, dtype=torch.float16, device=DEV)
    kv.cache_append(k, k, ints([0, 1, 2, 3]), *layer)
    for slots in (ints([0, 9, 1, 9, 2, 9, 3, 9])[::2], ints([0]).expand(4)):
        with pytest.raises(ValueError):
            kv.cache_append(k, k, slots, *layer)
    with pytest.raises(ValueError, match="no gradient"):
        kv.cache_append(k.clone().requires_grad_(), k, ints([0, 1, 2, 3]), *layer)
    with torch.no_grad():
        kv.cache_append(k.clone().requires_grad_(), k, ints([0, 1, 2, 3]), *layer)


def test_offsets_behind_32_bits(kv):
    """blocks that begin behind 4 GiB of codes"""
    N, H, P, D = 70000, 8, 64, 128
    k = torch.zeros((N, H, P, D), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.zeros((N, H, D, P), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    ks, vs = torch.ones(N, H, device=DEV), torch.ones(N, H, device=DEV)
    far = N - 2
    x = torch.randn(70, H, D, device=DEV).bfloat16()
    kv.cache_append(x, x, ints(list(range(far * P, far * P + 70))), k, v, ks, vs)
    small = [k[far:].clone(), v[far:].clone(), ks[far:].clone(), vs[far:].clone()]
    assert int(k[:4].view(torch.uint8).sum()) == 0 and int(small[0].view(torch.uint8).sum()) > 0
    q = torch.randn(1, 16, D, device=DEV).bfloat16()
    a = kv.flash_attention_cached(q, k, v, ks, vs, ints([[far, far + 1]]), ints([70]), ints([0, 1]))
    b = kv.flash_attention_cached(q, *small, ints([[0, 1]]), ints([70]), ints([0, 1]))
    assert torch.equal(a, b) and float(a.float().abs().max()) > 0
    q = torch.randn(70, 16, D, device=DEV).bfloat16()
    a = kv.flash_attention_cached(q, k, v, ks, vs, ints([[far, far + 1]]), ints([70]), ints([0, 70]))
    b = kv.flash_attention_cached(q, *small, ints([[0, 1]]), ints([70]), ints([0, 70]))
    assert torch.equal(a, b)


@BOTH
@pytest.mark.parametrize("new", [1, 50])
def test_strided_queries_and_output(kv, dtype, new):
    g = torch.Generator().manual_seed(3)
    k, v, ks, vs = random_cache(kv, g, 9, 2, 64, 128)
    T = 3 * new
    fused = torch.randn(T, 6 * 128 + 8, generator=g).to(dtype).to(DEV)
    q = fused[:, 128:128 * 5].unflatten(1, (4, 128))
    tables, lens, cu = ints(np.arange(9).reshape(3, 3)), ints([130 + new, 64 + new, new]), ints([0, new, 2 * new, T])
    room = torch.zeros(T, 4, 2, 128, dtype=dtype, device=DEV)
    want = kv.flash_attention_cached(q.contiguous(), k, v, ks, vs, tables, lens, cu)
    kv.flash_attention_cached(q, k, v, ks, vs, tables, lens, cu, out=room[:, :, 1])
    assert torch.equal(room[:, :, 1], want) and float(room[:, :, 0].float().abs().max()) == 0
    odd = torch.randn(T, 4, 129, generator=g).to(dtype).to(DEV)[..., 1:]
    assert torch.equal(kv.flash_attention_cached(odd, k, v, ks, vs, tables, lens, cu), kv.flash_attention_cached(odd.contiguous(), k, v, ks, vs, tables, lens, cu))
    heads_first = torch.randn(4, T, 128, generator=g).to(dtype).to(DEV).transpose(0, 1)
    assert torch.equal(kv.flash_attention_cached(heads_first, k, v, ks, vs, tables, lens, cu),
                       kv.flash_attention_cached(heads_first.contiguous(), k, v, ks, vs, tables, lens, cu))
    many_rows = torch.cat([tables, tables], 1)[:, :3]
    assert torch.equal(kv.flash_attention_cached(q, k, v, ks, vs, many_rows, lens, cu), want)


@pytest.mark.parametrize("new", [1, 40])
def test_reproducible(kv, new):
    g = torch.Generator().manual_seed(5)
    k, v, ks, vs = random_cache(kv, g, 40, 2, 64, 128)
    q = torch.randn(2 * new, 8, 128, generator=g).bfloat16().to(DEV)
    args = (k, v, ks, vs, ints(np.arange(40).reshape(2, 20)), ints([1250, 700]), ints([0, new, 2 * new]))
    first = kv.flash_attention_cached(q, *args)
    for _ in range(5):
        assert torch.equal(kv.flash_attention_cached(q, *args), first)


# ---- together ------------------------------------------------------------------------------------------------------------------------
def run_steps(kv, cache, steps, q, k, v):
    outs = []
    for i, (new, tokens, most) in enumerate(steps):
        step = cache.step(new, tokens)
        outs.append(cache.attend(0, q[i], k[i], v[i], step, max_q_len=most))
    return outs


def test_generation_steps(kv):
    """prompts, single tokens, a request that ends and a new one in its place: lengths, tables, codes and attention after every step"""
    B, H, Hkv, D, P = 3, 4, 2, 64, 16
    cache = kv.KVCache(2, 40, Hkv, D, requests=B, max_tokens=200, block_size=P)
    cache.k_cache.view(torch.uint8).fill_(0x7F)
    cache.v_cache.view(torch.uint8).fill_(0x7F)
    g = torch.Generator().manual_seed(1)
    history = [np.zeros((0, Hkv, D)) for _ in range(B)], [np.zeros((0, Hkv, D)) for _ in range(B)]
    for new in ([20, 0, 33], [1, 7, 1], [1, 1, 1], [-1, 1, 1], [18, 1, 1], [1, 1, 1]):
        tokens = sum(max(n, 0) for n in new) + 2
        q, k, v = (torch.randn(tokens, h, D, generator=g).half() for h in (H, Hkv, Hkv))
        step = cache.step(ints(new), tokens)
        out = cache.attend(1, q.to(DEV), k.to(DEV), v.to(DEV), step)
        at = 0
        for b in range(B):
            n = max(new[b], 0)
            for hist, x in zip(history, (k, v)):
                hist[b] = np.concatenate([hist[b][: 0 if new[b] < 0 else None], x[at:at + n].double().numpy()])
            at += n
        lens = cache.seq_lens.tolist()
        assert lens == [len(h) for h in history[0]]
        kval, vval = code_values(cache.k_cache[1]), code_values(cache.v_cache[1]).transpose(2, 3)
        ks, vs = cache.k_scale[1].cpu().double(), cache.v_scale[1].cpu().double()
        tables = cache.block_tables.tolist()
        for b in range(B):                       # the cache holds what was appended, to half a step of e4m3 (2^-4, and 2^-10 of the scale below its smallest normal
            for t in range(lens[b]):             # code), twice: a scale that grew rounded again
                blk = tables[b][t // P]
                for got, scale, hist in ((kval, ks, history[0]), (vval, vs, history[1])):
                    have = got[blk, :, t % P, :D].numpy() * scale[blk].numpy()[:, None]
                    assert (np.abs(have - hist[b][t]) <= 2 * (np.abs(hist[b][t]) * 2.0 ** -4 + 2.0 ** -10 * scale[blk].numpy()[:, None])).all()
        ref, mag = attention_reference(q.double(), kval, vval, ks, vs, tables, lens, step.cu_new.tolist(), D ** -0.5)
        n = step.cu_new.tolist()[-1]
        assert bool(((out[:n].cpu().double() - ref[:n]).abs() <= tolerance(torch.float16, ref, mag, 448 * float(vs.max()), max(lens))[:n]).all())
    used = sum(-(-n // P) for n in cache.seq_lens.tolist())
    assert cache.free_count.item() == 40 - used
    live = cache.free_blocks[: 40 - used].tolist() + [i for b, n in enumerate(cache.seq_lens.tolist()) for i in cache.block_tables[b].tolist()[: -(-n // P)]]
    assert sorted(live) == list(range(40))       # no block twice, none lost


def test_captured_step_replays(kv):
    """a captured step advances lengths, tables and pool with every replay, as the eager one does, other work and synchronisation between"""
    B, H, Hkv, D = 4, 8, 2, 128
    g = torch.Generator().manual_seed(2)
    caches = [kv.KVCache(1, 64, Hkv, D, requests=B, max_tokens=512) for _ in range(2)]
    q, k, v = (torch.randn(B, h, D, generator=g).bfloat16().to(DEV) for h in (H, Hkv, Hkv))
    prompt = [torch.randn(50 * B, h, D, generator=g).bfloat16().to(DEV) for h in (H, Hkv, Hkv)]
    ones = ints([1] * B)
    for c in caches:
        c.k_cache.view(torch.uint8).fill_(0x7F)      # (never written places are compared too)
        c.attend(0, *prompt, c.step(ints([50, 61, 39, 50]), 50 * B))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                # warm up on a copy of the state
        w = kv.KVCache(1, 64, Hkv, D, requests=B, max_tokens=512)
        w.attend(0, q, k, v, w.step(ones, B))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = caches[0].attend(0, q, k, v, caches[0].step(ones, B))
    for i in range(20):
        for t, h in ((q, H), (k, Hkv), (v, Hkv)):
            t.copy_(torch.randn(B, h, D, generator=g).mul(1 + i).bfloat16())
        graph.replay()
        want = caches[1].attend(0, q, k, v, caches[1].step(ones, B))
        junk = torch.randn(1 << 20, device=DEV).sum().item()
        assert junk == junk and torch.equal(out, want)
        assert torch.equal(caches[0].seq_lens, caches[1].seq_lens) and torch.equal(caches[0].block_tables, caches[1].block_tables)
        assert torch.equal(caches[0].k_cache.view(torch.uint8)[0, caches[0].block_tables[0, 0]], caches[1].k_cache.view(torch.uint8)[0, caches[1].block_tables[0, 0]])


def test_two_graphs_and_a_side_stream(kv):
    """two captured attention calls replayed on two streams at once: no workspace is shared"""
    g = torch.Generator().manual_seed(6)
    k, v, ks, vs = random_cache(kv, g, 300, 2, 64, 128)
    sets = []
    for i in range(2):
        q = torch.randn(2, 8, 128, generator=g).half().to(DEV)
        sets.append((q, k, v, ks, vs, ints(np.random.default_rng(i).permutation(300)[:200].reshape(2, 100)), ints([6000 - 100 * i, 3000 + i]), ints([0, 1, 2])))
    want = [kv.flash_attention_cached(*s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(kv.flash_attention_cached(*s))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    with torch.cuda.stream(streams[0]):
        a = kv.flash_attention_cached(*sets[0])
    b = kv.flash_attention_cached(*sets[1])
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_compiled(kv):
    """torch.compile carries the calls as opaque ops"""
    B, H, Hkv, D = 2, 4, 2, 64
    a, b = (kv.KVCache(1, 16, Hkv, D, requests=B, max_tokens=128) for _ in range(2))
    q, k, v = (torch.randn(6, h, D, device=DEV).half() for h in (H, Hkv, Hkv))
    new = ints([4, 2])

    def one(c):
        return c.attend(0, q * 1.0, k, v, c.step(new, 6), max_q_len=4)

    want = one(a)
    got = torch.compile(one, fullgraph=True, backend="aot_eager")(b)
    assert torch.equal(got, want) and torch.equal(a.seq_lens, b.seq_lens)


def test_refusals(kv):
    c = kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=16)
    layer = c._layer[0]
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV)
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV)
    lens, cu, slots = ints([1, 1]), ints([0, 1, 2]), ints([0, 16])
    call = lambda **kw: kv.flash_attention_cached(**{**dict(q=q, k_cache=layer[0], v_cache=layer[1], k_scale=layer[2], v_scale=layer[3], block_tables=c.block_tables, seq_lens=lens, cu_q=cu), **kw})  # noqa: E731
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :3]), dict(q=q[..., :60]), dict(seq_lens=lens.long()), dict(cu_q=cu[:2]), dict(block_tables=c.block_tables[:1]),
                dict(block_tables=c.block_tables.long()), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(max_q_len=0), dict(out=q.float()),
                dict(out=torch.zeros(2, 4, 65, dtype=torch.float16, device=DEV)[..., 1:]), dict(k_cache=layer[1]), dict(k_cache=layer[0].view(torch.uint8)),
                dict(k_scale=layer[2].double()), dict(v_scale=layer[3][:4]), dict(q=q.cpu()), dict(seq_lens=lens.cpu()), dict(q=q.clone().requires_grad_())):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    for bad in ((k.float(), k.float(), slots), (k, k[:1], slots), (k, k, slots.long()), (k, k, slots[:1]), (k[:, :1], k[:, :1], slots), (k[..., :60], k[..., :60], slots)):
        with pytest.raises((ValueError, TypeError)):
            kv.cache_append(*bad, *layer)
    for bad in (dict(block_size=24), dict(num_tokens=-1), dict(new_lens=lens.long()), dict(new_lens=ints([1])), dict(free_count=ints([1, 2])), dict(free_blocks=ints([[1]])),
                dict(block_tables=c.block_tables.t()), dict(new_lens=lens.cpu())):
        with pytest.raises((ValueError, TypeError)):
            kv.cache_tables(**{**dict(seq_lens=lens, new_lens=lens, block_tables=c.block_tables, free_blocks=c.free_blocks, free_count=c.free_count, num_tokens=2, block_size=16), **bad})
    with pytest.raises(ValueError):
        kv.KVCache(1, 8, 2, 60, requests=2, max_tokens=64)
    with pytest.raises(ValueError):
        kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=48)
    assert call().shape == q.shape
