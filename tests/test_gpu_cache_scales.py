"""GPU tests of flash_attention_cached where value scales differ widely: a row's error is held against the row's own magnitude, whatever the scales of blocks are
that it does not see or gives no weight."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 64


@pytest.fixture(scope="module")
def kv():
    import flash_attention_amd.kv_cache as kv

    return kv


def reference(q, k, v, vs, lens):
    """one head in 64 bits: q [n, D], k [L, D] with their scale, v [L, D] code values, vs [L]; the out, sum p |v| and the largest p times its value's scale"""
    n, L = q.shape[0], k.shape[0]
    s = q @ k.t() * D ** -0.5
    see = torch.arange(L)[None] <= (lens - n + torch.arange(n))[:, None]
    p = torch.softmax(torch.where(see, s, -float("inf")), 1)
    value = v * vs[:, None]
    return p @ value, p @ value.abs(), (p * vs).amax(1, keepdim=True)


def check(kv, dtype, P, k, v, vs, n, rows_told):
    """k, v: [L, D] code values (k's scale is 1), vs: the value scale of every block; q is 8 in column 0 and random behind it"""
    L, blocks, g = k.shape[0], vs.numel(), torch.Generator().manual_seed(1)
    q = torch.randn(n, 1, D, generator=g).mul(0.02)
    q[:, :, 0] = 8.0
    q = q.to(dtype)
    pad = torch.zeros(blocks * P - L, D)
    kc = torch.cat([k, pad]).view(blocks, 1, P, D).to(torch.float8_e4m3fn)
    vc = torch.cat([v, pad]).view(blocks, 1, P, D).transpose(2, 3).contiguous().to(torch.float8_e4m3fn)
    assert torch.equal(kc.float().view(-1, D)[:L], k) and torch.equal(vc.float().transpose(2, 3).reshape(-1, D)[:L], v)     # (codes as they are)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = kv.flash_attention_cached(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.ones(blocks, 1, device=DEV), vs.float().view(-1, 1).to(DEV), ints([list(range(blocks))]),
                                    ints([L]), ints([0, n]), max_q_len=rows_told).cpu().double()[:, 0]
    ref, mag, peak = reference(q[:, 0].double(), k.double(), v.double(), vs.double().repeat_interleave(P)[:L], L)
    # The output is rounded once (in half steps of u, of 2^-25 at least in f16) and every weight once: u (|o| + sum p |v|), bf16 another u |o| for its sum of rounded
    # weights.  Scores reach 2^7: 2^-14 sum p |v|.  A half weight below the smallest normal is off by 2^-25 at most where the row's largest weight times scale is held
    # at 2^7 and more: 2^-32 of that for each of L codes up to 448.
    u = torch.finfo(dtype).eps / 2
    tol = 2 * u * ref.abs() + (u + 2.0 ** -14) * mag + ((2.0 ** -25 + L * 448 * 2.0 ** -32 * peak) if dtype == torch.float16 else 1e-30)
    assert bool(((out - ref).abs() <= tol).all()), f"{float(((out - ref).abs() / mag).max()):.3e} of the row's magnitude"


def codes(shape, low, high, g):
    """e4m3 values of either sign between low and high"""
    x = (low + (high - low) * torch.rand(shape, generator=g)) * (1 - 2.0 * torch.randint(0, 2, shape, generator=g))
    return x.to(torch.float8_e4m3fn).float()


BOTH = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
BLOCKS = pytest.mark.parametrize("P", [16, 32, 64, 128])


@BOTH
@BLOCKS
@pytest.mark.parametrize("apart", [10, 16, 20, 24, 50])
def test_scales_of_later_tokens(kv, dtype, P, apart):
    """rows of a prompt in front of a block whose values are 2^apart larger"""
    g = torch.Generator().manual_seed(apart)
    blocks = 4 if P < 64 else 2
    L = blocks * P
    k, v = codes((L, D), 0, 1, g), codes((L, D), 8, 100, g)
    k[:, 0] = 0
    vs = torch.full((blocks,), 2.0 ** -10)
    vs[-1] *= 2.0 ** apart
    v[-P:] = 0                  # (what the last rows see stays inside the type)
    v[-P:, 0] = 2.0 ** -4 if apart < 24 else 0
    check(kv, dtype, P, k, v, vs, L, L)                       # (tiles where L passes 64, else the row kernel)
    check(kv, dtype, P, k, v, vs, min(L, 64), 1)
    check(kv, dtype, P, k[: L - P], v[: L - P], vs[:-1], L - P, L)


@BOTH
@BLOCKS
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("apart", [12, 18, 26, 50])
def test_scales_of_blocks_without_weight(kv, dtype, P, n, apart):
    """a block with values 2^apart larger, whose keys score 112 below the others, first, last or between them"""
    g = torch.Generator().manual_seed(apart + 1)
    blocks = max(6, 384 // P)
    L = blocks * P - 3
    for where in (0, blocks // 2, blocks - 1):
        k, v = codes((L, D), 0, 1, g), codes((L, D), 8, 100, g)
        k[:, 0] = 0
        vs = torch.full((blocks,), 2.0 ** -10)
        vs[where] *= 2.0 ** apart
        k[where * P:(where + 1) * P, 0] = -112
        check(kv, dtype, P, k, v, vs, n, n)


@BOTH
@BLOCKS
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("below", [11, 15, 18])
def test_light_weights_on_large_values(kv, dtype, P, n, below):
    """tokens whose scores are `below` under the others and whose values make up for it"""
    g = torch.Generator().manual_seed(below)
    blocks = 1024 // P
    L = blocks * P
    k, v = codes((L, D), 0, 0.5, g), codes((L, D), 0.5, 1, g)
    k[:, 0] = 0
    vs = torch.full((blocks,), 2.0 ** -10)
    heavy = max(1, 128 // P)
    vs[-heavy:] = 2.0 ** (round(below / 0.6931) - 16)
    k[-heavy * P:, 0] = -float(below)
    v[-heavy * P:] = codes((heavy * P, D), 20, 60, g).abs()
    check(kv, dtype, P, k, v, vs, n, n)


@BOTH
@BLOCKS
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -100, 2.0 ** -70, 2.0 ** -64, 2.0 ** -40])
@pytest.mark.parametrize("below", [0, 8])
def test_weights_of_values_of_zero(kv, dtype, P, n, scale, below):
    """blocks of zeros, whatever their scale, hold most of a row's weight: it stays in the sum"""
    g = torch.Generator().manual_seed(below + 3)
    blocks = max(6, 384 // P)
    L = blocks * P - 5
    k, v = codes((L, D), 0, 1, g), codes((L, D), 8, 100, g)
    k[:, 0] = -float(below)
    vs = torch.full((blocks,), 2.0 ** 6)
    for b in (0, blocks // 2, blocks - 2):
        vs[b] = scale
        v[b * P:(b + 1) * P] = 0
        k[b * P:(b + 1) * P, 0] = 0
    check(kv, dtype, P, k, v, vs, n, n)
