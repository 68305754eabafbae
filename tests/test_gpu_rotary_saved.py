"""GPU tests of qk_norm_rope's backward where autograd hands the saved tensors back in another layout than the forward's."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def rot():
    import flash_attention_amd.rotary as rot

    return rot


def operands(dtype, D, layout, seed=0):
    """q, k with strides of their own, positions as a slice of a wider tensor"""
    g = torch.Generator().manual_seed(seed)
    B, L, H, Hk = 2, 33, 4, 2
    fused = torch.randn(B, L, (H + 2 * Hk) * D, generator=g).to(dtype).to(DEV).unflatten(-1, (-1, D))
    q, k = fused[:, :, :H].transpose(1, 2), fused[:, :, H:H + Hk].transpose(1, 2)
    if layout == "transposed":                  # (columns behind rows in memory)
        q, k = (t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k))
    positions = torch.randint(-1, 2 * L, (B, 4 * L), generator=g).to(DEV)[:, L:2 * L]
    weights = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).to(DEV).requires_grad_() for _ in "qk"]
    grads = [torch.randn(t.shape, generator=g).to(dtype).to(DEV) for t in (q, k)]
    return [q.detach().requires_grad_(), k.detach().requires_grad_(), *weights], positions, grads


def gradients(rot, leaves, positions, grads, table):
    out = rot.qk_norm_rope(*leaves, table, positions)
    return torch.autograd.grad(out, leaves, grads)


def wide(t):
    """the tensor as a view of one with room behind every row"""
    room = torch.empty(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device) if t.ndim else torch.empty_like(t)
    return room[..., : t.shape[-1]].copy_(t) if t.ndim > 1 else t


HOOKS = {"contiguous": lambda t: t.contiguous(), "wide": lambda t: wide(t) if t.dtype != torch.float32 else t,
         "columns": lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.ndim > 2 else t}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80])
@pytest.mark.parametrize("layout", ["fused", "transposed"])
@pytest.mark.parametrize("hook", ["cpu", *HOOKS])
def test_saved_tensors_in_another_layout(rot, dtype, D, layout, hook):
    leaves, positions, grads = operands(dtype, D, layout)
    table = rot.rotary_table(80, D, device=DEV)
    want = gradients(rot, leaves, positions, grads, table)
    # The rows' gradients are formed row by row: the same to the bit.  The weights' are sums over rows, whose order goes by the layout: one rounding to the type each, and
    # at most a rounding of 32 bits per row against the size of what is added up (a turned gradient is at most the sum of its pair's).
    size = []
    for x, dy in zip(leaves[:2], grads):
        x, dy = x.detach().double(), dy.double().abs()
        xhat = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        size.append((((dy + dy.roll(D // 2, -1)) * xhat.abs()).sum((0, 1, 2)), x.shape[0] * x.shape[1] * x.shape[2]))

    def same(got):
        assert all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(got[:2], want[:2]))
        for a, b, (mag, rows) in zip(got[2:], want[2:], size):
            assert bool(((a.double() - b.double()).abs() <= torch.finfo(dtype).eps * 1.01 * b.double().abs() + 2 * (rows + 64) * 2.0 ** -24 * mag).all())

    for _ in range(2):
        with torch.autograd.graph.save_on_cpu() if hook == "cpu" else torch.autograd.graph.saved_tensors_hooks(HOOKS[hook], lambda t: t):
            got = gradients(rot, leaves, positions, grads, table)
        same(got)
        same(gradients(rot, leaves, positions, grads, table))             # (and nothing of the other layout is kept)


def test_saved_tensors_on_another_device_are_refused(rot):
    leaves, positions, grads = operands(torch.float16, 64, "fused")
    table = rot.rotary_table(80, 64, device=DEV)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        out = rot.qk_norm_rope(*leaves, table, positions)
    with pytest.raises((ValueError, TypeError)):
        torch.autograd.grad(out, leaves, grads)
