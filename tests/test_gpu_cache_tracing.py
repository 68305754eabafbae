"""GPU tests: traced calls of the cache and rotation operators run as the eager ones do, and tensors that a call changes say so."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_traced_step_runs(kv, rot):
    """the graph that a tracer records of a step does what the step does"""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(6, h, 64, generator=g).half().to(DEV) for h in (4, 2, 2))
    table, new = rot.rotary_table(128, 64, device=DEV), ints([4, 2])
    a, b, c = (kv.KVCache(1, 16, 2, 64, requests=2, max_tokens=128) for _ in range(3))

    def one(cache, new, q, k, v):
        step = cache.step(new, 6)
        q, k = rot.qk_norm_rope(q, k, None, None, table, step.positions)
        return cache.attend(0, q, k, v, step, max_q_len=4)

    want = one(a, new, q, k, v)
    graph = make_fx(lambda *args: one(b, *args))(new, q, k, v)            # (tracing runs the step once)
    assert b.seq_lens.tolist() == [4, 2]
    for t, s in ((b.seq_lens, c.seq_lens), (b.free_count, c.free_count), (b.free_blocks, c.free_blocks)):
        t.copy_(s)
    got = graph(new, q, k, v)
    assert torch.equal(got, want) and torch.equal(a.seq_lens, b.seq_lens) and torch.equal(a.block_tables, b.block_tables)


def test_the_backward_is_dispatched(rot):
    class Log(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func._schema.name)
            return func(*args, **(kwargs or {}))

    g = torch.Generator().manual_seed(1)
    leaves = [torch.randn(2, h, 10, 64, generator=g).half().to(DEV).requires_grad_() for h in (4, 2)] + [torch.ones(64, device=DEV).half().requires_grad_()]
    table = rot.rotary_table(20, 64, device=DEV)
    grads = [torch.randn(t.shape, generator=g).half().to(DEV) for t in leaves[:2]]
    run = lambda: torch.autograd.grad(rot.qk_norm_rope(*leaves, None, table), leaves, grads)  # noqa: E731
    want = run()
    with Log() as log:
        got = run()
    assert [n for n in log.names if n.startswith("flash")] == ["flash_attention_amd::qk_norm_rope", "flash_attention_amd::qk_norm_rope_bwd"]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
