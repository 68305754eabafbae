"""GPU tests: traced calls of the cache and rotation operators run as the eager ones do, and tensors that a call changes say so."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def kv():
    import flash_attention_amd.kv_cache as kv

    return kv


@pytest.fixture(scope="module")
def rot():
    import flash_attention_amd.rotary as rot

    return rot


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


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


class Log(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name)
        return func(*args, **(kwargs or {}))


def test_the_backward_is_dispatched(rot):
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


def test_a_backward_alone_is_dispatched(rot):
    """the mode is entered behind the forward"""
    g = torch.Generator().manual_seed(2)
    leaves = [torch.randn(2, h, 10, 64, generator=g).half().to(DEV).requires_grad_() for h in (4, 2)] + [torch.ones(64, device=DEV).half().requires_grad_()]
    table = rot.rotary_table(20, 64, device=DEV)
    for weights, wanted in (((leaves[2], None), leaves), ((None, leaves[2]), leaves), ((leaves[2], leaves[2].detach()), leaves), ((None, None), leaves[:2]), ((leaves[2].detach(), None), leaves[:1])):
        out = rot.qk_norm_rope(*leaves[:2], *weights, table)
        grads = [torch.randn(t.shape, generator=g).half().to(DEV) for t in out]
        want = torch.autograd.grad(out, wanted, grads, retain_graph=True)
        with Log() as log:
            got = torch.autograd.grad(out, wanted, grads)
        assert [n for n in log.names if n.startswith("flash")] == ["flash_attention_amd::qk_norm_rope_bwd"] and all(torch.equal(a, b) for a, b in zip(got, want))


def test_changed_tensors_say_so(kv):
    """version counters: a tensor that a call writes and a graph has saved is noticed"""
    cache = kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=16)
    layer = cache._layer[0]
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16, device=DEV), torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    state = (cache.block_tables, cache.free_blocks, cache.seq_lens, cache.free_count)
    before = [t._version for t in state]
    step = cache.step(ints([2, 1]), 3)
    assert all(t._version > n for t, n in zip(state, before))
    before = [t._version for t in state]
    kv.cache_tables(cache.seq_lens, ints([0, 0]), cache.block_tables, cache.free_blocks, cache.free_count, 3, 16)
    assert [t._version > n for t, n in zip(state, before)] == [True, True, False, False]
    before = [t._version for t in layer]
    cache.append(0, k, k, step)
    assert all(t._version > n for t, n in zip(layer, before)) and cache.k_cache._version == layer[0]._version
    out = torch.empty_like(q)
    before, read = out._version, [t._version for t in (q, *layer, cache.block_tables)]
    kv.flash_attention_cached(q, *layer, cache.block_tables, step.seq_lens, step.cu_new, out=out)
    assert out._version > before and [t._version for t in (q, *layer, cache.block_tables)] == read
    rows, table = torch.arange(2, device=DEV), torch.ones(65, 4, device=DEV, requires_grad=True)
    picked = table[cache.seq_lens.clamp_(max=64)] * table[rows]
    cache.step(ints([1, 1]), 2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        picked.sum().backward()


def test_calls_in_inference_mode(kv, rot):
    """tensors without version counters"""
    with torch.inference_mode():
        cache = kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=16)
        q, k, v = (torch.randn(3, h, 64, device=DEV).half() for h in (4, 2, 2))
        step = cache.step(ints([2, 1]), 3)
        q, k = rot.qk_norm_rope(q, k, None, None, rot.rotary_table(64, 64, device=DEV), step.positions)
        out = cache.attend(0, q, k, v, step, out=torch.empty_like(q))
    assert bool(torch.isfinite(out).all()) and cache.seq_lens.tolist() == [2, 1]
