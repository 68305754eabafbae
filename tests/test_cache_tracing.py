"""CPU tests: the cache and rotation operators under dispatch modes, tracers and forward-mode levels (fake GPU tensors; no kernel runs)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

import flash_attention_amd.kv_cache as kv
import flash_attention_amd.rotary as rot


class Log(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name)
        return func(*args, **(kwargs or {}))


def half(*shape, **kw):
    return torch.empty(*shape, device="cuda", dtype=torch.float16, **kw)


def step_of_a_layer(cache, new, q, k, v, table):
    step = cache.step(new, q.shape[0])
    q, k = rot.qk_norm_rope(q, k, None, None, table, step.positions)
    return cache.attend(0, q, k, v, step)


def inputs():
    cache = kv.KVCache(1, 8, 2, 64, requests=2, max_tokens=64, block_size=16)
    return cache, torch.empty(2, device="cuda", dtype=torch.int32), half(5, 4, 64), half(5, 2, 64), half(5, 2, 64), torch.empty(64, 64, device="cuda")


OPS = ["flash_attention_amd::cache_tables", "flash_attention_amd::qk_norm_rope", "flash_attention_amd::cache_append", "flash_attention_amd::cached"]


def test_a_dispatch_mode_sees_the_operators():
    with FakeTensorMode():
        args = inputs()
        with Log() as log:
            out = step_of_a_layer(*args)
    assert out.shape == (5, 4, 64) and [n for n in log.names if n.startswith("flash_attention_amd")] == OPS


def test_a_tracer_sees_the_operators():
    with FakeTensorMode():
        cache, *args = inputs()
        graph = make_fx(lambda *a: step_of_a_layer(cache, *a))(*args)
    assert [n.target.name().rsplit(".", 1)[0] for n in graph.graph.nodes if "flash_attention_amd" in str(n.target)] == OPS


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


def test_gradients_that_nothing_forms_are_refused():
    x, ints, ones = torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32), torch.ones(4, 2)
    codes = [torch.zeros(4, 2, *s, dtype=torch.uint8).view(torch.float8_e4m3fn) for s in ((16, 64), (64, 16))]
    wants = ones.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        kv.cache_append(x, x, ints, *codes, wants, ones)
    for kw in (dict(k_scale=wants), dict(v_scale=wants), dict(out=x.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no gradient"):
            kv.flash_attention_cached(**{**dict(q=x, k_cache=codes[0], v_cache=codes[1], k_scale=ones, v_scale=ones, block_tables=torch.zeros(1, 1, dtype=torch.int32),
                                                seq_lens=ints[:1], cu_q=ints[:2]), **kw})


def test_a_table_that_wants_a_gradient_is_refused():
    """eager, under a dispatch mode and compiled alike"""
    table = torch.zeros(8, 64, requires_grad=True)
    x = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="no gradient for the table"):
        rot.qk_norm_rope(x, x, None, None, table)
    with FakeTensorMode():
        q, table = half(4, 2, 64), torch.empty(8, 64, device="cuda", requires_grad=True)
        with pytest.raises(ValueError, match="no gradient for the table"):
            rot.qk_norm_rope(q, q, None, None, table)
        with torch.no_grad():
            rot.qk_norm_rope(q, q, None, None, table)
    compiled = torch.compile(lambda t: rot.qk_norm_rope(x, x, None, None, t), backend="eager")
    with pytest.raises(Exception, match="no gradient for the table"):
        compiled(torch.zeros(8, 64, requires_grad=True))


@pytest.mark.parametrize("tokens,told,used", [(5, None, 1), (8, None, 1), (12, None, 5), (500, None, 493), (500, 1, 1), (5, 5, 5)])
def test_the_hint_that_a_call_goes_by(tokens, told, used):
    """the documented guess, T - B + 1, and what the caller says in its place"""
    class Hint(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func._schema.name == "flash_attention_amd::cached":
                seen.append(args[9])
            return func(*args, **(kwargs or {}))

    seen = []
    with FakeTensorMode():
        cache = kv.KVCache(1, 64, 2, 64, requests=8, max_tokens=600, block_size=16)
        step = cache.step(torch.empty(8, device="cuda", dtype=torch.int32), tokens)
        with Hint():
            cache.attend(0, half(tokens, 4, 64), half(tokens, 2, 64), half(tokens, 2, 64), step, max_q_len=told)
    assert seen == [used]
