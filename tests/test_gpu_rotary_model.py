"""The decoder of demo/model.py with normed and rotated heads: its gradients against the plain formula, and its steps over the 8-bit cache against its own
forward pass."""

import pathlib
import sys

import pytest
import torch
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "demo"))
import model as demo_model  # noqa: E402
from model import TinyGPT, gpt2_init_  # noqa: E402

pytestmark = pytest.mark.gpu


def plain_norm_rope(q, k, q_weight, k_weight, table, positions=None, eps=1e-6):
    half = table.shape[1] // 2
    c, s = table[: q.shape[2], :half], table[: q.shape[2], half:]

    def one(x, w):
        y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
        a, b = y[..., :half], y[..., half:]
        return torch.cat((a * c - b * s, a * s + b * c), -1)

    return one(q, q_weight), one(k, k_weight)


def attention(q, k, v, attn_mask=None, dropout_p=0.0, is_causal=False, enable_gqa=False):
    """causal attention written out in 32 bits, whatever serves the call elsewhere (an override that another test installed takes some lengths only)"""
    assert q.dtype == torch.float32 and is_causal
    k, v = (t.repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v))
    s = (q @ k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    return s.masked_fill(torch.ones(s.shape[-2:], device=s.device, dtype=torch.bool).triu(1), float("-inf")).softmax(-1) @ v


@pytest.mark.parametrize("n_kv_head", [4, 2, 1])
def test_gradients_of_a_step(n_kv_head, monkeypatch):
    torch.manual_seed(3)
    net = gpt2_init_(TinyGPT(vocab=97, block=80, n_layer=2, n_head=4, n_embd=128, n_kv_head=n_kv_head, rotary=True)).cuda()
    with torch.no_grad():
        for blk in net.h:
            blk.attn.q_weight.uniform_(0.5, 1.5)
            blk.attn.k_weight.uniform_(0.5, 1.5)
    idx, tgt = (torch.randint(0, 97, (3, 77), device="cuda") for _ in range(2))

    def step():
        net.zero_grad(set_to_none=True)
        loss = F.cross_entropy(net(idx).view(-1, 97), tgt.view(-1))
        loss.backward()
        return loss.item(), {n: p.grad.clone() for n, p in net.named_parameters()}

    monkeypatch.setattr(F, "scaled_dot_product_attention", attention)
    loss, grads = step()
    monkeypatch.setattr(demo_model, "qk_norm_rope", plain_norm_rope)
    loss_plain, plain = step()
    # both passes round 32-bit values: 2^-24 each, some hundred of them in a row at most, and they add up at random: 2^-14 leaves a factor of ten
    assert abs(loss - loss_plain) <= 2 ** -14 * abs(loss_plain)
    for n, g in grads.items():
        assert (g - plain[n]).norm().item() <= 2 ** -14 * plain[n].norm().item() + 1e-9, n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n_kv_head,block_size", [(4, 64), (1, 16)])
def test_steps_over_the_cache(n_kv_head, block_size, dtype, monkeypatch):
    monkeypatch.setattr(F, "scaled_dot_product_attention", attention)
    torch.manual_seed(4)
    net = gpt2_init_(TinyGPT(vocab=97, block=160, n_layer=2, n_head=4, n_embd=256, n_kv_head=n_kv_head, rotary=True), std=0.05).cuda().eval()
    lens = [1, 70, 128, 33]
    prompts = [torch.randint(0, 97, (n,), device="cuda") for n in lens]
    logits = []
    hook = net.lm_head.register_forward_hook(lambda m, a, y: logits.append(y.float()))
    with torch.autocast("cuda", dtype=dtype):
        got = net.generate(prompts, 6, block_size)
        again = net.generate(prompts, 6, block_size)
    hook.remove()
    assert got.shape == (4, 6) and got.dtype == torch.int64 and torch.equal(got, again)
    for b, n in enumerate(lens):
        whole = torch.cat((prompts[b], got[b]))
        with torch.no_grad():
            want = net(whole[None, :-1])[0, n - 1:]
        here = torch.stack([logits[i][b] for i in range(6)])
        # a code is off by 2^-4 of its value at most and keys and values are codes: twice 2^-4 of the logits bounds it by far, another position does not stay inside
        assert (here - want).norm().item() <= 2 ** -3 * want.norm().item(), b


def test_refusals():
    net = TinyGPT(vocab=97, block=64, n_layer=1, n_head=4, n_embd=64, rotary=True).cuda().eval()
    one = torch.zeros(1, dtype=torch.int64)
    for prompts, new in (([], 1), ([one[:0]], 1), ([one], 0), ([one.repeat(60)], 5)):
        with pytest.raises(ValueError, match="prompts of 1 token"):
            net.generate(prompts, new)
    with pytest.raises(ValueError, match="eval mode"):
        net.train().generate([one], 1)
    with pytest.raises(ValueError, match="rotary=True"):
        TinyGPT(vocab=97, block=64, n_layer=1, n_head=4, n_embd=64).eval().generate([one], 1)
    with pytest.raises(ValueError, match="n_kv_head needs"):
        TinyGPT(vocab=97, block=64, n_layer=1, n_head=4, n_embd=64, n_kv_head=2)
