"""GPT-2-shaped decoder written fresh for the demos, the tests and bench.py's config-4 leg.

The reference's demo trains nanoGPT (demo/train.py:139-321) from a git submodule that is an EMPTY directory in the
reference tree, so there is no model code to follow; this is the standard pre-LN GPT-2 block at the GPT-2-small
shape (12 layers, 12 heads, n_embd 768) whose attention goes through `F.scaled_dot_product_attention(q, k, v,
is_causal=True)` on [B, H, T, hs] views of the fused [B, T, 3C] projection - exactly the call the automatic
override (`import flash_attention_amd.auto`) replaces, as in the reference's demo notebook (nb cell 5).

`TinyGPT(rotary=True)` is the same decoder as models of today have its attention: query and key heads normed and rotated by their positions
(`qk_norm_rope`) in place of learned positions, fewer key/value heads on request, and `generate()` over an 8-bit block cache (`KVCache`).  It needs the GPU."""

import torch
import torch.nn as nn
import torch.nn.functional as F

try:
    from flash_attention_amd.kv_cache import KVCache
    from flash_attention_amd.rotary import qk_norm_rope, rotary_table
except ModuleNotFoundError as e:        # (the plain model needs torch alone)
    if e.name != "flash_attention_amd":
        raise
    KVCache = qk_norm_rope = rotary_table = None


class CausalSelfAttention(nn.Module):
    def __init__(self, n_embd, n_head, dropout=0.0, n_kv_head=None, rotary=False):
        super().__init__()
        n_kv_head = n_head if n_kv_head is None else n_kv_head
        if n_kv_head != n_head and not rotary:
            raise ValueError("n_kv_head needs rotary=True")
        if rotary and qk_norm_rope is None:
            raise ModuleNotFoundError("rotary=True needs flash_attention_amd on the path", name="flash_attention_amd")
        self.n_head, self.n_kv_head, self.n_embd, self.dropout, self.rotary = n_head, n_kv_head, n_embd, dropout, rotary
        self.c_attn = nn.Linear(n_embd, (n_head + 2 * n_kv_head) * (n_embd // n_head))
        self.c_proj = nn.Linear(n_embd, n_embd)
        self.resid_dropout = nn.Dropout(dropout)
        if rotary:
            self.q_weight, self.k_weight = (nn.Parameter(torch.ones(n_embd // n_head)) for _ in range(2))

    def heads(self, x):
        """[..., heads, head dim] views of the fused projection: q, k, v"""
        return self.c_attn(x).unflatten(-1, (-1, self.n_embd // self.n_head)).split((self.n_head, self.n_kv_head, self.n_kv_head), dim=-2)

    def forward(self, x, table=None):
        B, T, C = x.shape
        if self.rotary:
            q, k, v = (t.transpose(1, 2) for t in self.heads(x))
            q, k = qk_norm_rope(q, k, self.q_weight, self.k_weight, table)
        else:
            q, k, v = self.c_attn(x).split(self.n_embd, dim=2)
            q, k, v = (t.view(B, T, self.n_head, C // self.n_head).transpose(1, 2) for t in (q, k, v))
        # (nanoGPT's call: attention dropout while training - the reference's override raises for it, sdpa.py:25-28; this one serves it)
        gqa = {"enable_gqa": True} if self.n_kv_head != self.n_head else {}
        y = F.scaled_dot_product_attention(q, k, v, attn_mask=None, dropout_p=self.dropout if self.training else 0.0, is_causal=True, **gqa)
        return self.resid_dropout(self.c_proj(y.transpose(1, 2).contiguous().view(B, T, C)))

    def cached(self, x, table, cache, layer, step, max_q_len):
        """packed tokens [T, C] of a step: keys and values into the cache, attention over it"""
        q, k, v = self.heads(x)
        q, k = qk_norm_rope(q, k, self.q_weight, self.k_weight, table, step.positions)
        return self.c_proj(cache.attend(layer, q, k, v, step, max_q_len=max_q_len).flatten(1))


class Block(nn.Module):
    def __init__(self, n_embd, n_head, dropout=0.0, n_kv_head=None, rotary=False):
        super().__init__()
        self.ln_1, self.ln_2 = nn.LayerNorm(n_embd), nn.LayerNorm(n_embd)
        self.attn = CausalSelfAttention(n_embd, n_head, dropout, n_kv_head, rotary)
        self.mlp = nn.Sequential(nn.Linear(n_embd, 4 * n_embd), nn.GELU(), nn.Linear(4 * n_embd, n_embd), nn.Dropout(dropout))

    def forward(self, x, table=None):
        x = x + self.attn(self.ln_1(x), table)
        return x + self.mlp(self.ln_2(x))

    def cached(self, x, *state):
        x = x + self.attn.cached(self.ln_1(x), *state)
        return x + self.mlp(self.ln_2(x))


class TinyGPT(nn.Module):
    def __init__(self, vocab=50304, block=1024, n_layer=12, n_head=12, n_embd=768, dropout=0.0, n_kv_head=None, rotary=False):
        super().__init__()
        self.block, self.head_dim, self.rotary, self._table = block, n_embd // n_head, rotary, None
        self.wte, self.wpe = nn.Embedding(vocab, n_embd), None if rotary else nn.Embedding(block, n_embd)
        self.drop = nn.Dropout(dropout)
        self.h = nn.ModuleList(Block(n_embd, n_head, dropout, n_kv_head, rotary) for _ in range(n_layer))
        self.ln_f = nn.LayerNorm(n_embd)
        self.lm_head = nn.Linear(n_embd, vocab, bias=False)

    def table(self, device):
        """cosines and sines of the block's positions: 32-bit whatever the model's type, and no parameter"""
        if self._table is None or self._table.device != device:
            with torch.inference_mode(False):           # (one that an evaluation makes has to serve training too)
                self._table = rotary_table(self.block, self.head_dim, device=device)
        return self._table

    def forward(self, idx):
        if self.rotary:
            table = self.table(idx.device)
            x = self.drop(self.wte(idx))
        else:
            table = None
            x = self.drop(self.wte(idx) + self.wpe(torch.arange(idx.shape[1], device=idx.device)))
        for blk in self.h:
            x = blk(x, table)
        return self.lm_head(self.ln_f(x))

    @torch.no_grad()
    def generate(self, prompts, new_tokens, block_size=64):
        """Greedy continuations of prompts of different lengths (1-D tensors of tokens, each of one at least): int64 [prompts, new_tokens].  One step takes the
        prompts, packed; every other one token of each.  Queries have to be 16-bit: run it under autocast or with a model of 16 bits."""
        lens = [p.numel() for p in prompts]
        if not self.rotary or self.training:
            raise ValueError("generate() needs TinyGPT(rotary=True) in eval mode")
        if not lens or min(lens) < 1 or new_tokens < 1 or max(lens) + new_tokens > self.block:
            raise ValueError("generate() needs prompts of 1 token and more that end inside the block with their continuations")
        dev, attn = self.wte.weight.device, self.h[0].attn
        cache = KVCache(len(self.h), sum((n + new_tokens + block_size - 1) // block_size for n in lens), attn.n_kv_head, self.head_dim, requests=len(lens),
                        max_tokens=max(lens) + new_tokens, block_size=block_size, device=dev)
        table, idx, new, longest, out = self.table(dev), torch.cat([p.to(dev) for p in prompts]), torch.tensor(lens, dtype=torch.int32, device=dev), max(lens), []
        for _ in range(new_tokens):
            step = cache.step(new, idx.numel())
            x = self.wte(idx)
            for layer, blk in enumerate(self.h):
                x = blk.cached(x, table, cache, layer, step, longest)
            idx = self.lm_head(self.ln_f(x[step.cu_new[1:].long() - 1])).argmax(-1)
            out.append(idx)
            new, longest = torch.ones_like(new), 1
        return torch.stack(out, 1)


def gpt2_init_(model: nn.Module, std: float = 0.02) -> nn.Module:
    """GPT-2 style init: keeps activations O(1) through 12 layers."""
    for p in model.parameters():
        if p.dim() > 1:
            nn.init.normal_(p, std=std)
    return model
