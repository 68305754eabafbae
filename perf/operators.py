"""What is measured of the operators around attention over an 8-bit key/value cache: listed and drawn cases, their inputs, their
plain forms and their values in 64 bits.

  rope    norm of every query and key head with the position rotation, forward alone or with its backward
  tables  block tables, positions and slots of a step from the requests' lengths
  append  new keys and values into the cache: e4m3 codes with one power-of-two scale per block of tokens and head
  attend  causal attention of ragged query runs over that cache

`own` selects the calls of this package; otherwise elementary torch operations in 32 bits (64 for index sums and long sums), rounded once.
Cache layout: k_cache [blocks, kv heads, block size, width], v_cache [blocks, kv heads, width, block size] in float8_e4m3fn, width the head
dim rounded up to a multiple of 64; k_scale, v_scale [blocks, kv heads] float32; value = code * scale."""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
E4M3_MAX = 448.0
MIN_EXPONENT = -100        # the smallest scale is 2 ** MIN_EXPONENT


def _package():
    import os
    import sys

    path = os.path.join(os.getcwd(), "flash-attention-ipu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_attention_amd.kv_cache as kv_cache
    import flash_attention_amd.rotary as rotary

    return kv_cache, rotary


# ---- cases -----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of 64 requests: every launch is a few microseconds
        {"name": "rope_step", "op": "rope", "train": False, "layout": "thd", "batch": 1, "length": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "dtype": "bf16"},
        # a prompt batch of odd length in 32 bits, half of the head rotated, neighbours paired
        {"name": "rope_prompt_f32", "op": "rope", "train": False, "layout": "bhld", "batch": 3, "length": 4001, "heads": 16, "kv_heads": 4, "dim": 64,
         "rotary": 32, "interleaved": True, "dtype": "f32"},
        # GPT-2 small's attention call in training: batch 8, 12 heads of 64, 1024 positions, heads inside the row
        {"name": "rope_train_small", "op": "rope", "train": True, "layout": "bhld_inner", "batch": 8, "length": 1024, "heads": 12, "kv_heads": 12, "dim": 64,
         "rotary": 64, "interleaved": False, "dtype": "f16"},
        # grouped-query training at 4096 positions, head dim 128
        {"name": "rope_train_large", "op": "rope", "train": True, "layout": "bhld", "batch": 4, "length": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "dtype": "bf16"},
        # a decoding step: 64 requests get a token each
        {"name": "tables_step", "op": "tables", "requests": 64, "max_cached": 8192, "max_new": 1, "idle": 0, "block": 64},
        # a step that takes in many prompts beside running requests and requests that end
        {"name": "tables_prompts", "op": "tables", "requests": 512, "max_cached": 4096, "max_new": 257, "idle": 16, "block": 16},
        # a decoding step's keys and values
        {"name": "append_step", "op": "append", "requests": 64, "max_cached": 8192, "max_new": 1, "kv_heads": 8, "dim": 128, "block": 64, "dtype": "bf16"},
        # prompts of uneven length behind what their requests hold already
        {"name": "append_prompts", "op": "append", "requests": 24, "max_cached": 1000, "max_new": 2048, "kv_heads": 8, "dim": 128, "block": 64, "dtype": "f16"},
        # one request, short cache, 12 heads of 64: the smallest attention call of a generation loop
        {"name": "attend_one", "op": "attend", "requests": 1, "max_cached": 1000, "max_new": 1, "heads": 12, "kv_heads": 12, "dim": 64, "block": 16, "dtype": "f16"},
        # 64 requests of uneven length, grouped heads
        {"name": "attend_batch", "op": "attend", "requests": 64, "max_cached": 8192, "max_new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "dtype": "bf16"},
        # few requests with long caches: the long axis has to be split
        {"name": "attend_long", "op": "attend", "requests": 3, "max_cached": 131072, "max_new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "block": 128, "dtype": "bf16"},
        # prompts taken in by pieces of up to 2048 tokens: products of matrices
        {"name": "attend_prompts", "op": "attend", "requests": 4, "max_cached": 8192, "max_new": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "rope", "tables", "append", "append", "attend", "attend", "attend", "attend"])
    kv_heads, group = rng.choice([1, 2, 4, 8, 12, 5]), rng.choice([1, 2, 4, 8, 3])
    if op == "rope":
        dim = rng.choice([64, 128, 96, 80, 256, 32])
        rotary = rng.choice([dim, dim, dim // 2])
        train = rng.random() < 0.5
        batch, length = _log_int(rng, 1, 8), _log_int(rng, 1, 4096)
        room = 4 * 4096 * 40 * 128
        while batch * length * kv_heads * (group + 1) * dim > room // 2:
            length = max(1, length // 2)
        return {"op": op, "train": train, "layout": rng.choice(["thd", "bhld", "bhld_inner"]), "batch": batch, "length": length, "heads": kv_heads * group,
                "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": rng.random() < 0.3, "dtype": rng.choice(["bf16", "f16", "f32"])}
    block = rng.choice([16, 32, 64, 128])
    if op == "tables":
        return {"op": op, "requests": _log_int(rng, 1, 512), "max_cached": _log_int(rng, 1, 8192), "max_new": rng.choice([1, 1, 5, 64, 257]),
                "idle": rng.choice([0, 3, 16]), "block": block}
    dim = rng.choice([64, 128, 128, 256, 80, 192])
    dtype = rng.choice(["bf16", "f16"])
    if op == "append":
        return {"op": op, "requests": _log_int(rng, 1, 64), "max_cached": _log_int(rng, 1, 4000), "max_new": rng.choice([1, 1, 7, 300]), "kv_heads": min(kv_heads, 8),
                "dim": dim, "block": block, "dtype": dtype}
    requests, new = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, _log_int(rng, 5, 700)])
    cached = _log_int(rng, 1, 32768)
    while requests * cached * kv_heads * dim > 64 * 4096 * 8 * 128 // 2 or requests * (cached + new) * new * kv_heads * group > 4 * 4096 * 1024 * 32:
        cached, requests = max(1, cached * 3 // 4), max(1, requests * 3 // 4)
        new = max(1, new * 3 // 4)
    return {"op": op, "requests": requests, "max_cached": cached, "max_new": new, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "block": block, "dtype": dtype}


# ---- lengths of a case: plain numbers, the same for every seed, so that a case's work is one number ---------------------------------
def _lengths(case):
    """(tokens held before, tokens that come) of every request, as numpy integers; some requests hold nothing, some get nothing"""
    r = np.random.RandomState(1234 + case["requests"] * 7 + case["max_cached"])
    n = case["requests"]
    held = np.floor(case["max_cached"] * r.uniform(0.1, 1.0, n)).astype(np.int64)
    new = np.maximum(1, np.floor(case["max_new"] * r.uniform(0.1, 1.0, n)).astype(np.int64)) if case["max_new"] > 1 else np.ones(n, np.int64)
    held[0], new[0] = case["max_cached"], case["max_new"]
    if n >= 8 and case["max_new"] > 1:
        held[n // 2] = 0
        if case["op"] != "attend":
            new[n // 3] = 0
    for k in range(case.get("idle", 0)):
        if 2 * k + 1 < n:
            new[2 * k + 1] = -1           # (a request that ends: its blocks go back to the pool)
    return held, new


def _blocks(tokens, block):
    return -(-tokens // block)


def _width(dim):
    return -(-dim // 64) * 64


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = _generator(seed)
    return {"rope": _prepare_rope, "tables": _prepare_tables, "append": _prepare_append, "attend": _prepare_attend}[case["op"]](case, g)


def _prepare_rope(case, g):
    B, L, D, dt = case["batch"], case["length"], case["dim"], DTYPES[case["dtype"]]

    def operand(heads):
        if case["layout"] == "thd":
            return _randn((B * L, heads, D), g, dt)
        if case["layout"] == "bhld_inner":
            return _randn((B, L, heads, D), g, dt).transpose(1, 2)
        return _randn((B, heads, L, D), g, dt)

    s = {"case": case, "q": operand(case["heads"]), "k": operand(case["kv_heads"]),
         "q_weight": (1 + 0.1 * _randn((D,), g)).to(dt), "k_weight": (1 + 0.1 * _randn((D,), g)).to(dt)}
    top = 2 * L + 64
    # cos and sin of position * 10000 ** (-2 i / rotary), formed in 64 bits and kept in 32, as a model keeps them
    angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -2.0 * torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64) / case["rotary"])
    s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    start = torch.randint(0, L + 64, (B, 1), generator=g, device="cuda", dtype=torch.int32)
    s["positions"] = start + torch.arange(L, device="cuda", dtype=torch.int32)
    if case["layout"] == "thd":
        s["positions"] = s["positions"].reshape(-1)
    if case["train"]:
        s["dq_out"] = torch.empty_like(s["q"]).copy_(_randn(s["q"].shape, g))
        s["dk_out"] = torch.empty_like(s["k"]).copy_(_randn(s["k"].shape, g))
        for name in ("q", "k", "q_weight", "k_weight"):
            s[name].requires_grad_(True)
    return s


def _pool(case, g, held, extra):
    """block table of the requests (random blocks, unused entries -1), the free blocks behind it and the number of blocks in all"""
    P, n = case["block"], case["requests"]
    per = _blocks(held, P)
    width = int(_blocks(held + np.maximum(0, extra), P).max())
    total = int(per.sum() + _blocks(np.maximum(0, extra), P).sum()) + n + 3
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    at = np.concatenate([[0], np.cumsum(per)])
    column, row = np.meshgrid(np.arange(width), np.arange(n))
    take = torch.from_numpy(np.where(column < per[row], at[row] + column, total)).cuda()
    tables = torch.cat([ids, torch.full((1,), -1, device="cuda", dtype=torch.int32)])[take]
    used = int(per.sum())
    return tables.contiguous(), ids[used:].contiguous(), total


def _prepare_tables(case, g):
    held, new = _lengths(case)
    tables, free, total = _pool(case, g, held, new)
    pool = torch.full((total,), -1, device="cuda", dtype=torch.int32)
    pool[: free.numel()] = free
    ints = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
    return {"case": case, "seq_lens": ints(held), "new_lens": ints(new), "tables": tables, "pool": pool, "free": ints([free.numel()]),
            "tokens": int(np.maximum(0, new).sum()) + 5}           # (a batch padded by some tokens, as captured steps are)


def _codes(shape, g):
    """e4m3 codes as normal keys and values leave them: the largest of a block between half and all of the type's range"""
    out = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        n = min(1 << 28, flat.numel() - at)
        flat[at:at + n] = (100 * _randn((n,), g)).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return out


def _cache(case, g, total):
    H, P, W = case["kv_heads"], case["block"], _width(case["dim"])
    k, v = _codes((total, H, P, W), g), _codes((total, H, W, P), g)
    if W != case["dim"]:
        k[..., case["dim"]:] = 0
        v[:, :, case["dim"]:] = 0
    scale = lambda: torch.exp2(torch.randint(-8, -5, (total, H), generator=g, device="cuda").float())  # noqa: E731
    return {"k_cache": k, "v_cache": v, "k_scale": scale(), "v_scale": scale()}


def _prepare_append(case, g):
    held, new = _lengths(case)
    tables, _, total = _pool(case, g, held + np.maximum(0, new), np.zeros_like(new))
    s = {"case": case, **_cache(case, g, total)}
    request = np.repeat(np.arange(len(new)), new)
    position = np.concatenate([held[b] + np.arange(new[b]) for b in range(len(new))])
    position_t = torch.from_numpy(position).cuda()
    slots = tables[torch.from_numpy(request).cuda(), position_t // case["block"]].long() * case["block"] + position_t % case["block"]
    s["slots"] = torch.cat([slots, slots.new_full((3,), -1)]).to(torch.int32)      # (and three tokens of padding)
    s["k"], s["v"] = (_randn((s["slots"].numel(), case["kv_heads"], case["dim"]), g, DTYPES[case["dtype"]]) for _ in "kv")
    return s


def _prepare_attend(case, g):
    held, new = _lengths(case)
    tables, _, total = _pool(case, g, held + new, np.zeros_like(new))
    ints = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
    return {"case": case, **_cache(case, g, total), "tables": tables, "seq_lens": ints(held + new), "cu_q": ints(np.concatenate([[0], np.cumsum(new)])),
            "max_q_len": int(new.max()), "q": _randn((int(new.sum()), case["heads"], case["dim"]), g, DTYPES[case["dtype"]])}


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return {"rope": _own_rope, "tables": _own_tables, "append": _own_append, "attend": _own_attend}[s["case"]["op"]](s)
    return {"rope": _plain_rope, "tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]](s)


def _own_rope(s):
    _, rotary = _package()
    q, k = rotary.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], s["positions"], eps=EPS, interleaved=s["case"]["interleaved"])
    if not s["case"]["train"]:
        return q, k
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["dq_out"], s["dk_out"]))
    return (q.detach(), k.detach(), *grads)


def _own_tables(s):
    kv_cache, _ = _package()
    step = kv_cache.cache_tables(s["seq_lens"], s["new_lens"], s["tables"], s["pool"], s["free"], s["tokens"], s["case"]["block"])
    return step.seq_lens, step.free_count, step.cu_new, step.positions, step.slots, step.granted, s["tables"], s["pool"]


def _own_append(s):
    kv_cache, _ = _package()
    kv_cache.cache_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _own_attend(s):
    kv_cache, _ = _package()
    return kv_cache.flash_attention_cached(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"], s["seq_lens"], s["cu_q"],
                                           max_q_len=s["max_q_len"])


# ---- plain forms -----------------------------------------------------------------------------------------------------------------
def _cos_sin(s):
    """cos and sin of every position's rotation, the same for all heads"""
    rows = s["table"][s["positions"].long()][:, None]
    half = s["case"]["rotary"] // 2
    return rows[..., :half], rows[..., half:]


def _split(s, x):
    """the two halves of the rotated pairs and the columns behind them"""
    R = s["case"]["rotary"]
    if s["case"]["interleaved"]:
        return x[..., 0:R:2], x[..., 1:R:2], x[..., R:]
    return x[..., : R // 2], x[..., R // 2: R], x[..., R:]


def _join(s, a, b, rest):
    if s["case"]["interleaved"]:
        return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)
    return torch.cat([a, b, rest], -1)


def _plain_rope_forward(s, x, w):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    c, sn = _cos_sin(s)
    a, b, rest = _split(s, y)
    return _join(s, a * c - b * sn, a * sn + b * c, rest)


def _plain_rope_backward(s, x, w, dout):
    x, w, dout = x.float(), w.float(), dout.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    c, sn = _cos_sin(s)
    a, b, rest = _split(s, dout)
    dy = _join(s, a * c + b * sn, b * c - a * sn, rest)          # the rotation turned back
    xhat = x * r
    dw = (dy * xhat).double().sum(tuple(range(x.ndim - 1)))
    dx = dy * w
    return r * (dx - xhat * (dx * xhat).mean(-1, keepdim=True)), dw


def _plain_rope(s):
    with torch.no_grad():
        dt = s["q"].dtype
        out = [_plain_rope_forward(s, s[x], s[x + "_weight"]).to(dt) for x in "qk"]
        if not s["case"]["train"]:
            return tuple(out)
        grads = [_plain_rope_backward(s, s[x], s[x + "_weight"], s["d%s_out" % x]) for x in "qk"]
        return (*out, grads[0][0].to(dt), grads[1][0].to(dt), grads[0][1].to(dt), grads[1][1].to(dt))


def _plain_tables(s):
    P, tables, pool = s["case"]["block"], s["tables"], s["pool"]
    width, tokens = tables.shape[1], s["tokens"]
    held, new = s["seq_lens"].long(), s["new_lens"].long()
    ends = new < 0
    count = new.clamp(min=0)
    cu = torch.cat([count.new_zeros(1), count.cumsum(0)])
    have = (held + P - 1) // P
    # blocks of the requests that end go back to the pool, behind the free ones
    back = torch.where(ends, have, 0)
    back_at = back.cumsum(0) - back
    free = s["free"].long()
    column = torch.arange(width, device="cuda")
    spare = pool.numel()
    returned = ends[:, None] & (column < have[:, None])
    at = torch.where(returned, free + back_at[:, None] + column, spare).clamp(max=spare)
    wide = torch.cat([pool, pool.new_zeros(1)])
    wide[at.reshape(-1)] = torch.where(returned, tables, 0).reshape(-1)
    pool.copy_(wide[:spare])
    free = free + back.sum()
    # a request is served if its tokens fit the batch and the table and the blocks of all before it and its own are there
    need = (held + count + P - 1) // P - have
    fits = ((held + count + P - 1) // P <= width) & (cu[1:] <= tokens)
    need = torch.where(ends | ~fits, 0, need)
    upto = need.cumsum(0)
    served = ~ends & fits & ((need == 0) | (upto <= free))
    first = upto - need
    fresh = served[:, None] & (column >= have[:, None]) & (column < (have + need)[:, None])
    taken = free - 1 - (first - have)[:, None] - column
    tables.copy_(torch.where(fresh, pool[taken.clamp(0, spare - 1)], tables))
    granted = torch.where(served, count, 0)
    total = torch.where(ends, 0, held + granted)
    free = free - torch.where(served, need, 0).sum()
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=held.numel() - 1)
    position = held[b] + t - cu[b]
    live = (t < cu[-1]) & (granted[b] > 0)
    slot = tables[b, (position // P).clamp(0, width - 1)].long() * P + position % P
    i32 = torch.int32
    return (total.to(i32), free.to(i32), cu.to(i32), torch.where(live, position, -1).to(i32), torch.where(live, slot, -1).to(i32), granted.to(i32), tables, pool)


def _exponent(largest):
    """smallest e with largest <= 448 * 2 ** e, not below MIN_EXPONENT"""
    mantissa, e = torch.frexp(largest)                  # largest = mantissa * 2 ** e, 0.5 <= mantissa < 1;  448 = 0.875 * 2 ** 9
    e = e - 9 + (mantissa > 0.875)
    return torch.where(largest > 0, e, MIN_EXPONENT).clamp(min=MIN_EXPONENT)


def _plain_append_one(x, slots, cache, scale, P, by_token):
    """one of the two caches; by_token: [blocks, heads, P, width], else [blocks, heads, width, P]"""
    H, D = x.shape[1], x.shape[2]
    touched, place = torch.unique(slots // P, return_inverse=True)                        # the blocks that get tokens
    offset = slots % P
    codes = cache.view(torch.uint8)[touched].view(torch.float8_e4m3fn).float()
    codes = codes if by_token else codes.transpose(2, 3)
    new = torch.zeros_like(codes)
    new[place, :, offset, :D] = x.float()
    written = torch.zeros(touched.numel(), P, device="cuda", dtype=torch.bool)
    written[place, offset] = True
    fresh, old = written[:, :1], scale[touched]
    wanted = torch.exp2(_exponent(new.abs().amax((2, 3))).float())
    grown = torch.where(fresh, wanted, torch.maximum(wanted, old))
    factor = torch.where(fresh, 1.0, old / grown)
    codes = torch.where(written[:, None, :, None], new / grown[:, :, None, None], codes * factor[:, :, None, None])
    codes = (codes if by_token else codes.transpose(2, 3)).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[touched] = codes.view(torch.uint8)
    scale[touched] = grown


def _plain_append(s):
    P, live = s["case"]["block"], s["slots"] >= 0
    slots = s["slots"][live].long()
    _plain_append_one(s["k"][live], slots, s["k_cache"], s["k_scale"], P, True)
    _plain_append_one(s["v"][live], slots, s["v_cache"], s["v_scale"], P, False)
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _gathered(s, cache, scale, by_token):
    """[requests, kv heads, tokens, dim] of every request's blocks, in 32 bits"""
    at = s["tables"].clamp(min=0).long()
    x = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at][..., None, None]
    x = x if by_token else x.transpose(-1, -2)
    return x.transpose(1, 2).flatten(2, 3)[..., : s["case"]["dim"]]


def _plain_attend(s):
    case, q, cu, lens = s["case"], s["q"], s["cu_q"].long(), s["seq_lens"].long()
    B, H, Hk, D, n = case["requests"], case["heads"], case["kv_heads"], case["dim"], s["max_q_len"]
    i = torch.arange(n, device="cuda")
    count = cu[1:] - cu[:-1]
    rows = q.float()[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)]                      # [B, n, H, D]
    rows = rows.reshape(B, n, Hk, H // Hk, D).transpose(1, 2).reshape(B, Hk, -1, D)
    k, v = _gathered(s, s["k_cache"], s["k_scale"], True), _gathered(s, s["v_cache"], s["v_scale"], False)
    p = torch.matmul(rows * D ** -0.5, k.transpose(-1, -2))                               # [B, Hk, n * group, tokens]
    last = (lens - count)[:, None] + i                                                    # the last key that a row may see
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]                     # [B, n, tokens]
    seen = seen[:, None, :, None].expand(B, Hk, n, H // Hk, -1).reshape(p.shape)
    p = p.masked_fill_(~seen, -math.inf)
    p = torch.exp(p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)))
    v = v.masked_fill(~(torch.arange(k.shape[2], device="cuda") < lens[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_(min=1e-38)
    o = o.reshape(B, Hk, n, H // Hk, D).transpose(1, 2).reshape(B, n, H, D)
    t = torch.arange(q.shape[0], device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=B - 1)
    return o[b, t - cu[b]].to(q.dtype)


# ---- values in 64 bits, written apart from the plain forms -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    return None


def _exact_rope(s):
    """Through complex numbers and autograd: rotation is multiplication by exp(i * angle)."""
    case = s["case"]
    R = case["rotary"]
    turn = torch.complex(s["table"][:, : R // 2].double(), s["table"][:, R // 2:].double())[s["positions"].long()].unsqueeze(1)

    def forward(x, w):
        y = w * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
        if case["interleaved"]:
            z = torch.complex(y[..., :R].unflatten(-1, (R // 2, 2))[..., 0], y[..., :R].unflatten(-1, (R // 2, 2))[..., 1]) * turn
            return torch.cat([torch.view_as_real(z).flatten(-2), y[..., R:]], -1)
        z = torch.complex(y[..., : R // 2], y[..., R // 2: R]) * turn
        return torch.cat([z.real, z.imag, y[..., R:]], -1)

    out, dx, dw = [], [], []
    for name in "qk":
        x, w = (s[n].detach().double().requires_grad_(case["train"]) for n in (name, name + "_weight"))
        y = forward(x, w)
        out.append(y.detach())
        if case["train"]:
            a, b = torch.autograd.grad(y, (x, w), s["d%s_out" % name].double())
            dx.append(a)
            dw.append(b)
    return (*out, *dx, *dw)


def _nearest_e4m3(x):
    """numpy: the nearest e4m3 value (ties to the even code) of |x| <= 448"""
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(x / step) * step


def _exact_append(s):
    P, slots = s["case"]["block"], s["slots"].cpu().numpy()
    live = np.flatnonzero(slots >= 0)
    by_block = {}
    for t in live:
        by_block.setdefault(int(slots[t]) // P, []).append(t)
    if len(by_block) * s["k"].shape[1] > 12000:
        return None
    done = []
    for name, x in (("k", s["k"]), ("v", s["v"])):
        cache, scale, x = s[name + "_cache"].float(), s[name + "_scale"].cpu().numpy().astype(np.float64), x.double().cpu().numpy()
        touched = sorted(by_block)
        at = torch.tensor(touched, device="cuda")
        tiles = cache[at].cpu().numpy().astype(np.float64)
        if name == "v":
            tiles = tiles.transpose(0, 1, 3, 2)
        tiles = tiles.copy()
        for n, block in enumerate(touched):
            ts = by_block[block]
            rows = slots[ts] % P
            largest = np.abs(x[ts]).max((0, 2))
            e = np.ceil(np.log2(np.maximum(largest, 1e-40) / 448.0))
            wanted = np.exp2(np.maximum(e, MIN_EXPONENT))
            new = wanted if rows.min() == 0 else np.maximum(wanted, scale[block])
            if rows.min() != 0:
                tiles[n] = _nearest_e4m3(tiles[n] * (scale[block] / new)[:, None, None])
            tiles[n][:, rows] = 0
            tiles[n][:, rows, : x.shape[2]] = _nearest_e4m3(x[ts].transpose(1, 0, 2) / new[:, None, None])
            scale[block] = new
        cache = cache.double()
        tiles = tiles if name == "k" else np.ascontiguousarray(tiles.transpose(0, 1, 3, 2))
        cache[at] = torch.from_numpy(tiles).cuda()
        done.append((cache, torch.from_numpy(scale).cuda()))
    return done[0][0], done[1][0], done[0][1], done[1][1]


def _exact_attend(s):
    case, P = s["case"], s["case"]["block"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    lens, cu = s["seq_lens"].tolist(), s["cu_q"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["requests"]):
        at = s["tables"][b, : _blocks(lens[b], P)].long()
        n = cu[b + 1] - cu[b]
        last = lens[b] - n + torch.arange(n, device="cuda")
        for h in range(Hk):
            k = (s["k_cache"][at, h].double() * s["k_scale"][at, h].double()[:, None, None]).reshape(-1, _width(D))[: lens[b], :D]
            v = (s["v_cache"][at, h].double() * s["v_scale"][at, h].double()[:, None, None]).transpose(1, 2).reshape(-1, _width(D))[: lens[b], :D]
            for j in range(h * (H // Hk), (h + 1) * (H // Hk)):
                score = s["q"][cu[b]:cu[b + 1], j].double() @ k.t() / math.sqrt(D)
                score = torch.where(torch.arange(lens[b], device="cuda") <= last[:, None], score, -math.inf)
                out[cu[b]:cu[b + 1], j] = torch.softmax(score, -1) @ v
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "rope":
        rows = case["batch"] * case["length"]
        size = 4 if case["dtype"] == "f32" else 2
        values = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 5 if case["train"] else 2                     # x -> y; and with the backward x, dy -> dx
        top = min(rows, 2 * case["length"] + 64)
        return {"bytes": values * size * passes + top * case["rotary"] * 4 + rows * 4, "flops": values * (10 if not case["train"] else 30)}
    held, new = _lengths(case)
    if case["op"] == "tables":
        tokens, gone = int(np.maximum(0, new).sum()) + 5, int(_blocks(held, case["block"])[new < 0].sum())
        fresh = int((_blocks(held + np.maximum(0, new), case["block"]) - _blocks(held, case["block"]))[new >= 0].sum())
        return {"bytes": 4 * (5 * len(new) + 2 * tokens + 2 * fresh + 2 * gone + 3), "flops": 0}
    D = case["dim"]
    if case["op"] == "append":
        tokens = int(new.sum())
        touched = int((_blocks(held + new, case["block"]) - held // case["block"])[new > 0].sum())
        return {"bytes": 2 * tokens * case["kv_heads"] * D * (2 + 1) + 2 * touched * case["kv_heads"] * 8 + 4 * tokens, "flops": 4 * tokens * case["kv_heads"] * D}
    pairs = sum(int(n * h + n * (n + 1) // 2) for h, n in zip(held, new))
    blocks = int(_blocks(held + new, case["block"]).sum())
    return {"bytes": 2 * int((held + new).sum()) * case["kv_heads"] * D + 2 * blocks * case["kv_heads"] * 4 + 4 * blocks + 2 * 2 * int(new.sum()) * case["heads"] * D,
            "flops": 4 * pairs * case["heads"] * D}
