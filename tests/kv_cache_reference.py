"""Plain 64-bit forms of the cache operators, request by request, for the tests (independent of the package)."""

import numpy as np
import torch

E4M3_MAX = 448.0


def e4m3_values():
    """value of every code, NaN included"""
    v = np.zeros(256)
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        x = float("nan") if (e == 15 and m == 7) else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        v[c] = -x if s else x
    return v


def nearest_e4m3(x):
    """nearest e4m3 value, ties to the even code; |x| <= 448 or NaN"""
    with np.errstate(all="ignore"):
        _, e = np.frexp(x)
        step = np.exp2(np.maximum(e - 1, -6) - 3.0)
        return np.where(np.isfinite(x), np.rint(x / step) * step, np.nan)


def tables_reference(held, new, tables, pool, free, tokens, P):
    """sequential: the rules of cache_tables one request after the other"""
    held, new, tables, pool, free = list(held), list(new), [list(r) for r in tables], list(pool), int(free)
    width = len(tables[0])
    blocks = lambda n: -(-n // P)  # noqa: E731
    for b in range(len(held)):
        if new[b] < 0:
            for j in range(blocks(held[b])):
                pool[free] = tables[b][j]
                free += 1
    start, needed, take, granted, cu = 0, 0, free, [], [0]
    for b in range(len(held)):
        n = max(new[b], 0)
        start += n
        cu.append(start)
        fits = new[b] >= 0 and blocks(held[b] + n) <= width and start <= tokens
        need = blocks(held[b] + n) - blocks(held[b]) if fits else 0
        needed += need
        ok = fits and (need == 0 or needed <= free)
        if ok:
            for j in range(need):
                take -= 1
                tables[b][blocks(held[b]) + j] = pool[take]
        granted.append(n if ok else 0)
        held[b] = 0 if new[b] < 0 else held[b] + granted[b]
    pos, slot = [-1] * tokens, [-1] * tokens
    for b in range(len(held)):
        for i in range(granted[b]):
            p = held[b] - granted[b] + i
            pos[cu[b] + i] = p
            slot[cu[b] + i] = tables[b][p // P] * P + p % P
    return dict(seq_lens=held, free=take, cu=cu, granted=granted, positions=pos, slots=slot, tables=tables, pool=pool)


def append_reference(x, slots, values, scale, P):
    """x [T, H, D] float64, values [blocks, H, P, W] (code values), scale [blocks, H]: both changed in place, run by run"""
    T = len(slots)
    t = 0
    while t < T:
        if slots[t] < 0 or slots[t] >= values.shape[0] * P:
            t += 1
            continue
        n = 1
        while t + n < T and slots[t + n] == slots[t] + n and slots[t + n] % P != 0:
            n += 1
        blk, off = int(slots[t]) // P, int(slots[t]) % P
        for h in range(x.shape[1]):
            run = x[t:t + n, h]
            finite = np.abs(run[np.isfinite(run)])
            largest = finite.max() if finite.size else 0.0
            e = -100
            if largest > 0:
                m, e2 = np.frexp(largest)                  # 448 = 0.875 * 2 ** 9
                e = max(-100, int(e2) - 9 + (1 if m > 0.875 else 0))
            wanted = 2.0 ** e
            if off == 0:
                now = wanted
            else:
                now = max(wanted, scale[blk, h])
                if now != scale[blk, h]:
                    values[blk, h] = nearest_e4m3(values[blk, h] * (scale[blk, h] / now))
            scale[blk, h] = now
            row = np.zeros((n, values.shape[3]))
            row[:, : x.shape[2]] = np.where(np.isfinite(run), run, np.nan) / now
            values[blk, h, off:off + n] = nearest_e4m3(row)
        t += n


def attention_reference(q, k_values, v_values, k_scale, v_scale, tables, lens, cu, scale):
    """q [T, H, D] float64; k_values / v_values [blocks, Hkv, P, W] code values; returns out and the same with |v| (for tolerances)"""
    T, H, D = q.shape
    N, Hkv, P, _ = k_values.shape
    out, mag = torch.full((T, H, D), float("nan"), dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        if n <= 0:
            continue
        L = lens[b]
        ids = [int(i) for i in tables[b][: -(-L // P)]]
        ok = torch.tensor([0 <= ids[t // P] < N for t in range(L)], dtype=torch.bool) if L else torch.zeros(0, dtype=torch.bool)
        pick = [i if 0 <= i < N else 0 for i in ids]
        rows = slice(cu[b], cu[b] + n)
        if L == 0 or not bool(ok.any()):
            out[rows] = 0
            continue
        see = (torch.arange(L)[None] <= (L - n + torch.arange(n))[:, None]) & ok            # [n, L]
        for hk in range(Hkv):
            k = (k_values[pick, hk] * k_scale[pick, hk][:, None, None]).reshape(-1, k_values.shape[3])[:L, :D]
            v = (v_values[pick, hk] * v_scale[pick, hk][:, None, None]).reshape(-1, v_values.shape[3])[:L, :D]
            nan = torch.isnan(v)
            hit = (see.double() @ nan.double()) > 0                                          # [n, D]: the row sees a NaN value in that column
            v = torch.where(nan, 0.0, v)
            for h in range(hk * (H // Hkv), (hk + 1) * (H // Hkv)):
                s = torch.where(see, q[rows, h] @ k.t() * scale, -float("inf"))
                p = torch.where(see.any(1, keepdim=True), torch.softmax(s, 1), 0.0)
                out[rows, h] = torch.where(hit, float("nan"), p @ v)
                mag[rows, h] = p @ v.abs()
    return out, mag
