"""Attention over a block cache of 8-bit keys and values: checks and calls of fa_cache_tables, fa_cache_append and fa_cache_attn.

The reference attends to whole sequences only (it rejects query.shape != key.shape, sdpa.py:33-37); this is the counterpart of its op for a
generation loop.  No length, table or slot is read on the host: a step enqueues kernels only and can be captured in a HIP graph."""

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version
from torch.library import custom_op

from . import _native

BLOCK_SIZES = (16, 32, 64, 128)
_I64x4 = ctypes.c_int64 * 4
_BLOCKS = {}


def _i64x4(key):
    blk = _BLOCKS.get(key)
    if blk is None:
        if len(_BLOCKS) > 4096:
            _BLOCKS.clear()
        blk = _BLOCKS[key] = _I64x4(*key)
    return blk


_LAYOUTS = {}       # (shapes, strides, dtypes) that passed the checks -> what the call needs of them


def _remember(key, value):
    if len(_LAYOUTS) > 4096:
        _LAYOUTS.clear()
    _LAYOUTS[key] = value
    return value


def cache_width(head_dim: int) -> int:
    """columns that a head takes in the cache: the head dim rounded up to a multiple of 64"""
    return (head_dim + 63) // 64 * 64


class CacheStep(NamedTuple):
    """What a step did and where its tokens are (cache_tables)."""

    seq_lens: torch.Tensor      # int32 [B]      tokens that every request holds afterwards
    free_count: torch.Tensor    # int32 [1]      free blocks afterwards
    cu_new: torch.Tensor        # int32 [B + 1]  where every request's tokens begin among the step's tokens
    granted: torch.Tensor       # int32 [B]      tokens that every request was served: all of its own or 0
    positions: torch.Tensor     # int32 [T]      position of every token in its request, -1 = padding or not served
    slots: torch.Tensor         # int32 [T]      its place in the cache (block * block size + offset), -1 likewise


def _ints(name, what, t, shape=None):
    if not t.is_cuda:
        raise ValueError(f"{name} needs GPU tensors ({what})")
    if t.dtype != torch.int32:
        raise TypeError(f"{name}: {what} must be int32 (got {t.dtype})")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name}: {what} must have shape {shape} (got {tuple(t.shape)})")
    if t.ndim and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: {what} must be contiguous along its last dimension")


def _table(name, block_tables, requests):
    _ints(name, "block_tables", block_tables)
    if block_tables.ndim != 2 or block_tables.shape[0] != requests or block_tables.shape[1] < 1:
        raise ValueError(f"{name}: block_tables must be [{requests}, blocks] (got {tuple(block_tables.shape)})")
    return block_tables.shape[1], block_tables.stride(0) if requests > 1 else block_tables.shape[1]


def _tables_call(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, seq_out, free_out, cu_new, granted, positions, slots):
    lib = _native._LIB or _native.load_native_library()
    B = seq_lens.shape[0]
    stream, prev = _native.stream_of(seq_lens.device)
    try:
        rc = lib.fa_cache_tables(seq_lens.data_ptr(), new_lens.data_ptr(), block_tables.data_ptr(), block_tables.stride(0) if B > 1 else block_tables.shape[1],
                                 block_tables.shape[1], free_blocks.data_ptr(), free_blocks.shape[0], free_count.data_ptr(), B, num_tokens, block_size,
                                 seq_out.data_ptr(), free_out.data_ptr(), cu_new.data_ptr(), granted.data_ptr(), positions.data_ptr(), slots.data_ptr(), stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _native._raise(rc)


@custom_op("flash_attention_amd::cache_tables", mutates_args=("block_tables", "free_blocks", "seq_out", "free_out", "cu_new", "granted", "positions", "slots"))
def _tables_op(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor, free_count: torch.Tensor, num_tokens: int,
               block_size: int, seq_out: torch.Tensor, free_out: torch.Tensor, cu_new: torch.Tensor, granted: torch.Tensor, positions: torch.Tensor,
               slots: torch.Tensor) -> None:
    _tables_call(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, seq_out, free_out, cu_new, granted, positions, slots)


def _check_tables(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, inplace):
    """(int32 values of the outputs in all, one by one)"""
    name = "cache_tables"
    if seq_lens.ndim != 1 or seq_lens.shape[0] < 1:
        raise ValueError(f"{name}: seq_lens must be [requests] (got {tuple(seq_lens.shape)})")
    B = seq_lens.shape[0]
    _ints(name, "seq_lens", seq_lens)
    _ints(name, "new_lens", new_lens, (B,))
    _ints(name, "free_count", free_count, (1,))
    _ints(name, "free_blocks", free_blocks)
    if free_blocks.ndim != 1 or free_blocks.shape[0] < 1:
        raise ValueError(f"{name}: free_blocks must be [blocks] (got {tuple(free_blocks.shape)})")
    _table(name, block_tables, B)
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"{name}: block_size must be one of {BLOCK_SIZES} (got {block_size})")
    if num_tokens < 0:
        raise ValueError(f"{name}: num_tokens must be >= 0 (got {num_tokens})")
    sizes = [B + 1, B, num_tokens, num_tokens] + ([] if inplace else [B, 1])
    return sum(sizes), sizes


def cache_tables(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor, free_count: torch.Tensor, num_tokens: int,
                 block_size: int, inplace: bool = False) -> CacheStep:
    """
    Block tables, positions and slots of one step, on the device.

    seq_lens     int32 [B]: tokens that the requests hold;   new_lens  int32 [B]: tokens that come, 0 for none, negative for a request that ends
    block_tables int32 [B, blocks]: changed in place where blocks are added
    free_blocks  int32 [N], free_count int32 [1]: the pool; free_blocks[:free_count] are free.  Blocks of requests that end are put behind them (in
                 place) before blocks are taken from the end.
    num_tokens   rows of the step's token tensors: at least the sum of new_lens; the rows behind it get -1
    inplace      True: the new lengths and the new count overwrite seq_lens and free_count (a captured step then advances with every replay)

    A request is served whole or not at all (granted): its tokens have to end inside num_tokens, its blocks have to fit its table row, and the pool has
    to hold what all such requests up to and including it need.  Nothing is read back: look at `granted` when the host next waits for the device.
    """
    dispatch = torch.compiler.is_compiling() or _native.dispatch_modes()
    if dispatch:
        sizes = _check_tables(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, inplace)
    else:
        key = (seq_lens.shape, seq_lens.stride(), seq_lens.dtype, new_lens.shape, new_lens.stride(), new_lens.dtype, block_tables.shape, block_tables.stride(), block_tables.dtype,
               free_blocks.shape, free_blocks.stride(), free_blocks.dtype, free_count.shape, free_count.dtype, num_tokens, block_size, inplace)
        sizes = _LAYOUTS.get(key)
        if sizes is None:
            sizes = _remember(key, _check_tables(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, inplace))
    dev = seq_lens.device
    if not (seq_lens.is_cuda and new_lens.device == dev and block_tables.device == dev and free_blocks.device == dev and free_count.device == dev):
        raise ValueError("cache_tables: all tensors must be on one GPU")
    # one allocation: cu_new, granted, positions, slots and, unless in place, lengths and count
    parts = torch.split_with_sizes(seq_lens.new_empty(sizes[0]), sizes[1])
    cu_new, granted, positions, slots = parts[:4]
    seq_out, free_out = (seq_lens, free_count) if inplace else parts[4:]
    if dispatch:
        _tables_op(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, seq_out, free_out, cu_new, granted, positions, slots)
    else:
        _tables_call(seq_lens, new_lens, block_tables, free_blocks, free_count, num_tokens, block_size, seq_out, free_out, cu_new, granted, positions, slots)
        increment_version((block_tables, free_blocks, seq_lens, free_count) if inplace else (block_tables, free_blocks))
    return CacheStep(seq_out, free_out, cu_new, granted, positions, slots)


def _check_cache(name, k_cache, v_cache, k_scale, v_scale, heads_kv, D):
    """(width, blocks, block size, block strides) of a cache that holds `heads_kv` heads of `D` columns"""
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{name}: caches must be float8_e4m3fn (got {k_cache.dtype}, {v_cache.dtype})")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise TypeError(f"{name}: scales must be float32")
    if D < 8 or D > 256 or D % 8:
        raise ValueError(f"{name}: head dim must be a multiple of 8 up to 256 (got {D})")
    W = (D + 63) // 64 * 64
    if k_cache.ndim != 4 or v_cache.ndim != 4 or k_cache.shape[2] not in BLOCK_SIZES:
        raise ValueError(f"{name}: k_cache must be [blocks, heads, block size, width], block size one of {BLOCK_SIZES} (got {tuple(k_cache.shape)})")
    N, H, P, _ = k_cache.shape
    if k_cache.shape != (N, heads_kv, P, W) or v_cache.shape != (N, heads_kv, W, P) or N < 1:
        raise ValueError(f"{name}: {heads_kv} heads of {D} need k_cache [blocks, {heads_kv}, block size, {W}] and v_cache [blocks, {heads_kv}, {W}, block size] "
                         f"(got {tuple(k_cache.shape)}, {tuple(v_cache.shape)})")
    if k_scale.shape != (N, H) or v_scale.shape != (N, H) or (H > 1 and (k_scale.stride(1) != 1 or v_scale.stride(1) != 1)):
        raise ValueError(f"{name}: scales must be [{N}, {H}] with the heads contiguous")
    ks, vs, kss, vss = k_cache.stride(), v_cache.stride(), k_scale.stride(0), v_scale.stride(0)
    if ks[1:] != (P * W, W, 1) or vs[1:] != (P * W, P, 1):
        if (H > 1 or ks[2:] != (W, 1) or vs[2:] != (P, 1)):
            raise ValueError(f"{name}: everything inside a block must be contiguous")
    if N == 1:        # (a single block's stride says nothing)
        return W, N, P, (H * P * W, H * P * W, H, H)
    return W, N, P, (ks[0], vs[0], kss, vss)


def _append_call(k, v, slots, k_cache, v_cache, k_scale, v_scale):
    name = "cache_append"
    key = (k.shape, k.stride(), v.shape, v.stride(), k.dtype, v.dtype, slots.shape, slots.stride(), slots.dtype, k_cache.shape, k_cache.stride(), v_cache.shape, v_cache.stride(),
           k_cache.dtype, v_cache.dtype, k_scale.shape, k_scale.stride(), v_scale.shape, v_scale.stride(), k_scale.dtype, v_scale.dtype)
    known = _LAYOUTS.get(key)
    if known is None:
        if k.dtype not in (torch.float16, torch.bfloat16) or v.dtype != k.dtype:
            raise TypeError(f"{name}: k and v must have the same dtype out of float16, bfloat16 (got {k.dtype}, {v.dtype})")
        if k.ndim != 3 or v.shape != k.shape:
            raise ValueError(f"{name}: k and v must be [tokens, heads, head dim] (got {tuple(k.shape)}, {tuple(v.shape)})")
        _ints(name, "slots", slots, (k.shape[0],))
        W, N, P, strides = _check_cache(name, k_cache, v_cache, k_scale, v_scale, k.shape[1], k.shape[2])
        rows = all(t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 for t in (k, v))
        known = _remember(key, (W, N, P, _i64x4(strides), rows, _i64x4((k.stride(0), k.stride(1), v.stride(0), v.stride(1))), _native.FA_DTYPE[k.dtype]))
    W, N, P, strides, rows, tokens, dtype = known
    dev = k.device
    if not (k.is_cuda and dev == v.device == slots.device == k_cache.device == v_cache.device == k_scale.device == v_scale.device):
        raise ValueError(f"{name}: all tensors must be on one GPU")
    kp, vp = k.data_ptr(), v.data_ptr()
    if not rows or kp % 16 or vp % 16:           # (rows that a 16-byte load does not fit: copied)
        k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        kp, vp = k.data_ptr(), v.data_ptr()
        tokens = _i64x4((k.stride(0), k.stride(1), v.stride(0), v.stride(1)))
    lib = _native._LIB or _native.load_native_library()
    T, H, D = k.shape
    if T == 0:
        return
    stream, prev = _native.stream_of(dev)
    try:
        rc = lib.fa_cache_append(kp, vp, slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), T, H, D, W, N, P, tokens,
                                 strides, dtype, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _native._raise(rc)


@custom_op("flash_attention_amd::cache_append", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def _append_op(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor) -> None:
    _append_call(k, v, slots, k_cache, v_cache, k_scale, v_scale)


def cache_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor) -> None:
    """
    Keys and values of a step's tokens into the cache, as e4m3 codes with one power-of-two scale per block and head; in place, without a gradient.

    k, v     [T, heads, D] float16 or bfloat16, D a multiple of 8 up to 256 (strided views are read as they are where their rows are 16-byte aligned)
    slots    int32 [T] (CacheStep.slots); tokens with a slot below 0 or outside the cache are skipped
    k_cache  float8_e4m3fn [blocks, heads, block size, width], v_cache [blocks, heads, width, block size]; width = cache_width(D), block size 16, 32, 64 or 128
    k_scale, v_scale  float32 [blocks, heads]; value = code * scale

    A run (tokens whose slots follow each other inside a block) that starts its block sets the block's scale to the smallest power of two that holds its
    largest value; later runs raise it where they need to, and the block's codes are brought along.  inf and NaN are stored as NaN.  One call may bring
    one run to a block: two runs in one block, or a slot twice, leave that block's contents unspecified.
    """
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad or k_scale.requires_grad or v_scale.requires_grad):
        raise ValueError("cache_append has no gradient: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _native.refuse_tangents("cache_append", k, v, k_cache, v_cache, k_scale, v_scale)
    if torch.compiler.is_compiling() or _native.dispatch_modes():
        return _append_op(k, v, slots, k_cache, v_cache, k_scale, v_scale)
    _append_call(k, v, slots, k_cache, v_cache, k_scale, v_scale)
    increment_version((k_cache, v_cache, k_scale, v_scale))


def _rows_overlap(t):
    """whether rows of [T, heads, D] with a unit stride on D can share memory: every larger stride has to step over all that the smaller ones span"""
    span = t.shape[2]
    for stride, n in sorted((s, n) for s, n in zip(t.stride()[:2], t.shape[:2]) if n > 1):
        if stride < span:
            return True
        span += stride * (n - 1)
    return False


def _attn_call(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, softmax_scale, max_q_len, out, granted):
    name = "flash_attention_cached"
    key = (q.shape, q.stride(), q.dtype, None if out is None else (out.shape, out.stride(), out.dtype), max_q_len, k_cache.shape, k_cache.stride(), v_cache.shape, v_cache.stride(), k_cache.dtype,
           v_cache.dtype, k_scale.shape, k_scale.stride(), v_scale.shape, v_scale.stride(), k_scale.dtype, v_scale.dtype, block_tables.shape, block_tables.stride(),
           block_tables.dtype, seq_lens.shape, seq_lens.stride(), seq_lens.dtype, cu_q.shape, cu_q.stride(), cu_q.dtype,
           None if granted is None else (granted.shape, granted.stride(), granted.dtype))
    lib = _native._LIB or _native.load_native_library()
    known = _LAYOUTS.get(key)
    if known is None:
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"{name}: q must be float16 or bfloat16 (got {q.dtype})")
        if q.ndim != 3 or q.shape[1] < 1:
            raise ValueError(f"{name}: q must be [tokens, heads, head dim] (got {tuple(q.shape)})")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or out.stride(0) % 8 or out.stride(1) % 8):
            raise ValueError(f"{name}: out must have q's shape and dtype and 16-byte rows")
        if out is not None and _rows_overlap(out):
            raise ValueError(f"{name}: rows of out must not share memory (strides {out.stride()})")
        T, H, D = q.shape
        heads_kv = k_cache.shape[1] if k_cache.ndim == 4 else 0
        if heads_kv < 1 or H % heads_kv:
            raise ValueError(f"{name}: the cache's heads must divide q's (got {tuple(k_cache.shape)}, {tuple(q.shape)})")
        W, N, P, strides = _check_cache(name, k_cache, v_cache, k_scale, v_scale, heads_kv, D)
        _ints(name, "seq_lens", seq_lens)
        if seq_lens.ndim != 1 or seq_lens.shape[0] < 1:
            raise ValueError(f"{name}: seq_lens must be [requests] (got {tuple(seq_lens.shape)})")
        B = seq_lens.shape[0]
        _ints(name, "cu_q", cu_q, (B + 1,))
        if granted is not None:
            _ints(name, "granted", granted, (B,))
        width, table_stride = _table(name, block_tables, B)
        if max_q_len < 1:
            raise ValueError(f"{name}: max_q_len must be >= 1 (got {max_q_len})")
        nbytes = lib.fa_cache_attn_workspace(B, T, H, heads_kv, D, P, width, max_q_len)
        if nbytes < 0:
            _native._raise(int(nbytes))
        rows = q.stride(2) == 1 and q.stride(0) % 8 == 0 and q.stride(1) % 8 == 0
        known = _remember(key, ((B, T, H, heads_kv, D, W, N, P, width, table_stride, max_q_len), nbytes, rows,
                                _i64x4((q.stride(0), q.stride(1)) + (out.stride()[:2] if out is not None else (H * D, D))), _i64x4(strides), _native.FA_DTYPE[q.dtype]))
    sizes, nbytes, rows, tokens, strides, dtype = known
    dev = q.device
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=dev)     # (the first takes half the time)
    if not (q.is_cuda and dev == out.device == k_cache.device == v_cache.device == k_scale.device == v_scale.device == block_tables.device == seq_lens.device
            == cu_q.device and (granted is None or granted.device == dev)):
        raise ValueError(f"{name}: all tensors must be on one GPU")
    if out.data_ptr() % 16:
        raise ValueError(f"{name}: out must be 16-byte aligned")
    if sizes[1] == 0:
        return out
    if not rows or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        tokens = _i64x4((q.stride(0), q.stride(1), out.stride(0), out.stride(1)))
    # (a workspace of its own for every call: the allocator orders its reuse on the stream, and a captured graph keeps the one it was captured with)
    ws = seq_lens.new_empty((nbytes + 3) // 4) if nbytes else None
    stream, prev = _native.stream_of(dev)
    try:
        rc = lib.fa_cache_attn_granted(q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_tables.data_ptr(),
                                       seq_lens.data_ptr(), cu_q.data_ptr(), None if granted is None else granted.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
                                       *sizes, tokens, strides, dtype, softmax_scale, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _native._raise(rc)
    return out


@custom_op("flash_attention_amd::cached", mutates_args=("out",))
def _attn_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
             seq_lens: torch.Tensor, cu_q: torch.Tensor, softmax_scale: float, max_q_len: int, out: torch.Tensor, granted: Optional[torch.Tensor] = None) -> None:
    _attn_call(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, softmax_scale, max_q_len, out, granted)


def flash_attention_cached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                           seq_lens: torch.Tensor, cu_q: torch.Tensor, softmax_scale: Optional[float] = None, max_q_len: Optional[int] = None,
                           out: Optional[torch.Tensor] = None, granted: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    Causal attention of a step's queries over the cached keys and values of their requests; for inference (no gradient).

    q            [T, heads, D] float16 or bfloat16, D a multiple of 8 up to 256; heads a multiple of the cache's heads (grouped queries)
    k_cache, v_cache, k_scale, v_scale   as cache_append fills them; the step's own keys and values are appended first
    block_tables int32 [B, blocks];  seq_lens int32 [B]: tokens that every request holds, the step's included
    cu_q         int32 [B + 1]: request b's queries are the rows cu_q[b] .. cu_q[b + 1] - 1 of q, the last of its seq_lens[b] tokens
                 (CacheStep.cu_new).  A query sees the keys up to its own position.
    softmax_scale  default D ** -0.5
    max_q_len    the most queries of one request, as far as the host knows; chooses the kernel, never the result.  Default: max(1, T - B + 1), a guess that holds where
                 every request has a token: T == B is a step of single tokens.  Where rows of the batch are idle (no tokens in this step) a prompt can be longer: say
                 so, or it runs on the kernel for few rows, which reads the request's cache once for every 16 or 32 of its rows.  Give prompts and single tokens calls of
                 their own where both are many: one long cache is split over the chip by the kernel for single tokens only.
    out          [T, heads, D], default a new tensor.  Rows behind cu_q[B] are not written: a new tensor holds anything there.
    granted      int32 [B] (CacheStep.granted): the rows of a request that was refused, whose tokens are not in the cache, give zeros.  Default: every request counts
                 as served, and the rows of a refused one as the last tokens of what it holds.
    returns      out.  A query that sees no key (an empty request) gives zeros.
    """
    if q.ndim != 3:
        raise ValueError(f"flash_attention_cached: q must be [tokens, heads, head dim] (got {tuple(q.shape)})")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or k_scale.requires_grad or v_scale.requires_grad
                                    or (out is not None and out.requires_grad)):
        raise ValueError("flash_attention_cached has no gradient: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _native.refuse_tangents("flash_attention_cached", q, k_cache, v_cache, k_scale, v_scale, out)
    if softmax_scale is None:
        softmax_scale = q.shape[2] ** -0.5
    elif not 0.0 < softmax_scale < float("inf"):
        raise ValueError(f"flash_attention_cached: softmax_scale must be finite and > 0 (got {softmax_scale})")
    if max_q_len is None:
        max_q_len = max(1, q.shape[0] - seq_lens.shape[0] + 1) if seq_lens.ndim == 1 else 1
    if torch.compiler.is_compiling() or _native.dispatch_modes():
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _attn_op(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, softmax_scale, max_q_len, out, granted)
        return out
    if out is None:
        return _attn_call(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, softmax_scale, max_q_len, None, granted)
    _attn_call(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_q, softmax_scale, max_q_len, out, granted)
    increment_version(out)
    return out


class KVCache:
    """
    The cache of a model's attention layers and the state of its requests.

        cache = KVCache(layers, blocks, kv_heads, head_dim, requests=B, max_tokens=4096)
        step = cache.step(new_lens, num_tokens)              # once per model step
        y = cache.attend(layer, q, k, v, step)               # in every layer: k and v appended, then attention

    `requests` rows are held; a row that is free holds 0 tokens.  step() advances lengths, tables and pool in place, on the device.
    """

    def __init__(self, layers: int, blocks: int, kv_heads: int, head_dim: int, requests: int, max_tokens: int, block_size: int = 64, device="cuda"):
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"KVCache: block_size must be one of {BLOCK_SIZES} (got {block_size})")
        if min(layers, blocks, kv_heads, requests, max_tokens) < 1 or head_dim < 8 or head_dim > 256 or head_dim % 8:
            raise ValueError("KVCache: layers, blocks, kv_heads, requests and max_tokens must be >= 1, head_dim a multiple of 8 up to 256")
        W = cache_width(head_dim)
        self.layers, self.blocks, self.kv_heads, self.head_dim, self.block_size, self.max_tokens = layers, blocks, kv_heads, head_dim, block_size, max_tokens
        self.k_cache = torch.empty((layers, blocks, kv_heads, block_size, W), dtype=torch.float8_e4m3fn, device=device)
        self.v_cache = torch.empty((layers, blocks, kv_heads, W, block_size), dtype=torch.float8_e4m3fn, device=device)
        self.k_scale = torch.ones((layers, blocks, kv_heads), dtype=torch.float32, device=device)
        self.v_scale = torch.ones((layers, blocks, kv_heads), dtype=torch.float32, device=device)
        self.block_tables = torch.full((requests, (max_tokens + block_size - 1) // block_size), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free_blocks = torch.arange(blocks, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), blocks, dtype=torch.int32, device=device)
        self._layer = [tuple(t[i] for t in (self.k_cache, self.v_cache, self.k_scale, self.v_scale)) for i in range(layers)]

    def step(self, new_lens: torch.Tensor, num_tokens: int) -> CacheStep:
        """lengths, tables and pool brought to the next step (cache_tables, in place)"""
        return cache_tables(self.seq_lens, new_lens, self.block_tables, self.free_blocks, self.free_count, num_tokens, self.block_size, inplace=True)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: CacheStep) -> None:
        cache_append(k, v, step.slots, *self._layer[layer])

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: CacheStep, softmax_scale: Optional[float] = None,
               max_q_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """the step's keys and values into the layer's cache, then its queries' attention (zeros for a request that was refused).  A step that brings a prompt while
        other rows are idle should say so in max_q_len: the default takes every row to have a token (flash_attention_cached)"""
        self.append(layer, k, v, step)
        return flash_attention_cached(q, *self._layer[layer], self.block_tables, step.seq_lens, step.cu_new, softmax_scale, max_q_len, out, step.granted)
