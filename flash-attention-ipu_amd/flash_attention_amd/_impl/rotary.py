"""Norm of query and key heads with the position rotation (fa_qk_norm_rope_*): checks, autograd, `torch.library` ops.

The operands are what the attention entry points of this package take ([B, H, L, D], any strides with a unit one on D) or the packed tokens of a
serving step ([T, H, D]); outputs and gradients keep the operands' layout.  The reference has no counterpart: its op takes queries and keys
as they are (sdpa.py:55-59)."""

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable
from torch.library import custom_op

from . import _native


def rotary_table(max_positions: int, rotary_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """float32 [max_positions, rotary_dim]: the cosines of the rotary_dim / 2 angles position * theta ** (-2 i / rotary_dim), then their sines.  Angles are formed
    in 64 bits: in 32 they lose a thousandth of a turn at position 10 ** 5."""
    if rotary_dim < 2 or rotary_dim % 2 or max_positions < 1 or not theta > 0:
        raise ValueError("rotary_table expects max_positions >= 1, an even rotary_dim >= 2 and theta > 0")
    turn = theta ** (-2.0 * torch.arange(rotary_dim // 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * turn
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _strides(t):
    """(batch, head, row) strides of [B, H, L, D] or [T, H, D]"""
    st = t.stride()
    return (st[0], st[1], st[2]) if len(st) == 4 else (0, st[1], st[0])


def _like(t: torch.Tensor) -> torch.Tensor:
    """uninitialised, in t's layout: heads inside the rows if t has them there, contiguous otherwise"""
    if t.ndim == 4 and t.stride(1) < t.stride(2):
        B, H, L, D = t.shape
        return t.new_empty_strided((B, H, L, D), (L * H * D, D, H * D, 1))
    return t.new_empty(t.shape)


_I64x12, _I64x18 = ctypes.c_int64 * 12, ctypes.c_int64 * 18
_BLOCKS = {}


def _stride_args(tensors):
    key = tuple(t.stride() for t in tensors)
    blk = _BLOCKS.get(key)
    if blk is None:
        if len(_BLOCKS) > 4096:
            _BLOCKS.clear()
        flat = [x for t in tensors for x in _strides(t)]
        blk = _BLOCKS[key] = (_I64x12 if len(tensors) == 4 else _I64x18)(*flat)
    return blk


def _geometry(q, k, table, positions):
    """(table pointer, rows, positions pointer, their bytes, their batch stride, B, L, heads, heads_kv, D, R)"""
    if q.ndim == 4:
        B, H, L, D = q.shape
    else:
        L, H, D = q.shape
        B = 1
    rows, R = table.shape
    if positions is None:
        ptr, nbytes, pos_sb = None, 4, 0
    else:
        ptr, nbytes = positions.data_ptr(), positions.element_size()
        pos_sb = positions.stride(0) if positions.ndim == 2 else 0
    return table.data_ptr(), rows, ptr, nbytes, pos_sb, B, L, H, k.shape[1], D, R


def _weight_dtype(q, w):
    return _native.FA_DTYPE[q.dtype if w is None else w.dtype]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    q, k = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k))
    q_out, k_out = _like(q), _like(k)
    if q.numel() and k.numel():
        lib = _native.load_native_library()
        geo = _geometry(q, k, table, positions)
        stream, prev = _native._stream_for(q)
        try:
            rc = lib.fa_qk_norm_rope_fwd(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), _ptr(q_weight), _ptr(k_weight),
                                         _weight_dtype(q, q_weight if q_weight is not None else k_weight), *geo, _stride_args((q, k, q_out, k_out)),
                                         _native.FA_DTYPE[q.dtype], eps, 1 if interleaved else 0, stream)
        finally:
            if prev >= 0:
                torch.cuda.set_device(prev)
        if rc != 0:
            _native._raise(rc)
    return q_out, k_out


def _bwd_impl(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, eps, interleaved, need_q_weight, need_k_weight):
    q, k, dq_out, dk_out = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, dq_out, dk_out))
    dq, dk = _like(q), _like(k)
    dqw = torch.empty_like(q_weight) if need_q_weight else None
    dkw = torch.empty_like(k_weight) if need_k_weight else None
    if q.numel() and k.numel():
        lib = _native.load_native_library()
        geo = _geometry(q, k, table, positions)
        ws, nbytes = None, 0
        if need_q_weight or need_k_weight:
            nbytes = lib.fa_qk_norm_rope_workspace(*geo[5:10])
            ws = torch.empty(nbytes // 4, dtype=torch.float32, device=q.device)
        stream, prev = _native._stream_for(q)
        try:
            rc = lib.fa_qk_norm_rope_bwd(q.data_ptr(), k.data_ptr(), dq_out.data_ptr(), dk_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), _ptr(q_weight), _ptr(k_weight),
                                         _ptr(dqw), _ptr(dkw), _weight_dtype(q, q_weight if q_weight is not None else k_weight), _ptr(ws), nbytes, *geo,
                                         _stride_args((q, k, dq_out, dk_out, dq, dk)), _native.FA_DTYPE[q.dtype], eps, 1 if interleaved else 0, stream)
        finally:
            if prev >= 0:
                torch.cuda.set_device(prev)
        if rc != 0:
            _native._raise(rc)
    else:
        dqw, dkw = (None if w is None else w.zero_() for w in (dqw, dkw))
    return dq, dk, dqw, dkw


# ---- torch.compile: opaque ops with fake implementations and a registered backward (a weight that is None travels as an empty tensor) -----------
@custom_op("flash_attention_amd::qk_norm_rope", mutates_args=())
def _op(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], table: torch.Tensor,
        positions: Optional[torch.Tensor], eps: float, interleaved: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved)


@_op.register_fake
def _(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    q, k = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k))
    return _like(q), _like(k)


@custom_op("flash_attention_amd::qk_norm_rope_bwd", mutates_args=())
def _op_bwd(q: torch.Tensor, k: torch.Tensor, dq_out: torch.Tensor, dk_out: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
            table: torch.Tensor, positions: Optional[torch.Tensor], eps: float,
            interleaved: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    dq, dk, dqw, dkw = _bwd_impl(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, eps, interleaved, q_weight is not None, k_weight is not None)
    return dq, dk, q.new_empty(0) if dqw is None else dqw, q.new_empty(0) if dkw is None else dkw


@_op_bwd.register_fake
def _(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, eps, interleaved):
    q, k = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k))
    return (_like(q), _like(k), q.new_empty(0) if q_weight is None else torch.empty_like(q_weight),
            q.new_empty(0) if k_weight is None else torch.empty_like(k_weight))


def _op_setup(ctx, inputs, output):
    q, k, q_weight, k_weight, table, positions, eps, interleaved = inputs
    ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
    ctx.eps, ctx.interleaved = eps, interleaved


def _op_backward(ctx, dq_out, dk_out):
    q, k, q_weight, k_weight, table, positions = ctx.saved_tensors
    dq, dk, dqw, dkw = _op_bwd(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, ctx.eps, ctx.interleaved)
    return dq, dk, None if q_weight is None else dqw, None if k_weight is None else dkw, None, None, None, None


_op.register_autograd(_op_backward, setup_context=_op_setup)


class _QkNormRopeFn(torch.autograd.Function):
    """eager path: the same two calls without the dispatcher's cost"""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, table, positions = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dqw, dkw = _bwd_impl(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, ctx.eps, ctx.interleaved, need[2], need[3])
        return dq, dk, dqw, dkw, None, None, None, None




def _check(q, k, q_weight, k_weight, table, positions, eps):
    name = "qk_norm_rope"
    if not (q.is_cuda and k.is_cuda and table.is_cuda):
        raise ValueError(f"{name} needs GPU tensors")
    if q.ndim not in (3, 4) or k.ndim != q.ndim:
        raise ValueError(f"{name} expects q and k of shape [B, H, L, D] or [T, H, D]")
    if q.dtype not in _native.FA_DTYPE or k.dtype != q.dtype:
        raise TypeError(f"{name}: q and k must have the same dtype out of float16, bfloat16, float32 (got {q.dtype}, {k.dtype})")
    tokens = (q.shape[0], q.shape[2]) if q.ndim == 4 else (q.shape[0],)
    if q.shape[-1] != k.shape[-1] or ((k.shape[0], k.shape[2]) if k.ndim == 4 else (k.shape[0],)) != tokens:
        raise ValueError(f"{name}: q and k must agree but for their heads (got {tuple(q.shape)}, {tuple(k.shape)})")
    D = q.shape[-1]
    if D < 2 or D > 512 or D % 2:
        raise ValueError(f"{name}: head dim must be even and at most 512 (got {D})")
    if table.ndim != 2 or table.dtype != torch.float32 or not table.is_contiguous() or table.shape[0] < 1 or table.shape[1] < 2 or table.shape[1] % 2 or table.shape[1] > D:
        raise ValueError(f"{name}: table must be a contiguous float32 [positions, rotary dim] with an even rotary dim up to the head dim (rotary_table)")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (D,) or w.dtype not in (q.dtype, torch.float32) or w.dtype != weights[0].dtype or w.stride(0) != 1:
            raise ValueError(f"{name}: weights must be contiguous [{D}], both in the operands' dtype or both float32")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: positions must be int32 or int64 (got {positions.dtype})")
        if tuple(positions.shape) not in ((tokens, tokens[1:]) if len(tokens) == 2 else (tokens,)):
            raise ValueError(f"{name}: positions must be [L] or [B, L] for [B, H, L, D], [T] for [T, H, D] (got {tuple(positions.shape)})")
    if any(t.device != q.device for t in (k, table, *weights, *(() if positions is None else (positions,)))):
        raise ValueError(f"{name}: all tensors must be on one device")
    if table.requires_grad:
        raise ValueError(f"{name} has no gradient for the table")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"{name}: eps must be finite and >= 0 (got {eps})")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], table: torch.Tensor,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """
    Root-mean-square norm of every query and key head, then the rotation by its position, in one pass; differentiable in q, k and the weights.

    q, k        [B, H, L, D] and [B, H_kv, L, D], or packed tokens [T, H, D] and [T, H_kv, D]; float16, bfloat16 or float32; D even, up to 512
    q_weight, k_weight   [D] in the operands' dtype or float32, or None for ones
    table       float32 [positions, rotary dim] from rotary_table(); a rotary dim below D leaves the columns behind it unrotated
    positions   int32 or int64, [L] or [B, L] ([T] for packed tokens); None = 0, 1, ...  Rows with a negative position are padding: zeros come out.
                A position that the table lacks gives NaN.
    interleaved False: columns (i, i + rotary dim / 2) are a pair; True: (2 i, 2 i + 1)
    returns     (q, k) normed and rotated, in the operands' layout
    """
    _check(q, k, q_weight, k_weight, table, positions, eps)
    if positions is not None and positions.ndim and positions.stride(-1) != 1 and positions.shape[-1] > 1:
        positions = positions.contiguous()
    if torch.compiler.is_compiling():
        return _op(q, k, q_weight, k_weight, table, positions, float(eps), bool(interleaved))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return _QkNormRopeFn.apply(q, k, q_weight, k_weight, table, positions, float(eps), bool(interleaved))
    return _fwd_impl(q, k, q_weight, k_weight, table, positions, float(eps), bool(interleaved))
