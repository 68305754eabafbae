"""Norm of query and key heads with the position rotation (fa_qk_norm_rope_*): checks, autograd, `torch.library` ops.

The operands are what the attention entry points of this package take ([B, H, L, D], any strides with a unit one on D) or the packed tokens of a
serving step ([T, H, D]); outputs and gradients keep the operands' layout.  The reference has no counterpart: its op takes queries and keys
as they are (sdpa.py:55-59)."""

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
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


_I64x12, _I64x18 = ctypes.c_int64 * 12, ctypes.c_int64 * 18
_CALLS = {}         # layout of the operands -> what the native calls need of it


class _Call:
    """Everything about a call that follows from shapes, strides and dtypes: checked and formed once for each of them."""

    __slots__ = ("sizes", "table_rows", "position_bytes", "position_stride", "weight_dtype", "dtype", "fwd_strides", "bwd_strides", "workspace")

    def __init__(self, q, k, q_weight, k_weight, table, positions):
        if q.ndim == 4:
            B, H, L, D = q.shape
        else:
            L, H, D = q.shape
            B = 1
        self.sizes = (B, L, H, k.shape[1], D, table.shape[1])
        self.table_rows = table.shape[0]
        self.position_bytes = 4 if positions is None else positions.element_size()
        self.position_stride = positions.stride(0) if positions is not None and positions.ndim == 2 else 0
        weight = q_weight if q_weight is not None else k_weight
        self.dtype = _native.FA_DTYPE[q.dtype]
        self.weight_dtype = self.dtype if weight is None else _native.FA_DTYPE[weight.dtype]
        self.fwd_strides = None
        self.bwd_strides = {}
        self.workspace = _native.load_native_library().fa_qk_norm_rope_workspace(B, L, H, k.shape[1], D)


def _call_for(q, k, q_weight, k_weight, table, positions):
    key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, None if q_weight is None else (q_weight.shape, q_weight.stride(), q_weight.dtype),
           None if k_weight is None else (k_weight.shape, k_weight.stride(), k_weight.dtype), table.shape, table.stride(), table.dtype,
           None if positions is None else (positions.shape, positions.stride(), positions.dtype))
    call = _CALLS.get(key)
    if call is None:
        _check(q, k, q_weight, k_weight, table, positions)
        if len(_CALLS) > 4096:
            _CALLS.clear()
        call = _CALLS[key] = _Call(q, k, q_weight, k_weight, table, positions)
    dev = q.device
    if not (q.is_cuda and k.device == dev and table.device == dev and (q_weight is None or q_weight.device == dev) and (k_weight is None or k_weight.device == dev)
            and (positions is None or positions.device == dev)):
        raise ValueError("qk_norm_rope: all tensors must be on one GPU")
    return call


def _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    call = _call_for(q, k, q_weight, k_weight, table, positions)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)          # (the operands' layout: heads inside the rows stay there)
    if call.sizes[0] and call.sizes[1]:
        if call.fwd_strides is None:
            call.fwd_strides = _I64x12(*(x for t in (q, k, q_out, k_out) for x in _strides(t)))
        stream, prev = _native.stream_of(q.device)
        try:
            rc = _native._LIB.fa_qk_norm_rope_fwd(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), None if q_weight is None else q_weight.data_ptr(),
                                                  None if k_weight is None else k_weight.data_ptr(), call.weight_dtype, table.data_ptr(), call.table_rows,
                                                  None if positions is None else positions.data_ptr(), call.position_bytes, call.position_stride, *call.sizes,
                                                  call.fwd_strides, call.dtype, eps, interleaved, stream)
        finally:
            if prev >= 0:
                torch.cuda.set_device(prev)
        if rc != 0:
            _native._raise(rc)
    return q_out, k_out


def _bwd_impl(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, eps, interleaved, need_q_weight, need_k_weight):
    # (not the forward's call: hooks on saved tensors may hand them back with other strides, as torch.autograd.graph.save_on_cpu does)
    if q.stride(-1) != 1 or k.stride(-1) != 1:
        q, k = q.contiguous(), k.contiguous()
    if positions is not None and positions.stride(-1) != 1:
        positions = positions.contiguous()
    call = _call_for(q, k, q_weight, k_weight, table, positions)
    if dq_out.stride(-1) != 1 or dk_out.stride(-1) != 1:
        dq_out, dk_out = dq_out.contiguous(), dk_out.contiguous()
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dqw = torch.empty_like(q_weight) if need_q_weight else None
    dkw = torch.empty_like(k_weight) if need_k_weight else None
    if not (call.sizes[0] and call.sizes[1]):
        return dq, dk, None if dqw is None else dqw.zero_(), None if dkw is None else dkw.zero_()
    key = (dq_out.stride(), dk_out.stride())
    strides = call.bwd_strides.get(key)
    if strides is None:
        if len(call.bwd_strides) > 256:
            call.bwd_strides.clear()
        strides = call.bwd_strides[key] = _I64x18(*(x for t in (q, k, dq_out, dk_out, dq, dk) for x in _strides(t)))
    ws, nbytes = None, 0
    if need_q_weight or need_k_weight:
        nbytes = call.workspace
        ws = table.new_empty(nbytes // 4)
    stream, prev = _native.stream_of(q.device)
    try:
        rc = _native._LIB.fa_qk_norm_rope_bwd(q.data_ptr(), k.data_ptr(), dq_out.data_ptr(), dk_out.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                              None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
                                              None if dqw is None else dqw.data_ptr(), None if dkw is None else dkw.data_ptr(), call.weight_dtype,
                                              None if ws is None else ws.data_ptr(), nbytes, table.data_ptr(), call.table_rows,
                                              None if positions is None else positions.data_ptr(), call.position_bytes, call.position_stride, *call.sizes, strides,
                                              call.dtype, eps, interleaved, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _native._raise(rc)
    return dq, dk, dqw, dkw


# ---- torch.compile: opaque ops with fake implementations and a registered backward (a weight that is None travels as an empty tensor) -----------
@custom_op("flash_attention_amd::qk_norm_rope", mutates_args=())
def _op(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], table: torch.Tensor,
        positions: Optional[torch.Tensor], eps: float, interleaved: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved)


@_op.register_fake
def _(q, k, q_weight, k_weight, table, positions, eps, interleaved):
    return torch.empty_like(q), torch.empty_like(k)


@custom_op("flash_attention_amd::qk_norm_rope_bwd", mutates_args=())
def _op_bwd(q: torch.Tensor, k: torch.Tensor, dq_out: torch.Tensor, dk_out: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
            table: torch.Tensor, positions: Optional[torch.Tensor], eps: float,
            interleaved: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    dq, dk, dqw, dkw = _bwd_impl(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, eps, interleaved, q_weight is not None, k_weight is not None)
    return dq, dk, q.new_empty(0) if dqw is None else dqw, q.new_empty(0) if dkw is None else dkw


@_op_bwd.register_fake
def _(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, eps, interleaved):
    return (torch.empty_like(q), torch.empty_like(k), q.new_empty(0) if q_weight is None else torch.empty_like(q_weight),
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


def _backward(ctx, dq_out, dk_out):
    q, k, q_weight, k_weight, table, positions = ctx.saved_tensors
    need = ctx.needs_input_grad
    if torch.compiler.is_compiling() or _native.dispatch_modes():         # (a tracer that looks on at the backward alone)
        dq, dk, dqw, dkw = _op_bwd(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, ctx.eps, ctx.interleaved)
        return dq, dk, dqw if need[2] else None, dkw if need[3] else None, None, None, None, None
    return (*_bwd_impl(q, k, dq_out, dk_out, q_weight, k_weight, table, positions, ctx.eps, ctx.interleaved, need[2], need[3]), None, None, None, None)


_backward_once = once_differentiable(_backward)


class _QkNormRopeFn(torch.autograd.Function):
    """eager path: the same two calls without the dispatcher's cost"""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, table, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved)

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        # (a double backward raises; the wrapper that sees to it costs 10 us a call and matters only where a graph of the backward is asked for)
        if torch.is_grad_enabled():
            return _backward_once(ctx, dq_out, dk_out)
        return _backward(ctx, dq_out, dk_out)


def _check(q, k, q_weight, k_weight, table, positions):
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

    A training step can be captured.  As everywhere in torch, a captured backward() must not meet an eager graph of the same leaves that is still alive: free its
    outputs first, or take the gradients with torch.autograd.grad.
    """
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"qk_norm_rope: eps must be finite and >= 0 (got {eps})")
    if q.stride(-1) != 1 or k.stride(-1) != 1:
        q, k = q.contiguous(), k.contiguous()
    if positions is not None and positions.ndim and positions.stride(-1) != 1:
        positions = positions.contiguous()
    grad = torch.is_grad_enabled()
    if grad and table.requires_grad:
        raise ValueError("qk_norm_rope has no gradient for the table")
    if forward_ad._current_level >= 0:
        _native.refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight, table)
    if torch.compiler.is_compiling() or _native.dispatch_modes():
        _check(q, k, q_weight, k_weight, table, positions)
        return _op(q, k, q_weight, k_weight, table, positions, float(eps), bool(interleaved))
    if grad and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad) or (k_weight is not None and k_weight.requires_grad)):
        return _QkNormRopeFn.apply(q, k, q_weight, k_weight, table, positions, eps, interleaved)
    return _fwd_impl(q, k, q_weight, k_weight, table, positions, eps, interleaved)
