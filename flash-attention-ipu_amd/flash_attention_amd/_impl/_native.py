"""ctypes binding of libflash_attention.so (the C ABI declared in include/flash_attention_amd.h).

Library discovery follows the reference loader (flash_attention_ipu/__init__.py:4-23): first
`<pkg-parent>/build/libflash_attention.so`, then `<pkg-parent>/libflash_attention<EXT_SUFFIX>`;
`FLASH_ATTENTION_AMD_LIB` overrides both.  There is NO fallback: a missing library is an
ImportError at import time, and a GPU tensor can only be served by the HIP kernels in it.
"""

import ctypes
import os
import pathlib
import sysconfig

import torch
from torch.autograd import forward_ad

_LIB = None
_LIB_PATH = None

FA_DTYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
ABI_VERSION = 7


class FaPlan(ctypes.Structure):
    _fields_ = [
        ("kernel", ctypes.c_int32),
        ("block_q", ctypes.c_int32),
        ("block_kv", ctypes.c_int32),
        ("waves", ctypes.c_int32),
        ("chunk_q", ctypes.c_int32),
        ("chunk_kv", ctypes.c_int32),
        ("grid", ctypes.c_int64),
        ("lds_bytes", ctypes.c_int64),
        ("qb", ctypes.c_int32),
        ("sched", ctypes.c_int32),
        ("skipmax", ctypes.c_int32),
        ("source", ctypes.c_int32),
        ("pair", ctypes.c_int32),
        ("balanced", ctypes.c_int32),
        ("xs", ctypes.c_int32),
    ]


def candidate_paths():
    root = pathlib.Path(__file__).resolve().parent.parent.parent
    name = "libflash_attention.so"
    paths = []
    env = os.environ.get("FLASH_ATTENTION_AMD_LIB")
    if env:
        paths.append(pathlib.Path(env))
    paths.append(root / "build" / name)
    paths.append((root / name).with_suffix(sysconfig.get_config_vars().get("EXT_SUFFIX") or ".so"))
    return paths


def load_native_library():
    global _LIB, _LIB_PATH
    if _LIB is not None:
        return _LIB
    tried = candidate_paths()
    for path in tried:
        if path.exists():
            lib = ctypes.CDLL(str(path))
            _declare(lib)
            if lib.fa_abi_version() != ABI_VERSION:
                raise ImportError(f"{path}: ABI version {lib.fa_abi_version()} != {ABI_VERSION}")
            _LIB, _LIB_PATH = lib, path
            return lib
    raise ImportError(f"Cannot find libflash_attention.so - tried {[str(p) for p in tried]}")


def library_path():
    return _LIB_PATH


def _declare(lib):
    i32, i64, vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
    p64 = ctypes.POINTER(ctypes.c_int64)
    lib.fa_abi_version.restype = ctypes.c_int
    lib.fa_abi_version.argtypes = []
    lib.fa_last_error.restype = ctypes.c_char_p
    lib.fa_last_error.argtypes = []
    lib.fa_error_string.restype = ctypes.c_char_p
    lib.fa_error_string.argtypes = [ctypes.c_int]
    lib.fa_infer_output_shape.restype = ctypes.c_int
    lib.fa_infer_output_shape.argtypes = [p64, i32, p64]
    lib.fa_plan.restype = ctypes.c_int
    lib.fa_plan.argtypes = [i64, i64, i64, i32, i32, i32, ctypes.c_float, i32, ctypes.POINTER(FaPlan)]
    lib.fa_debug_set_option.restype = ctypes.c_int
    lib.fa_debug_set_option.argtypes = [ctypes.c_char_p, i32]
    lib.fa_debug_get_option.restype = ctypes.c_int
    lib.fa_debug_get_option.argtypes = [ctypes.c_char_p, ctypes.POINTER(i32)]
    lib.fa_fwd.restype = ctypes.c_int
    lib.fa_fwd.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, p64, p64, p64, p64,
                           i32, i32, i32, ctypes.c_float, i32, vp]
    lib.fa_bwd.restype = ctypes.c_int
    lib.fa_bwd.argtypes = [vp] * 10 + [i64, i64, i64, i64, i64, ctypes.POINTER(ctypes.c_int64 * 3), i32, ctypes.c_float, i32, vp]
    u64 = ctypes.c_uint64
    lib.fa_fwd_ex.restype = ctypes.c_int
    lib.fa_fwd_ex.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, p64, p64, p64, p64,
                              i32, i32, i32, ctypes.c_float, i32, vp, i32, p64, ctypes.c_float, u64, u64, vp, vp]
    lib.fa_bwd_ex.restype = ctypes.c_int
    lib.fa_bwd_ex.argtypes = [vp] * 10 + [i64, i64, i64, i64, i64, ctypes.POINTER(ctypes.c_int64 * 3), i32, ctypes.c_float, i32,
                                          vp, i32, p64, ctypes.c_float, u64, u64, vp, vp]
    lib.fa_probe_clock.restype = ctypes.c_int
    lib.fa_probe_clock.argtypes = [ctypes.c_void_p, i32, ctypes.c_void_p]
    lib.fa_probe_mfma_peak.restype = ctypes.c_double
    lib.fa_probe_mfma_peak.argtypes = [i32, i32, i32]
    lib.fa_fwd_qkv_packed.restype = ctypes.c_int
    lib.fa_fwd_qkv_packed.argtypes = [vp, vp, vp, i64, i64, i64, i32, i32, i32, vp]
    f32 = ctypes.c_float
    rope = [vp, i64, vp, i32, i64, i64, i64, i64, i64, i64, i64, vp, i32, f32, i32, vp]      # table .. stream
    lib.fa_qk_norm_rope_fwd.restype = ctypes.c_int
    lib.fa_qk_norm_rope_fwd.argtypes = [vp] * 6 + [i32] + rope
    lib.fa_qk_norm_rope_workspace.restype = i64
    lib.fa_qk_norm_rope_workspace.argtypes = [i64] * 5
    lib.fa_qk_norm_rope_bwd.restype = ctypes.c_int
    lib.fa_qk_norm_rope_bwd.argtypes = [vp] * 10 + [i32, vp, i64] + rope
    lib.fa_cache_tables.restype = ctypes.c_int
    lib.fa_cache_tables.argtypes = [vp, vp, vp, i64, i64, vp, i64, vp, i64, i64, i64] + [vp] * 7
    lib.fa_cache_append.restype = ctypes.c_int
    lib.fa_cache_append.argtypes = [vp] * 7 + [i64] * 6 + [vp, vp, i32, vp]
    lib.fa_cache_attn_workspace.restype = i64
    lib.fa_cache_attn_workspace.argtypes = [i64] * 8
    lib.fa_cache_attn.restype = ctypes.c_int
    lib.fa_cache_attn.argtypes = [vp] * 10 + [i64] * 12 + [vp, vp, i32, f32, vp]
    lib.fa_cache_attn_granted.restype = ctypes.c_int
    lib.fa_cache_attn_granted.argtypes = [vp] * 11 + [i64] * 12 + [vp, vp, i32, f32, vp]


def _raise(rc):
    lib = load_native_library()
    msg = lib.fa_last_error().decode() or lib.fa_error_string(rc).decode()
    if rc in (-2, -3, -4, -5, -7, -9, -11, -12, -14, -15):
        raise ValueError(f"flash_attention_amd: {msg}")
    raise RuntimeError(f"flash_attention_amd: {msg} (code {rc})")


def plan(G, L, D, dtype, num_chunks_q, num_chunks_kv, softmax_scale: float = 1.0, causal: bool = True) -> FaPlan:
    """The tile plan fa_fwd would launch for contiguous operands (same selection function, host only)."""
    lib = load_native_library()
    out = FaPlan()
    rc = lib.fa_plan(G, L, D, FA_DTYPE[dtype], num_chunks_q, num_chunks_kv, float(softmax_scale), int(bool(causal)),
                     ctypes.byref(out))
    if rc != 0:
        _raise(rc)
    return out


_KERNEL_CODE = {"auto": 0, "": 0, None: 0, "dma": ord("d"), "pipe": ord("p"), "pipe16": ord("x"), "kh": ord("h")}
_OPTION_AUTO = {"kernel": 0, "qb": 0, "waves": 0, "sched": 0, "skipmax": -1, "f32_generic": 0, "table": 1, "split": 0, "pair": -1,
                "balance": -1, "subsets": -1, "bsplit": -1, "bbal": -1}


def set_debug_option(name: str, value) -> None:
    """TEST / TUNING ONLY: fa_debug_set_option (kernel accepts 'dma' | 'pipe' | 'pipe16' | 'kh' | 'auto')."""
    lib = load_native_library()
    if name == "kernel" and not isinstance(value, int):
        value = _KERNEL_CODE[value]
    rc = lib.fa_debug_set_option(name.encode(), int(value))
    if rc != 0:
        _raise(rc)


def get_debug_option(name: str) -> int:
    lib = load_native_library()
    val = ctypes.c_int32(0)
    rc = lib.fa_debug_get_option(name.encode(), ctypes.byref(val))
    if rc != 0:
        _raise(rc)
    return val.value


class debug_options:
    """Context manager for tests and tuning tools: force knobs of the tile plan; on exit every knob is back at the value
    it had on entry (contexts nest).  Knobs not named keep their current value.

        with _native.debug_options(kernel="pipe", qb=2, waves=4): ...
    """

    def __init__(self, **knobs):
        unknown = set(knobs) - set(_OPTION_AUTO)
        if unknown:
            raise ValueError(f"unknown debug option(s) {sorted(unknown)}; known: {sorted(_OPTION_AUTO)}")
        self.knobs = {k: v for k, v in knobs.items() if v is not None}
        self.saved = {}

    def __enter__(self):
        self.saved = {k: get_debug_option(k) for k in self.knobs}
        for k, v in self.knobs.items():
            set_debug_option(k, v)
        return self

    def __exit__(self, *exc):
        for k, v in self.saved.items():
            set_debug_option(k, v)
        return False


def _strides3(arr):
    return (ctypes.c_int64 * 3)(*arr)


_I64x3 = ctypes.c_int64 * 3
_I64x24 = ctypes.c_int64 * 24
_P_I64x3 = ctypes.POINTER(ctypes.c_int64 * 3)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _on_device_of:
    """`with _on_device_of(t) as stream:` - the raw HIP stream PyTorch is enqueueing on for t's device, switching the
    current device only when it is not t's (the common single-device case costs two C calls, not a context manager
    and a Stream object: the Python side of a launch is ~10 us, which matters for small attention calls)."""

    __slots__ = ("idx", "prev")

    def __init__(self, t: torch.Tensor):
        self.idx = t.device.index
        self.prev = -1

    def __enter__(self):
        cur = torch.cuda.current_device()
        if self.idx is not None and cur != self.idx:
            self.prev = cur
            torch.cuda.set_device(self.idx)
        idx = cur if self.idx is None else self.idx
        if _raw_stream is not None:
            return _raw_stream(idx)
        return torch.cuda.current_stream(idx).cuda_stream

    def __exit__(self, *exc):
        if self.prev >= 0:
            torch.cuda.set_device(self.prev)
        return False


def fwd_packed(qkv: torch.Tensor, out: torch.Tensor, lse, num_chunks_q: int, num_chunks_kv: int):
    """qkv: contiguous CUDA [3,G,L,D]; out: contiguous [G,L,D]; lse: None or fp32 [G,L]."""
    lib = load_native_library()
    _, G, L, D = qkv.shape
    with _on_device_of(qkv) as stream:
        rc = lib.fa_fwd_qkv_packed(qkv.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
                                   G, L, D, num_chunks_q, num_chunks_kv, FA_DTYPE[qkv.dtype], stream)
    if rc != 0:
        _raise(rc)


def fwd_strided(q, k, v, out, lse, G, L, D, heads, qs, ks, vs, os_, num_chunks_q, num_chunks_kv, scale,
                causal: bool = True, heads_kv=None):
    """Strided three-view forward: see fa_fwd in include/flash_attention_amd.h."""
    lib = load_native_library()
    with _on_device_of(q) as stream:
        rc = lib.fa_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                        lse.data_ptr() if lse is not None else None, G, L, D, heads,
                        heads if heads_kv is None else heads_kv,
                        _strides3(qs), _strides3(ks), _strides3(vs), _strides3(os_),
                        num_chunks_q, num_chunks_kv, FA_DTYPE[q.dtype], float(scale), int(bool(causal)), stream)
    if rc != 0:
        _raise(rc)


def group_strides(t: torch.Tensor, heads: int):
    """(outer, inner, row) element strides of a [G, L, D] (heads == 1) or [B, H, L, D] tensor."""
    if t.ndim == 3:
        return (t.stride(0), 0, t.stride(1))
    return (t.stride(0), t.stride(1), t.stride(2))


def bwd(q, k, v, out, dout, lse, dq, dk, dv, G, L, D, heads, scale, causal: bool = True, heads_kv=None):
    """Backward through the C ABI (fa_bwd).  Tensors are [G,L,D] or [B,H,L,D] views with unit inner stride; with
    heads_kv < heads (grouped-query attention) k, v, dk, dv are [B,H_kv,L,D]."""
    lib = load_native_library()
    if q.ndim == 3:
        flat = [x for t in (q, k, v, out, dout, dq, dk, dv) for x in (t.stride(0), 0, t.stride(1))]
    else:
        flat = [x for t in (q, k, v, out, dout, dq, dk, dv) for x in (t.stride(0), t.stride(1), t.stride(2))]
    arr = _I64x24(*flat)        # laid out exactly as int64_t[8][3]
    dsum = torch.empty((G, L), dtype=torch.float32, device=q.device)
    with _on_device_of(q) as stream:
        rc = lib.fa_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(),
                        dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dsum.data_ptr(), G, L, D, heads,
                        heads if heads_kv is None else heads_kv,
                        ctypes.cast(arr, _P_I64x3), FA_DTYPE[q.dtype], float(scale), int(bool(causal)), stream)
    if rc != 0:
        _raise(rc)


# ---- the eager training path of the SDPA override ([B, H, L, D] views, any head / batch strides) -----------------------------------------
# A GPT-2-sized attention layer is ~25 us of forward and ~70 us of backward kernels; the Python in front of the two C calls used to cost more
# than that (168 us of host per forward + backward).  These two entry points do nothing per call that can be done
# once per distinct layout: the ctypes stride blocks are cached by the tensors' stride tuples (one `Tensor.stride()` per operand instead of
# three, no array construction), LSE and the backward's Dsum workspace are two halves of ONE fp32 allocation made by the forward (addressed
# by pointer arithmetic: no views), and the current device is consulted once.
_STRIDE_BLOCKS = {}


def _stride_block(key, n):
    """cached ctypes int64 block of the first three strides of each of the `n` stride tuples in `key`"""
    blk = _STRIDE_BLOCKS.get(key)
    if blk is None:
        if len(_STRIDE_BLOCKS) > 8192:      # (layouts per process are few; a pathological caller just rebuilds)
            _STRIDE_BLOCKS.clear()
        if n == 1:
            blk = _I64x3(*key[:3])
        else:
            arr = _I64x24(*[x for st in key for x in st[:3]])
            blk = (arr, ctypes.cast(arr, _P_I64x3))
        _STRIDE_BLOCKS[key] = blk
    return blk


def _stream_for(t: torch.Tensor):
    """(raw stream of t's device, previous device or -1): switches the current device only when it is not t's"""
    idx = t.device.index
    cur = torch.cuda.current_device()
    prev = -1
    if idx is not None and cur != idx:
        prev = cur
        torch.cuda.set_device(idx)
        cur = idx
    return (_raw_stream(cur) if _raw_stream is not None else torch.cuda.current_stream(cur).cuda_stream), prev


_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def stream_of(device: torch.device):
    """(raw stream of a device that holds tensors, device to go back to or -1): _stream_for without torch.cuda's initialisation checks"""
    idx, cur = device.index, _get_device()
    prev = -1
    if cur != idx:
        prev = cur
        torch.cuda.set_device(idx)
    return (_raw_stream(idx) if _raw_stream is not None else torch.cuda.current_stream(idx).cuda_stream), prev


# Eager calls pass the dispatcher by; one that is compiled (torch.compiler.is_compiling()) or that a dispatch mode looks on at, a tracer's among them, goes through its op.
dispatch_modes = torch._C._len_torch_dispatch_stack


def refuse_tangents(name, *tensors):
    """no forward-mode derivative here: a dual tensor would lose its tangent without a word (called inside of a forward-mode level only)"""
    if any(t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{name} has no forward-mode derivative")


def fwd_bhld(q, k, v, out, lse_ptr, num_chunks_q, num_chunks_kv, scale, causal):
    """fa_fwd on [B, H, L, D] views (k / v may carry fewer heads) with unit stride on D; lse_ptr: device address of [B * H, L] fp32 or None."""
    lib = _LIB or load_native_library()
    B, H, L, D = q.shape
    stream, prev = _stream_for(q)
    try:
        rc = lib.fa_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_ptr, B * H, L, D, H, k.shape[1],
                        _stride_block(q.stride(), 1), _stride_block(k.stride(), 1), _stride_block(v.stride(), 1), _stride_block(out.stride(), 1),
                        num_chunks_q, num_chunks_kv, FA_DTYPE[q.dtype], scale, 1 if causal else 0, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _raise(rc)


def bwd_bhld(q, k, v, out, dout, lse_ptr, dq, dk, dv, dsum_ptr, scale, causal):
    """fa_bwd on [B, H, L, D] views (k, v, dk, dv [B, H_kv, L, D]); lse_ptr / dsum_ptr: device addresses of two [B * H, L] fp32 blocks."""
    lib = _LIB or load_native_library()
    B, H, L, D = q.shape
    _, strides = _stride_block((q.stride(), k.stride(), v.stride(), out.stride(), dout.stride(), dq.stride(), dk.stride(), dv.stride()), 8)
    stream, prev = _stream_for(q)
    try:
        rc = lib.fa_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse_ptr, dq.data_ptr(), dk.data_ptr(),
                        dv.data_ptr(), dsum_ptr, B * H, L, D, H, k.shape[1], strides, FA_DTYPE[q.dtype], scale, 1 if causal else 0, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _raise(rc)


def bwd_packed(qkv, out, dout, lse_ptr, dqkv, dsum_ptr):
    """fa_bwd of the packed op: qkv / dqkv contiguous [3, G, L, D], out / dout contiguous [G, L, D]; q, k, v and their gradients are
    addressed inside the packed tensors by pointer arithmetic (no index views), the stride block is one cached entry per (L, D)."""
    lib = _LIB or load_native_library()
    _, G, L, D = qkv.shape
    st = (L * D, 0, D, 0)
    _, strides = _stride_block((st,) * 8, 8)
    step = G * L * D * qkv.element_size()
    p, dp = qkv.data_ptr(), dqkv.data_ptr()
    stream, prev = _stream_for(qkv)
    try:
        rc = lib.fa_bwd(p, p + step, p + 2 * step, out.data_ptr(), dout.data_ptr(), lse_ptr, dp, dp + step, dp + 2 * step, dsum_ptr,
                        G, L, D, 1, 1, strides, FA_DTYPE[qkv.dtype], 1.0, 1, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _raise(rc)


MASK_NONE, MASK_BOOL, MASK_BIAS = 0, 1, 2


def _mask_args(mask, q):
    """(pointer, kind, strides) of an attention mask already expanded to [B, H, L, L] (stride 0 = broadcast, unit stride on the
    key dimension): torch.bool -> boolean bytes, the operand dtype -> additive bias."""
    if mask is None:
        return None, MASK_NONE, None
    kind = MASK_BOOL if mask.dtype in (torch.bool, torch.uint8) else MASK_BIAS
    if kind == MASK_BIAS and mask.dtype != q.dtype:
        raise ValueError("a float attn_mask must have the dtype of the query")
    return mask.data_ptr(), kind, _strides3((mask.stride(0), mask.stride(1), mask.stride(2)))


_U64 = 2 ** 64 - 1


def _mask_args_cached(mask, q):
    """(pointer, kind, cached stride block) of a mask already expanded to [B, H, L, L] - _mask_args without the per-call ctypes array"""
    if mask is None:
        return None, MASK_NONE, None
    kind = MASK_BOOL if mask.dtype in (torch.bool, torch.uint8) else MASK_BIAS
    if kind == MASK_BIAS and mask.dtype != q.dtype:
        raise ValueError("a float attn_mask must have the dtype of the query")
    return mask.data_ptr(), kind, _stride_block(mask.stride(), 1)


def fwd_ex_bhld(q, k, v, out, lse_ptr, scale, causal, mask, dropout_p, seed, offset, state):
    """fa_fwd_ex on [B, H, L, D] views, the eager training path's lean form (cached stride blocks; lse_ptr: a device address or None)"""
    lib = _LIB or load_native_library()
    B, H, L, D = q.shape
    mptr, kind, mst = _mask_args_cached(mask, q)
    stream, prev = _stream_for(q)
    try:
        rc = lib.fa_fwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse_ptr, B * H, L, D, H, k.shape[1],
                           _stride_block(q.stride(), 1), _stride_block(k.stride(), 1), _stride_block(v.stride(), 1), _stride_block(out.stride(), 1),
                           1, 1, FA_DTYPE[q.dtype], scale, 1 if causal else 0, mptr, kind, mst, dropout_p, seed & _U64, offset & _U64,
                           state.data_ptr() if state is not None else None, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _raise(rc)


def bwd_ex_bhld(q, k, v, out, dout, lse_ptr, dq, dk, dv, dsum_ptr, scale, causal, mask, dropout_p, seed, offset, state):
    """fa_bwd_ex on [B, H, L, D] views (k, v, dk, dv [B, H_kv, L, D]), the eager training path's lean form"""
    lib = _LIB or load_native_library()
    B, H, L, D = q.shape
    _, strides = _stride_block((q.stride(), k.stride(), v.stride(), out.stride(), dout.stride(), dq.stride(), dk.stride(), dv.stride()), 8)
    mptr, kind, mst = _mask_args_cached(mask, q)
    stream, prev = _stream_for(q)
    try:
        rc = lib.fa_bwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse_ptr, dq.data_ptr(), dk.data_ptr(),
                           dv.data_ptr(), dsum_ptr, B * H, L, D, H, k.shape[1], strides, FA_DTYPE[q.dtype], scale, 1 if causal else 0,
                           mptr, kind, mst, dropout_p, seed & _U64, offset & _U64, state.data_ptr() if state is not None else None, stream)
    finally:
        if prev >= 0:
            torch.cuda.set_device(prev)
    if rc != 0:
        _raise(rc)


def fwd_ex(q, k, v, out, lse, L, D, scale, causal, mask, dropout_p, seed, offset, state=None):
    """fa_fwd_ex on [B, H, L, D] views (k, v may carry fewer heads); mask: None or a [B, H, L, L] view (see _mask_args);
    state: None or an int64 [2] DEVICE tensor {seed, offset} read by the kernels instead of the two integers (graph-safe dropout)."""
    lib = load_native_library()
    B, H = q.shape[0], q.shape[1]
    st = lambda t: _strides3((t.stride(0), t.stride(1), t.stride(2)))  # noqa: E731
    mptr, kind, mst = _mask_args(mask, q)
    with _on_device_of(q) as stream:
        rc = lib.fa_fwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
                           B * H, L, D, H, k.shape[1], st(q), st(k), st(v), st(out), 1, 1, FA_DTYPE[q.dtype], float(scale),
                           int(bool(causal)), mptr, kind, mst, float(dropout_p), int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 64 - 1),
                           state.data_ptr() if state is not None else None, stream)
    if rc != 0:
        _raise(rc)


def bwd_ex(q, k, v, out, dout, lse, dq, dk, dv, L, D, scale, causal, mask, dropout_p, seed, offset, state=None):
    """fa_bwd_ex on [B, H, L, D] views (k, v, dk, dv [B, H_kv, L, D])."""
    lib = load_native_library()
    B, H = q.shape[0], q.shape[1]
    flat = [x for t in (q, k, v, out, dout, dq, dk, dv) for x in (t.stride(0), t.stride(1), t.stride(2))]
    arr = _I64x24(*flat)
    dsum = torch.empty((B * H, L), dtype=torch.float32, device=q.device)
    mptr, kind, mst = _mask_args(mask, q)
    with _on_device_of(q) as stream:
        rc = lib.fa_bwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(),
                           dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dsum.data_ptr(), B * H, L, D, H, k.shape[1],
                           ctypes.cast(arr, _P_I64x3), FA_DTYPE[q.dtype], float(scale), int(bool(causal)),
                           mptr, kind, mst, float(dropout_p), int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 64 - 1),
                           state.data_ptr() if state is not None else None, stream)
    if rc != 0:
        _raise(rc)
