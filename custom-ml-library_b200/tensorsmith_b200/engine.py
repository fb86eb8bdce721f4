"""Array-level entry points of the B200 attention engine.

These functions take CUDA device arrays (torch tensors are used as the device
allocator and stream source; any strided 4-D view is accepted), fill the C-ABI
parameter structs of include/ts_attn.h and launch on the current stream.  They
allocate outputs and workspaces on the caller's side of the ABI, exactly as the
C contract requires, and never compute anything on the host.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
import struct
from typing import NamedTuple

import torch

from . import _lib

_DTYPE_CODES = {
    torch.float32: _lib.F32,
    torch.float16: _lib.F16,
    torch.bfloat16: _lib.BF16,
    torch.float64: _lib.F64,
}

# Largest (query heads per KV head) x (query tokens) the split-K decode kernel takes.
DECODE_MAX_ROWS = 8


def lse_dtype(dtype: torch.dtype) -> torch.dtype:
    """LSE is fp32 (softmax statistics of half/fp32 inputs), fp64 for fp64 inputs."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"the B200 attention engine does not support dtype {dtype}") from None


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("the B200 attention engine needs CUDA device tensors")


def view4(t: torch.Tensor) -> _lib.View4:
    if t.dim() != 4:
        raise ValueError("expected a [batch, heads, sequence, channels] view")
    return _lib.View4(t.data_ptr(), (ctypes.c_int64 * 4)(*t.stride()))


def _stream_handle(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# Calls that cost a few microseconds on the device pack their structs in one go (the layouts of _lib.AttnParams,
# _lib.Kv4Cache, _lib.PagePool and so on) instead of field by field.
_ATTN_STRUCT = struct.Struct("@" + "P4q" * 4 + "P3q" + "8i" + "d" + "iq" + "P" + "iP4q")
_VIEW_STRUCT = struct.Struct("@P4q")
_KV4_STRUCT = struct.Struct("@PqPq6i")
_POOL_STRUCT = struct.Struct("@Pqqqii")
_WINDOW_STRUCT = struct.Struct("@ii")
_TREE_STRUCT = struct.Struct("@Pqii")
_KEEP_STRUCT = struct.Struct("@PP4q4q8iPPPq")
_LOGPROB_STRUCT = struct.Struct("@Pq4iPqPPPPP")


def _packed_view(t) -> _lib.View4:
    return _lib.View4.from_buffer_copy(_VIEW_STRUCT.pack(t.data_ptr(), *t.stride()))


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


_SAME_DEVICE = contextlib.nullcontext()


def _on(index: int):
    """A context in which ``index`` is the current device, as the C ABI wants it."""
    return _SAME_DEVICE if torch.cuda.current_device() == index else torch.cuda.device(index)


def _one_device(first, *others) -> int:
    """The CUDA device that all the given tensors live on."""
    index = first.get_device()
    if index < 0 or any(t is not None and t.get_device() != index for t in others):
        raise ValueError("the B200 attention engine needs CUDA device tensors, all on one device")
    return index


def default_scale(head_dim: int) -> float:
    """1/sqrt(D), the reference default (nn/attention.py:60)."""
    return 1.0 / math.sqrt(head_dim)


def _mask_args(mask, shape, dtype):
    """Broadcast a bool / float mask to [B, H, Tq, Tk] strides (0 on broadcast axes).

    Additive masks are passed in the accumulation type (fp64 for fp64 inputs, else fp32)."""
    if mask is None:
        return _lib.MASK_NONE, None, (0, 0, 0, 0), None
    if mask.dtype == torch.bool:
        kind = _lib.MASK_BOOL
        keep = mask
    elif mask.is_floating_point():
        kind = _lib.MASK_ADD_F32
        acc = lse_dtype(dtype)
        keep = mask if mask.dtype == acc else mask.to(acc)
    else:
        raise TypeError("attention masks must be boolean or floating point")
    try:
        expanded = keep.expand(*shape)
    except RuntimeError as error:
        raise ValueError("attention mask is not broadcastable to [B,H,Q,K]") from error
    return kind, expanded.data_ptr(), tuple(expanded.stride()), keep


def make_params(q, k, v, o, lse, *, is_causal=False, scale=None, causal_offset=0, kv_lens=None,
                mask=None):
    """Fill ts_attn_params; returns (params, keepalive) -- keep the tuple alive until launch."""
    b, hq, tq, d = q.shape
    hkv, tk, dv = k.shape[1], k.shape[2], v.shape[3]
    p = _lib.AttnParams()
    p.q, p.k, p.v, p.o = view4(q), view4(k), view4(v), view4(o)
    p.lse = lse.data_ptr() if lse is not None else None
    if lse is not None:
        p.lse_stride = (ctypes.c_int64 * 3)(*lse.stride())
    p.dtype = dtype_code(q.dtype)
    p.batch, p.q_heads, p.kv_heads = b, hq, hkv
    p.q_len, p.kv_len, p.head_dim, p.value_dim = tq, tk, d, dv
    p.scale = default_scale(d) if scale is None else float(scale)
    p.is_causal = 1 if is_causal else 0
    p.causal_offset = int(causal_offset)
    lens = None
    if kv_lens is not None:
        lens = kv_lens if kv_lens.dtype == torch.int32 else kv_lens.to(torch.int32)
        p.kv_lens = lens.data_ptr()
    kind, ptr, strides, keep = _mask_args(mask, (b, hq, tq, tk), q.dtype)
    p.mask_kind = kind
    p.mask = ptr
    p.mask_stride = (ctypes.c_int64 * 4)(*strides)
    return p, (lens, keep)


def _check_inputs(q, k, v):
    _require_cuda(q, k, v)
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise TypeError("attention inputs must have the same floating-point dtype")
    dtype_code(q.dtype)


def fwd_path(q, k, v, *, decode=False, is_causal=False, scale=None, causal_offset=0, kv_lens=None,
             mask=None) -> str:
    """Name of the kernel family the engine selects for this problem."""
    o = torch.empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]), dtype=q.dtype, device=q.device)
    p, keep = make_params(q, k, v, o, None, is_causal=is_causal, scale=scale,
                          causal_offset=causal_offset, kv_lens=kv_lens, mask=mask)
    code = _lib.lib().ts_attn_fwd_path(ctypes.byref(p), 1 if decode else 0)
    if code < 0:
        _lib.check(code, "ts_attn_fwd_path")
    return _lib.PATH_NAMES[code]


def _dropout_struct(dropout) -> _lib.Dropout:
    p, seed, offset = dropout
    if not 0.0 <= float(p) < 1.0:
        raise ValueError("dropout probability must be in [0, 1)")
    return _lib.Dropout(float(p), int(seed) & (2**64 - 1), int(offset) & (2**64 - 1))


def _window_struct(window, sinks, is_causal, mask, dropout) -> bytes:
    """The checked window of a call as a packed ts_window, or raises."""
    if window < 1 or sinks < 0 or max(window, sinks) >= 2**31:
        raise ValueError("a window must be positive and the number of sinks must not be negative")
    if not is_causal:
        raise ValueError("a sliding window needs is_causal")
    if mask is not None or dropout is not None:
        raise ValueError("a sliding window takes neither an explicit mask nor dropout")
    return _WINDOW_STRUCT.pack(window, sinks)


def _window_params(q, k, v, o, lse, scale, causal_offset, kv_lens) -> tuple:
    """(packed ts_attn_params of a causal problem, what must outlive the call)."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or o.dim() != 4:
        raise ValueError("expected a [batch, heads, sequence, channels] view")
    b, hq, tq, d = q.shape
    hkv, tk = k.shape[1], k.shape[2]
    if k.shape != (b, hkv, tk, d) or v.shape[:3] != (b, hkv, tk) or o.shape != (b, hq, tq, v.shape[3]):
        raise ValueError("query, key, value and output shapes do not match")
    if o.dtype != q.dtype:
        raise TypeError("the output must have the dtype of the inputs")
    if kv_lens is not None and kv_lens.dtype != torch.int32:
        kv_lens = kv_lens.to(torch.int32)
    if kv_lens is not None and (kv_lens.shape != (b,) or not kv_lens.is_contiguous() or not kv_lens.is_cuda):
        raise ValueError("kv_lens must be one length a row, on the device")
    if lse is not None and (lse.shape != (b, hq, tq) or lse.dtype != lse_dtype(q.dtype)):
        raise ValueError("lse must be [B, Hq, T], fp32 (fp64 for fp64 inputs)")
    return _ATTN_STRUCT.pack(
        q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), o.data_ptr(), *o.stride(),
        *((0, 0, 0, 0) if lse is None else (lse.data_ptr(), *lse.stride())), dtype_code(q.dtype), b, hq, hkv, tq, tk, d,
        v.shape[3], default_scale(d) if scale is None else float(scale), 1, int(causal_offset),
        0 if kv_lens is None else kv_lens.data_ptr(), _lib.MASK_NONE, 0, 0, 0, 0, 0), kv_lens


def _no_window(sinks) -> None:
    if sinks:
        raise ValueError("sinks need a window")


def window_path(q, k, v, *, window, sinks=0, causal_offset=0, scale=None, kv_lens=None) -> str:
    """Name of the kernel family that ``forward`` and ``backward`` select under a window."""
    w = _window_struct(window, sinks, True, None, None)
    o = torch.empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]), dtype=q.dtype, device=q.device)
    p, keep = _window_params(q, k, v, o, None, scale, causal_offset, kv_lens)
    code = _lib.lib().ts_attn_window_path(p, w)
    if code < 0:
        _lib.check(code, "ts_attn_window_path")
    return _lib.PATH_NAMES[code]


def forward(q, k, v, *, is_causal=False, scale=None, causal_offset=0, kv_lens=None, mask=None,
            need_lse=True, out=None, lse=None, dropout=None, window=None, sinks=0):
    """Attention forward: returns ``(out [B,Hq,Tq,Dv], lse [B,Hq,Tq] or None)``.

    ``window`` (with ``is_causal``): a query at position i sees the keys j <= i with i - j < window or j < ``sinks``.
    Pass both to ``backward``.

    ``lse`` is fp32 (fp64 for fp64 inputs), natural-log units, -inf on fully masked rows.
    ``dropout = (p, seed, offset)`` applies attention dropout (ts_attn_fwd_dropout); pass
    the same tuple to ``backward``."""
    _check_inputs(q, k, v)
    b, hq, tq, _ = q.shape
    if out is None:
        out = torch.empty((b, hq, tq, v.shape[3]), dtype=q.dtype, device=q.device)
    if need_lse and lse is None:
        lse = torch.empty((b, hq, tq), dtype=lse_dtype(q.dtype), device=q.device)
    if window is not None:
        w = _window_struct(window, sinks, is_causal, mask, dropout)
        index = _one_device(q, k, v, out, lse if need_lse else None, kv_lens)
        p, keep = _window_params(q, k, v, out, lse if need_lse else None, scale, causal_offset, kv_lens)
        handle = _lib.lib()
        with _on(index):
            need = handle.ts_attn_fwd_window_workspace_size(p, w)
            ws = q.new_empty((need,), dtype=torch.uint8) if need else None
            status = handle.ts_attn_fwd_window(p, w, ws.data_ptr() if need else None, need, _raw_stream(index))
        if status:
            _lib.check(status, "ts_attn_fwd_window")
        return out, (lse if need_lse else None)
    p, keep = make_params(q, k, v, out, lse if need_lse else None, is_causal=is_causal, scale=scale,
                          causal_offset=causal_offset, kv_lens=kv_lens, mask=mask)
    _no_window(sinks)
    if dropout is not None:
        d = _dropout_struct(dropout)
        _lib.check(_lib.lib().ts_attn_fwd_dropout(ctypes.byref(p), ctypes.byref(d), _stream_handle(q.device)),
                   "ts_attn_fwd_dropout")
    else:
        _lib.check(_lib.lib().ts_attn_fwd(ctypes.byref(p), _stream_handle(q.device)), "ts_attn_fwd")
    del keep
    return out, (lse if need_lse else None)


def decode_workspace_bytes(q, k, v, **kw) -> int:
    o = torch.empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]), dtype=q.dtype, device=q.device)
    p, keep = make_params(q, k, v, o, None, **kw)
    return int(_lib.lib().ts_attn_decode_workspace_size(ctypes.byref(p)))


def decode(q, k, v, *, is_causal=True, scale=None, causal_offset=0, kv_lens=None, mask=None,
           need_lse=False, out=None, lse=None, workspace=None):
    """Split-K decode for a few query tokens against a long KV cache."""
    _check_inputs(q, k, v)
    b, hq, tq, _ = q.shape
    if out is None:
        out = torch.empty((b, hq, tq, v.shape[3]), dtype=q.dtype, device=q.device)
    if need_lse and lse is None:
        lse = torch.empty((b, hq, tq), dtype=lse_dtype(q.dtype), device=q.device)
    p, keep = make_params(q, k, v, out, lse if need_lse else None, is_causal=is_causal, scale=scale,
                          causal_offset=causal_offset, kv_lens=kv_lens, mask=mask)
    handle = _lib.lib()
    need = int(handle.ts_attn_decode_workspace_size(ctypes.byref(p)))
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if (need and workspace is not None) else None
    ws_bytes = workspace.numel() * workspace.element_size() if (need and workspace is not None) else 0
    _lib.check(handle.ts_attn_decode(ctypes.byref(p), ws_ptr, ws_bytes, _stream_handle(q.device)),
               "ts_attn_decode")
    del keep
    return out, (lse if need_lse else None)


def decode_noalloc(q, k, v, *, is_causal=True, scale=None, causal_offset=0, kv_lens=None,
                   need_lse=False, out=None, lse=None):
    """Decode through ts_attn_decode_noalloc: no workspace, no device allocation by the engine.

    For callers that cannot allocate device memory at decode time (all HBM
    already handed to KV-cache pages, or no cudaMalloc allowed between decode
    steps).  The split partials go to the library's fixed 8 MiB per-device
    scratch; calls that overlap on one device race on it.  Pass ``out`` (and
    ``lse`` when ``need_lse``) preallocated to keep the call allocation-free."""
    _check_inputs(q, k, v)
    b, hq, tq, _ = q.shape
    if out is None:
        out = torch.empty((b, hq, tq, v.shape[3]), dtype=q.dtype, device=q.device)
    if need_lse and lse is None:
        lse = torch.empty((b, hq, tq), dtype=lse_dtype(q.dtype), device=q.device)
    p, keep = make_params(q, k, v, out, lse if need_lse else None, is_causal=is_causal, scale=scale,
                          causal_offset=causal_offset, kv_lens=kv_lens)
    status = _lib.lib().ts_attn_decode_noalloc(ctypes.byref(p), _stream_handle(q.device))
    if status == _lib.ERR_WORKSPACE:
        raise _lib.EngineError(status, "ts_attn_decode_noalloc: problem needs more than the fixed "
                               f"{_lib.NOALLOC_SCRATCH_BYTES >> 20} MiB decode scratch")
    _lib.check(status, "ts_attn_decode_noalloc")
    del keep
    return out, (lse if need_lse else None)


def _bwd_params(q, k, v, out, lse, dout, dq, dk, dv, **kw):
    fp, keep = make_params(q, k, v, out, lse, **kw)
    bp = _lib.AttnBwdParams()
    bp.fwd = fp
    bp.dout, bp.dq, bp.dk, bp.dv = view4(dout), view4(dq), view4(dk), view4(dv)
    return bp, keep


def bwd_path(q, k, v, out, lse, dout, **kw) -> str:
    """Name of the kernel family ts_attn_bwd selects for this problem."""
    bp, keep = _bwd_params(q, k, v, out, lse, dout, torch.empty_like(q), torch.empty_like(k),
                           torch.empty_like(v), **kw)
    code = _lib.lib().ts_attn_bwd_path(ctypes.byref(bp))
    if code < 0:
        _lib.check(code, "ts_attn_bwd_path")
    return _lib.PATH_NAMES[code]


def backward(q, k, v, out, lse, dout, *, is_causal=False, scale=None, causal_offset=0, kv_lens=None,
             mask=None, dq=None, dk=None, dv=None, dropout=None, window=None, sinks=0):
    """dQ, dK, dV of attention from the forward output and its LSE (``dropout``, ``window`` and ``sinks`` as given
    to the forward)."""
    _check_inputs(q, k, v)
    _require_cuda(out, lse, dout)
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    if dout.dtype != q.dtype:
        dout = dout.to(q.dtype)
    if window is not None:
        w = _window_struct(window, sinks, is_causal, mask, dropout)
        index = _one_device(q, k, v, out, lse, dout, dq, dk, dv, kv_lens)
        p, keep = _window_params(q, k, v, out, lse, scale, causal_offset, kv_lens)
        if dout.shape != out.shape or dq.shape != q.shape or dk.shape != k.shape or dv.shape != v.shape:
            raise ValueError("gradients must have the shapes of what they belong to")
        if dq.dtype != q.dtype or dk.dtype != q.dtype or dv.dtype != q.dtype:
            raise TypeError("gradients must have the dtype of the inputs")
        p += b"".join(_VIEW_STRUCT.pack(t.data_ptr(), *t.stride()) for t in (dout, dq, dk, dv))
        handle = _lib.lib()
        with _on(index):
            need = handle.ts_attn_bwd_window_workspace_size(p, w)
            ws = q.new_empty((max(need, 16),), dtype=torch.uint8)
            status = handle.ts_attn_bwd_window(p, w, ws.data_ptr(), ws.numel(), _raw_stream(index))
        if status:
            _lib.check(status, "ts_attn_bwd_window")
        return dq, dk, dv
    bp, keep = _bwd_params(q, k, v, out, lse, dout, dq, dk, dv, is_causal=is_causal, scale=scale,
                           causal_offset=causal_offset, kv_lens=kv_lens, mask=mask)
    handle = _lib.lib()
    _no_window(sinks)
    if dropout is not None:
        d = _dropout_struct(dropout)
        need = int(handle.ts_attn_bwd_dropout_workspace_size(ctypes.byref(bp)))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
        _lib.check(handle.ts_attn_bwd_dropout(ctypes.byref(bp), ctypes.byref(d), ws.data_ptr(), ws.numel(),
                                              _stream_handle(q.device)), "ts_attn_bwd_dropout")
        del keep
        return dq, dk, dv
    need = int(handle.ts_attn_bwd_workspace_size(ctypes.byref(bp)))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    _lib.check(handle.ts_attn_bwd(ctypes.byref(bp), ws.data_ptr(), ws.numel(), _stream_handle(q.device)),
               "ts_attn_bwd")
    del keep
    return dq, dk, dv


def dropout_mask(batch, heads, q_len, kv_len, dropout, device) -> torch.Tensor:
    """The uint8 keep mask [B, Hq, Tq, Tk] that ``dropout = (p, seed, offset)`` applies."""
    d = _dropout_struct(dropout)
    mask = torch.empty((batch, heads, q_len, kv_len), dtype=torch.uint8, device=device)
    _lib.check(_lib.lib().ts_attn_dropout_mask(ctypes.byref(d), batch, heads, q_len, kv_len, mask.data_ptr(),
                                               _stream_handle(mask.device)), "ts_attn_dropout_mask")
    return mask


class _DropoutGenerator:
    """(seed, offset) source for attention dropout: ``seed()`` resets it, every draw
    takes the next offset (the counter that keeps calls' masks independent)."""

    def __init__(self):
        self.seed_value = int(torch.initial_seed()) & (2**64 - 1)
        self.offset = 0

    def seed(self, value: int) -> None:
        self.seed_value = int(value) & (2**64 - 1)
        self.offset = 0

    def draw(self, p: float) -> tuple:
        args = (float(p), self.seed_value, self.offset)
        self.offset += 1
        return args


DROPOUT_GENERATOR = _DropoutGenerator()


def seed(value: int) -> None:
    """Seed the attention-dropout generator (tensorsmith's ``ts.seed``, device.py:226-232)."""
    DROPOUT_GENERATOR.seed(value)


def kv_append(key, value, key_cache, value_cache, *, position=0, positions=None, positions_out=None):
    """Write a [B,H,steps,C] chunk into [B,H,cap,C] caches at ``position`` (or per-row ``positions``)."""
    _require_cuda(key, value, key_cache, value_cache)
    p = _lib.KvAppendParams()
    p.key, p.value = view4(key), view4(value)
    p.key_cache, p.value_cache = view4(key_cache), view4(value_cache)
    p.src_dtype = dtype_code(key.dtype)
    p.cache_dtype = dtype_code(key_cache.dtype)
    if value.dtype != key.dtype or value_cache.dtype != key_cache.dtype:
        raise TypeError("key/value and their caches must share a dtype each")
    p.batch, p.heads, p.steps = key.shape[0], key.shape[1], key.shape[2]
    p.head_dim, p.value_dim, p.capacity = key.shape[3], value.shape[3], key_cache.shape[2]
    p.position = int(position)
    p.positions = positions.data_ptr() if positions is not None else None
    p.positions_out = positions_out.data_ptr() if positions_out is not None else None
    _lib.check(_lib.lib().ts_kv_append(ctypes.byref(p), _stream_handle(key.device)), "ts_kv_append")


def _storage_code(dtype: torch.dtype) -> int:
    return _lib.I8 if dtype == torch.int8 else dtype_code(dtype)


def kv_reorder(src, dst, index, length):
    """dst[b, :, :length] = src[index[b], :, :length] (beam reorder; int8 storage too)."""
    _require_cuda(src, dst, index)
    idx = index if index.dtype == torch.int32 else index.to(torch.int32)
    _lib.check(
        _lib.lib().ts_kv_reorder(view4(src), view4(dst), _storage_code(src.dtype), src.shape[0],
                                 src.shape[1], int(length), src.shape[3], idx.data_ptr(),
                                 _stream_handle(src.device)),
        "ts_kv_reorder",
    )


def _check_int8_cache(cache, scales):
    if cache.dtype != torch.int8 or cache.dim() != 4:
        raise TypeError("int8 cache storage must be an int8 [B, H, capacity, C] tensor")
    if scales.dtype != torch.float32 or not scales.is_contiguous() or scales.numel() != cache.shape[0] * cache.shape[1] * cache.shape[2]:
        raise ValueError("int8 cache scales must be contiguous fp32 [B, H, capacity(, 1)]")


def kv_append_int8(key, value, key_cache, value_cache, key_scales, value_scales, *, compute_dtype,
                   position=0, positions=None, positions_out=None):
    """Quantising append (nn/cache.py:70-82): rows rounded to ``compute_dtype``, then
    symmetric int8 with one fp32 scale per (row, head, token) written to the scale arrays."""
    _require_cuda(key, value, key_cache, value_cache, key_scales, value_scales)
    _check_int8_cache(key_cache, key_scales)
    _check_int8_cache(value_cache, value_scales)
    if value.dtype != key.dtype:
        raise TypeError("key/value must share a dtype")
    p = _lib.KvAppendParams()
    p.key, p.value = view4(key), view4(value)
    p.key_cache, p.value_cache = view4(key_cache), view4(value_cache)
    p.src_dtype = dtype_code(key.dtype)
    p.cache_dtype = dtype_code(compute_dtype)
    p.batch, p.heads, p.steps = key.shape[0], key.shape[1], key.shape[2]
    p.head_dim, p.value_dim, p.capacity = key.shape[3], value.shape[3], key_cache.shape[2]
    p.position = int(position)
    p.positions = positions.data_ptr() if positions is not None else None
    p.positions_out = positions_out.data_ptr() if positions_out is not None else None
    _lib.check(_lib.lib().ts_kv_append_int8(ctypes.byref(p), key_scales.data_ptr(), value_scales.data_ptr(),
                                            _stream_handle(key.device)), "ts_kv_append_int8")


def kv_dequant_int8(src, scales, out, length):
    """out[:, :, :length] = dtype(float(src) * scale) for an int8 cache (nn/cache.py:91-99)."""
    _require_cuda(src, scales, out)
    _check_int8_cache(src, scales)
    _lib.check(
        _lib.lib().ts_kv_dequant_int8(view4(src), scales.data_ptr(), src.shape[2], view4(out),
                                      dtype_code(out.dtype), src.shape[0], src.shape[1], int(length),
                                      src.shape[3], _stream_handle(src.device)),
        "ts_kv_dequant_int8",
    )


def _int8_params(q, k8, v8, out, lse, kw):
    _require_cuda(q, k8, v8)
    if k8.dtype != torch.int8 or v8.dtype != torch.int8:
        raise TypeError("int8 decode expects int8 key/value storage")
    dtype_code(q.dtype)
    return make_params(q, k8, v8, out, lse, **kw)


def decode_int8_workspace_bytes(q, k8, v8, **kw) -> int:
    o = torch.empty((q.shape[0], q.shape[1], q.shape[2], v8.shape[3]), dtype=q.dtype, device=q.device)
    p, keep = _int8_params(q, k8, v8, o, None, kw)
    return int(_lib.lib().ts_attn_decode_int8_workspace_size(ctypes.byref(p)))


def decode_int8(q, k8, v8, key_scales, value_scales, *, is_causal=True, scale=None, causal_offset=0,
                kv_lens=None, need_lse=False, out=None, lse=None, workspace=None):
    """Split-K decode reading an int8 cache directly (dequantisation fused into the scores
    and the P.V sum).  ``k8``/``v8`` are the first ``kv_len`` positions of the int8 storage;
    ``key_scales``/``value_scales`` the full contiguous [B, H, capacity] scale arrays."""
    _require_cuda(key_scales, value_scales)
    b, hq, tq, _ = q.shape
    if out is None:
        out = torch.empty((b, hq, tq, v8.shape[3]), dtype=q.dtype, device=q.device)
    if need_lse and lse is None:
        lse = torch.empty((b, hq, tq), dtype=lse_dtype(q.dtype), device=q.device)
    kw = dict(is_causal=is_causal, scale=scale, causal_offset=causal_offset, kv_lens=kv_lens)
    p, keep = _int8_params(q, k8, v8, out, lse if need_lse else None, kw)
    cap = key_scales.numel() // (k8.shape[0] * k8.shape[1])
    if (key_scales.dtype != torch.float32 or value_scales.dtype != torch.float32 or not key_scales.is_contiguous()
            or not value_scales.is_contiguous() or value_scales.numel() != key_scales.numel()):
        raise ValueError("int8 cache scales must be contiguous fp32 [B, H, capacity(, 1)]")
    handle = _lib.lib()
    need = int(handle.ts_attn_decode_int8_workspace_size(ctypes.byref(p)))
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if (need and workspace is not None) else None
    ws_bytes = workspace.numel() * workspace.element_size() if (need and workspace is not None) else 0
    _lib.check(handle.ts_attn_decode_int8(ctypes.byref(p), key_scales.data_ptr(), value_scales.data_ptr(), cap,
                                          ws_ptr, ws_bytes, _stream_handle(q.device)), "ts_attn_decode_int8")
    del keep
    return out, (lse if need_lse else None)


# -- the paged 4-bit cache ----------------------------------------------------


def int4_block_bytes(head_dim: int, page_size: int) -> int:
    """Bytes of one page and KV head, keys and values: 4.5 bits a value (ts_kv4_block_bytes)."""
    if head_dim <= 0 or head_dim > 256 or head_dim % 32 or page_size not in (16, 32, 64):
        raise ValueError("a 4-bit cache takes head dimensions that are multiples of 32 up to 256 and pages of "
                         "16, 32 or 64 tokens")
    return page_size * head_dim * 9 // 8


def int4_pool(num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, layers: int | None = None,
              device="cuda") -> torch.Tensor:
    """An empty pool: uint8 [num_pages, kv_heads, block], or [layers, num_pages, kv_heads, block]."""
    shape = (num_pages, kv_heads, int4_block_bytes(head_dim, page_size))
    if min(num_pages, kv_heads) <= 0 or (layers is not None and layers <= 0):
        raise ValueError("a pool needs at least one page, head and layer")
    return torch.empty(shape if layers is None else (layers,) + shape, dtype=torch.uint8, device=device)


def _int32_vector(t, name: str, size: int, index: int) -> int:
    if t.dtype != torch.int32 or t.get_device() != index or t.shape != (size,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of {size} on the pool's device")
    return t.data_ptr()


def _page_table(t, index: int, *, written: bool = False) -> tuple:
    """(pointer, stride, rows, slots) of a page table; rows that are ``written`` must not share entries."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.get_device() != index or t.stride(1) != 1 or 0 in t.shape:
        raise ValueError("a page table must be int32 [rows, slots] with contiguous rows on the pool's device")
    rows, slots = t.shape
    if written and rows > 1 and t.stride(0) < slots:
        raise ValueError("the rows of a page table that is written to must not overlap")
    return t.data_ptr(), t.stride(0), rows, slots


def _workspace(given, need: int, like):
    """``given`` where it holds ``need`` bytes, else as many new ones on the device of ``like``."""
    if given is None or given.numel() * given.element_size() < need:
        return like.new_empty((need,), dtype=torch.uint8)
    if given.get_device() != like.get_device() or not given.is_contiguous():
        raise ValueError("a workspace must be contiguous, on the pool's device")
    return given


class _Int4Cache:
    """A checked pool with its page table: the packed ts_kv4_cache and the sizes the callers need."""

    __slots__ = ("index", "rows", "slots", "heads", "packed")

    def __init__(self, pool, page_table, page_size: int, head_dim: int):
        if pool.dtype != torch.uint8 or pool.dim() != 3:
            raise TypeError("a 4-bit pool must be uint8 [pages, kv heads, block]")
        self.index = pool.get_device()
        if self.index < 0:
            raise ValueError("the B200 attention engine needs CUDA device tensors")
        pages, self.heads, block = pool.shape
        stride = pool.stride()
        if block != int4_block_bytes(head_dim, page_size) or stride[2] != 1 or stride[1] != block:
            raise ValueError("the pool's blocks do not match the head dimension and page size")
        table, table_stride, self.rows, self.slots = _page_table(page_table, self.index)
        self.packed = _KV4_STRUCT.pack(pool.data_ptr(), stride[0], table, table_stride, self.rows, self.slots, pages,
                                       self.heads, head_dim, page_size)


def kv_append_int4(key, value, pool, page_table, *, page_size, position=0, positions=None, positions_out=None):
    """Quantise a [B, Hkv, steps, D] chunk into the pages of its rows, at token ``position`` (or per-row
    ``positions``).  ``positions_out``, another vector, receives where the rows then end.  The table must hold a page
    for every token written (``kv_pages_reserve``)."""
    if key.dim() != 4:
        raise ValueError("key must be [rows, kv heads, tokens, head dimension] of the cache")
    rows, heads, steps, dim = key.shape
    cache = _Int4Cache(pool, page_table, page_size, dim)
    if rows != cache.rows or heads != cache.heads:
        raise ValueError("key must be [rows, kv heads, tokens, head dimension] of the cache")
    if value.shape != key.shape or key.get_device() != cache.index or value.get_device() != cache.index:
        raise ValueError("key and value must have the same shape, on the pool's device")
    if value.dtype != key.dtype:
        raise TypeError("key/value must share a dtype")
    status = _lib.lib().ts_kv_append_int4(
        _packed_view(key), _packed_view(value), dtype_code(key.dtype), steps, cache.packed, int(position),
        None if positions is None else _int32_vector(positions, "positions", rows, cache.index),
        None if positions_out is None else _int32_vector(positions_out, "positions_out", rows, cache.index),
        _raw_stream(cache.index))
    if status:
        _lib.check(status, "ts_kv_append_int4")


def kv_gather_int4(pool, page_table, length, *, page_size, dtype, starts=None, kv_lens=None):
    """The cached values of ``length`` tokens of every row, from token ``starts[b]`` (default 0): dequantised
    ``(keys, values)`` [B, Hkv, length, D] of ``dtype``; tokens at or past ``kv_lens[b]`` (optional) are zero."""
    head_dim = pool.shape[-1] * 8 // (9 * page_size) if page_size > 0 else 0
    cache = _Int4Cache(pool, page_table, page_size, head_dim)
    code, length = dtype_code(dtype), int(length)
    if length < 0:
        raise ValueError("length must not be negative")
    rows = cache.rows
    starts = None if starts is None else _int32_vector(starts, "starts", rows, cache.index)
    kv_lens = None if kv_lens is None else _int32_vector(kv_lens, "kv_lens", rows, cache.index)
    both = pool.new_empty((2, rows, cache.heads, length, head_dim), dtype=dtype)
    key, value = both.unbind(0)
    if length:
        status = _lib.lib().ts_kv_gather_int4(cache.packed, starts, kv_lens, _packed_view(key), _packed_view(value), code,
                                              length, _raw_stream(cache.index))
        if status:
            _lib.check(status, "ts_kv_gather_int4")
    return key, value


def _int4_attn_args(q, pool, page_table, kv_lens, page_size, max_len, is_causal, scale, out, lse):
    """(cache, packed ts_attn_params) of an attention_int4 call after its checks."""
    if q.dim() != 4:
        raise ValueError("expected a [batch, heads, sequence, channels] view")
    rows, heads, tokens, dim = q.shape
    cache = _Int4Cache(pool, page_table, page_size, dim)
    if q.get_device() != cache.index or rows != cache.rows or heads % cache.heads or heads * tokens == 0:
        raise ValueError("query rows and heads must match the cache, on its device")
    lens = _int32_vector(kv_lens, "kv_lens", rows, cache.index)
    whole = cache.slots * page_size
    max_len = whole if max_len is None else int(max_len)
    if not 0 <= max_len <= whole:
        raise ValueError("max_len must be between zero and the tokens the page table can hold")
    if lse is None:
        lse = (0, 0, 0, 0)
    elif lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.get_device() != cache.index:
        raise ValueError("lse must be fp32 [B, Hq, Tq] on the query's device")
    else:
        lse = (lse.data_ptr(), *lse.stride())
    if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != cache.index:
        raise ValueError("out must have the query's shape, dtype and device")
    none = (0, 0, 0, 0, 0)
    return cache, _ATTN_STRUCT.pack(q.data_ptr(), *q.stride(), *none, *none, out.data_ptr(), *out.stride(), *lse,
                                    dtype_code(q.dtype), rows, heads, cache.heads, tokens, max(1, max_len), dim, dim,
                                    default_scale(dim) if scale is None else float(scale), 1 if is_causal else 0, 0,
                                    lens, 0, *none)


def attention_int4_path(q, pool, page_table, kv_lens, *, page_size, max_len=None, is_causal=True, scale=None) -> str:
    """Name of the kernel family ``attention_int4`` selects: "decode" (straight over the pages) or "tcgen05"."""
    cache, params = _int4_attn_args(q, pool, page_table, kv_lens, page_size, max_len, is_causal, scale, q, None)
    code = _lib.lib().ts_attn_int4_path(params, cache.packed)
    if code < 0:
        _lib.check(code, "ts_attn_int4_path")
    return _lib.PATH_NAMES[code]


def attention_int4_workspace_bytes(q, pool, page_table, kv_lens, *, page_size, max_len=None, is_causal=True,
                                   scale=None) -> int:
    """Bytes of the ``workspace`` that ``attention_int4`` needs for these arguments."""
    cache, params = _int4_attn_args(q, pool, page_table, kv_lens, page_size, max_len, is_causal, scale, q, None)
    return int(_lib.lib().ts_attn_int4_workspace_size(params, cache.packed))


def attention_int4(q, pool, page_table, kv_lens, *, page_size, max_len=None, is_causal=True, scale=None,
                   need_lse=False, out=None, lse=None, workspace=None):
    """Attention of ``q`` [B, Hq, Tq, D] over a paged 4-bit cache: ``(out, lse or None)``.

    Row b sees its first ``kv_lens[b]`` tokens; with ``is_causal`` its Tq queries are the last of them
    (a row without a visible key gives zeros and an LSE of -inf).  ``max_len`` bounds ``kv_lens`` (default: what
    the table can hold); the work is split for it, so pass the real bound where it is known.  Chunks of a prompt may
    run on the prefill kernel (``attention_int4_path``), whose probabilities are rounded to q's type, where the
    kernel over the pages keeps 11 bits of them for bf16 and 22 for fp16 and fp32."""
    if out is None:
        out = q.new_empty(q.shape)
    if not need_lse:
        lse = None
    elif lse is None:
        lse = q.new_empty(q.shape[:3], dtype=torch.float32)
    cache, params = _int4_attn_args(q, pool, page_table, kv_lens, page_size, max_len, is_causal, scale, out, lse)
    handle = _lib.lib()
    need = handle.ts_attn_int4_workspace_size(params, cache.packed)
    if need:
        workspace = _workspace(workspace, need, pool)
    status = handle.ts_attn_int4(params, cache.packed, workspace.data_ptr() if need else None, need,
                                 _raw_stream(cache.index))
    if status:
        _lib.check(status, "ts_attn_int4")
    return out, lse


# -- drafted tokens over a cache -----------------------------------------------


def check_tree(parents, rows: int, nodes: int, index: int) -> None:
    """Raises unless ``parents`` are those of ``attention_tree`` for ``rows`` trees of ``nodes`` on device ``index``."""
    if parents.dtype != torch.int32 or parents.shape != (rows, nodes) or parents.get_device() != index or (
            parents.stride(1) != 1 and nodes > 1):
        raise ValueError("parents must be int32 [batch, nodes] with contiguous rows on the query's device")
    if nodes > _lib.TREE_MAX_NODES:
        raise ValueError(f"a tree has at most {_lib.TREE_MAX_NODES} nodes")


def _tree_args(q, k, v, kv_lens, parents, window, sinks, scale, out, lse):
    """(packed ts_attn_params, packed ts_tree, device index) of an attention_tree call after its checks."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("expected [batch, heads, sequence, channels] views")
    index = q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index:
        raise ValueError("the B200 attention engine needs CUDA device tensors, all on one device")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise TypeError("attention inputs must have the same floating-point dtype")
    code = dtype_code(q.dtype)
    rows, heads, nodes, dim = q.shape
    kv_heads, capacity, value_dim = v.shape[1:]
    if k.shape != (rows, kv_heads, capacity, dim) or v.shape[0] != rows:
        raise ValueError("query, key and value shapes do not match")
    if 0 in q.shape or 0 in v.shape or heads % kv_heads:
        raise ValueError("query heads must be a multiple of the cache heads, and nothing may be empty")
    lens = _int32_vector(kv_lens, "kv_lens", rows, index)
    tree, stride = 0, 0
    if parents is not None:
        check_tree(parents, rows, nodes, index)
        tree, stride = parents.data_ptr(), parents.stride(0)
    if window is None:
        _no_window(sinks)
        window = 0
    elif window < 1 or sinks < 0 or max(window, sinks) >= 2**31:
        raise ValueError("a window must be positive and the number of sinks must not be negative")
    if lse is None:
        lse = (0, 0, 0, 0)
    elif lse.shape != q.shape[:3] or lse.dtype != lse_dtype(q.dtype) or lse.get_device() != index:
        raise ValueError("lse must be [B, Hq, T] on the query's device, fp32 (fp64 for fp64 inputs)")
    else:
        lse = (lse.data_ptr(), *lse.stride())
    if out.shape != (rows, heads, nodes, value_dim) or out.dtype != q.dtype or out.get_device() != index:
        raise ValueError("out must be [B, Hq, T, Dv] of the query's dtype and device")
    scale = default_scale(dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("attention scale must be finite")
    return (_ATTN_STRUCT.pack(q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(),
                              out.data_ptr(), *out.stride(), *lse, code, rows, heads, kv_heads, nodes, capacity, dim,
                              value_dim, scale, 1, 0, lens, 0, 0, 0, 0, 0, 0),
            _TREE_STRUCT.pack(tree, stride, int(window), int(sinks)), index)


def _tree_out(q, v):
    return q.new_empty((*q.shape[:3], v.shape[-1]))


def attention_tree_path(q, k, v, kv_lens, parents=None, *, window=None, sinks=0, scale=None) -> str:
    """Name of the kernel family ``attention_tree`` selects: "tcgen05" or "simt"."""
    params, tree, _ = _tree_args(q, k, v, kv_lens, parents, window, sinks, scale, _tree_out(q, v), None)
    code = _lib.lib().ts_attn_tree_path(params, tree)
    if code < 0:
        _lib.check(code, "ts_attn_tree_path")
    return _lib.PATH_NAMES[code]


def attention_tree_workspace_bytes(q, k, v, kv_lens, parents=None, *, window=None, sinks=0, scale=None) -> int:
    """Bytes of the ``workspace`` that ``attention_tree`` needs for these arguments."""
    params, tree, _ = _tree_args(q, k, v, kv_lens, parents, window, sinks, scale, _tree_out(q, v), None)
    return int(_lib.lib().ts_attn_tree_workspace_size(params, tree))


def attention_tree(q, k, v, kv_lens, parents=None, *, window=None, sinks=0, scale=None, need_lse=False, out=None,
                   lse=None, workspace=None):
    """Attention of T drafted tokens a row, ``q`` [B, Hq, T, D], over a KV cache: ``(out, lse or None)``.

    The last T of row b's ``kv_lens[b]`` keys in ``k``, ``v`` [B, Hkv, capacity, D] are the drafted tokens (T = 1: a
    plain decode step).  ``parents`` (int32 [B, T]) makes them a tree of at most 64 nodes: node i's parent is an
    earlier node, or -1 for the committed tokens; it sees every committed token, its ancestors and itself.  Any other
    entry marks a padded node: its output is zero (LSE -inf), and neither it nor its children are seen by others.
    Without ``parents`` the tokens are a chain.  ``window`` and ``sinks`` as in ``forward``, by the nodes' positions
    (``tree_positions``)."""
    if out is None:
        out = _tree_out(q, v)
    if not need_lse:
        lse = None
    elif lse is None:
        lse = q.new_empty(q.shape[:3], dtype=lse_dtype(q.dtype))
    params, tree, index = _tree_args(q, k, v, kv_lens, parents, window, sinks, scale, out, lse)
    handle = _lib.lib()
    with _on(index):
        need = handle.ts_attn_tree_workspace_size(params, tree)
        if need:
            workspace = _workspace(workspace, need, q)
        status = handle.ts_attn_tree(params, tree, workspace.data_ptr() if need else None, need, _raw_stream(index))
    if status:
        _lib.check(status, "ts_attn_tree")
    return out, lse


def tree_positions(parents, lens):
    """Positions int32 [B, T] of drafted nodes: ``lens[b]`` committed tokens plus the node's depth, -1 for padded
    nodes.  ``rope`` takes them for the nodes' queries and keys."""
    index = parents.get_device()
    if parents.dtype != torch.int32 or parents.dim() != 2 or index < 0 or 0 in parents.shape or (
            parents.stride(1) != 1 and parents.shape[1] > 1):
        raise ValueError("parents must be int32 [batch, nodes] with contiguous rows on a CUDA device")
    rows, nodes = parents.shape
    positions = parents.new_empty((rows, nodes))
    with _on(index):
        status = _lib.lib().ts_tree_positions(parents.data_ptr(), parents.stride(0),
                                              _int32_vector(lens, "lens", rows, index), rows, nodes,
                                              positions.data_ptr(), _raw_stream(index))
    if status:
        _lib.check(status, "ts_tree_positions")
    return positions


def kv_keep(caches, base, path, counts):
    """Close caches behind the accepted path: of every ``(keys, values)`` pair [B, H, capacity, C] in ``caches``, slot
    ``base[b] + path[b, k]`` moves to slot ``base[b] + k`` for k < ``counts[b]``.

    ``path`` (int32 [B, N]) holds the accepted nodes in ascending order, ``base`` and ``counts`` int32 vectors.  All
    layers share their shapes, strides and dtype (int8 storage too; the scales of an int8 cache are caches of one
    channel) and lie in memory of their own."""
    keys, values = [], []
    for key, value in caches:
        keys.append(key)
        values.append(value)
    if not keys:
        raise ValueError("caches must be (keys, values) pairs")
    if len({t.data_ptr() for t in keys + values}) < 2 * len(keys):
        raise ValueError("a cache may be given only once")
    key, value = keys[0], values[0]
    index = key.get_device()
    if index < 0 or key.dim() != 4 or value.dim() != 4 or value.shape[:3] != key.shape[:3]:
        raise ValueError("caches must be [batch, heads, capacity, channels] on a CUDA device")
    if 0 in key.shape or 0 in value.shape or key.dtype != value.dtype:
        raise ValueError("caches must not be empty, keys and values of one dtype")
    for tensors in (keys, values):
        if len({(t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors}) > 1:
            raise ValueError("the caches of all layers must have the same shape, strides, dtype and device")
    key_stride, value_stride = key.stride(), value.stride()
    if value.get_device() != index or (key.shape[3] > 1 and key_stride[3] != 1) or (
            value.shape[3] > 1 and value_stride[3] != 1):
        raise ValueError("a cache's channels must be contiguous, keys and values on one device")
    rows, heads, capacity, dim = key.shape
    if path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != rows or path.get_device() != index or (
            path.stride(1) != 1 and path.shape[1] > 1):
        raise ValueError("path must be int32 [batch, nodes] with contiguous rows on the caches' device")
    base, counts = _int32_vector(base, "base", rows, index), _int32_vector(counts, "counts", rows, index)
    nodes = path.shape[1]
    if nodes == 0:
        return
    n = len(keys)
    pointers = (ctypes.c_void_p * (2 * n))(*[t.data_ptr() for t in keys], *[t.data_ptr() for t in values])
    at = ctypes.addressof(pointers)
    params = _KEEP_STRUCT.pack(at, at + n * ctypes.sizeof(ctypes.c_void_p), *key_stride[:3], 1, *value_stride[:3], 1,
                               _storage_code(key.dtype), n, rows, heads, dim, value.shape[3], capacity, nodes, base,
                               path.data_ptr(), counts, path.stride(0))
    with _on(index):
        status = _lib.lib().ts_kv_keep(params, _raw_stream(index))
    if status:
        _lib.check(status, "ts_kv_keep")


# -- log probabilities of tokens -------------------------------------------------


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` gives for [..., V] logits: fp32 ``logprob`` and ``entropy`` [...], ``top_logprobs``
    [..., top] and int64 ``top_indices`` [..., top]; ``norm`` [..., 2] is the backward's."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_indices: torch.Tensor
    norm: torch.Tensor

    @property
    def lse(self) -> torch.Tensor:
        """log sum exp of the logits."""
        return self.norm[..., 0] + self.norm[..., 1]


_LOGPROB_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _logit_rows(logits):
    """Logits [..., V] as [rows, V] with contiguous rows, without a copy where their strides allow it."""
    if logits.dtype not in _LOGPROB_DTYPES:
        raise TypeError("logits must be float32, float16 or bfloat16")
    if logits.get_device() < 0:
        raise ValueError("the B200 attention engine needs CUDA device tensors")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must be [..., vocabulary]")
    flat = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if flat.stride(1) != 1 or (flat.shape[0] > 1 and flat.stride(0) < 0):
        flat = flat.contiguous()
    return flat


def _target_rows(targets, logits):
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:-1] or targets.get_device() != logits.get_device():
        raise ValueError("targets must be int64 and have the shape of the logits without the vocabulary, on their device")
    return targets if targets.dim() == 1 and targets.is_contiguous() else targets.reshape(-1).contiguous()


def token_logprobs(logits, targets, *, top=0, ignore_index=-100) -> TokenLogprobs:
    """Log probabilities of ``targets`` [...] under softmax of ``logits`` [..., V], entropies (nats) and the ``top``
    most likely alternatives (at most 32; equal logits by index), in one pass.

    A target equal to ``ignore_index`` has log probability 0; one outside the vocabulary NaN.  A row of -inf has log
    probabilities of -inf and entropy 0."""
    flat = _logit_rows(logits)
    goal = _target_rows(targets, logits)
    rows, vocab = flat.shape
    if not 0 <= top <= min(vocab, _lib.TOP_TOKENS_MAX):
        raise ValueError(f"top must be between zero and {_lib.TOP_TOKENS_MAX}, and within the vocabulary")
    fp32 = dict(dtype=torch.float32, device=flat.device)
    logprob, entropy, norm = torch.empty((rows,), **fp32), torch.empty((rows,), **fp32), torch.empty((rows, 2), **fp32)
    values, indices = torch.empty((rows, top), **fp32), targets.new_empty((rows, top))
    if rows:
        index = flat.get_device()
        params = _LOGPROB_STRUCT.pack(flat.data_ptr(), flat.stride(0), dtype_code(flat.dtype), rows, vocab, top,
                                      goal.data_ptr(), ignore_index, logprob.data_ptr(), entropy.data_ptr(),
                                      norm.data_ptr(), values.data_ptr(), indices.data_ptr())
        with _on(index):
            status = _lib.lib().ts_token_logprobs_fwd(params, _raw_stream(index))
        if status:
            _lib.check(status, "ts_token_logprobs_fwd")
    shape = targets.shape
    if len(shape) != 1:
        logprob, entropy, norm = logprob.view(shape), entropy.view(shape), norm.view(*shape, 2)
        values, indices = values.view(*shape, top), indices.view(*shape, top)
    return TokenLogprobs(logprob, entropy, values, indices, norm)


def token_logprobs_backward(logits, targets, result, grad_logprob=None, grad_entropy=None, grad_top=None, *,
                            ignore_index=-100):
    """Gradient of the logits from those of ``result = token_logprobs(logits, targets)``: of its ``logprob``,
    ``entropy`` and ``top_logprobs`` (each fp32, optional)."""
    flat = _logit_rows(logits)
    goal = _target_rows(targets, logits)
    top, index = result.top_indices.shape[-1], flat.get_device()
    given = []
    for g, like in ((grad_logprob, result.logprob), (grad_entropy, result.entropy), (grad_top, result.top_logprobs)):
        if g is not None:
            if g.shape != like.shape or g.dtype != torch.float32 or g.get_device() != index:
                raise ValueError("gradients must be fp32 of the shapes of what they belong to, on the logits' device")
            g = g.contiguous()
        given.append(g)
    shape, fp32 = targets.shape, torch.float32
    for t, want, dtype in ((result.logprob, shape, fp32), (result.entropy, shape, fp32), (result.norm, (*shape, 2), fp32),
                           (result.top_logprobs, (*shape, top), fp32), (result.top_indices, (*shape, top), torch.int64)):
        if t.shape != want or t.dtype != dtype or t.get_device() != index:
            raise ValueError("the result belongs to other logits")
    rows, vocab = flat.shape
    grad = torch.empty((rows, vocab), dtype=flat.dtype, device=flat.device)
    if rows:
        entropy, norm, indices = (t.contiguous() for t in (result.entropy, result.norm, result.top_indices))
        params = _LOGPROB_STRUCT.pack(flat.data_ptr(), flat.stride(0), dtype_code(flat.dtype), rows, vocab, top,
                                      goal.data_ptr(), ignore_index, 0, entropy.data_ptr(), norm.data_ptr(), 0,
                                      indices.data_ptr())
        with _on(index):
            status = _lib.lib().ts_token_logprobs_bwd(params, *(None if g is None else g.data_ptr() for g in given),
                                                      grad.data_ptr(), grad.stride(0), _raw_stream(index))
        if status:
            _lib.check(status, "ts_token_logprobs_bwd")
    return grad if logits.dim() == 2 else grad.view(logits.shape)


# -- pages ---------------------------------------------------------------------


PAGES_SHORT, PAGES_BAD_INDEX, PAGES_NO_SLOT = 1, 2, 4  # error bits of counters[2]


def kv_pages_state(num_pages: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """``(refs, counters)`` of a pool without live pages: references to each page, and int32
    {free pages, a page below which none is free, error bits, unused}."""
    refs = torch.zeros(num_pages, dtype=torch.int32, device=device)
    return refs, torch.tensor([num_pages, 0, 0, 0], dtype=torch.int32, device=device)


def _page_pool(pool) -> tuple:
    """(packed ts_page_pool, pages, device index, page bytes, layers) of a pool of opaque pages, [pages, kv heads,
    block] or [layers, pages, kv heads, block]."""
    index, shape, stride = pool.get_device(), pool.shape, pool.stride()
    if index < 0:
        raise ValueError("the B200 attention engine needs CUDA device tensors")
    if len(shape) == 3:
        shape, stride = (1, *shape), (0, *stride)
    if len(shape) != 4 or stride[3] != 1 or stride[2] != shape[3]:
        raise ValueError("a page pool must be [layers, pages, kv heads, block] with contiguous pages")
    size = pool.element_size()
    page = shape[2] * shape[3] * size
    return (_POOL_STRUCT.pack(pool.data_ptr(), stride[0] * size, stride[1] * size, page, shape[0], shape[1]), shape[1],
            index, page, shape[0])


def kv_pages_copy(src_pool, src, dst_pool, dst):
    """Copy page ``src[i]`` of one pool to page ``dst[i]`` of another (or the same), in every layer; pairs with a
    negative or out-of-range entry are skipped.  No page may be both read and written."""
    a, _, index, page, layers = _page_pool(src_pool)
    b, _, other, other_page, other_layers = _page_pool(dst_pool)
    count = src.shape[0]
    from_ptr, to_ptr = _int32_vector(src, "src", count, index), _int32_vector(dst, "dst", count, index)
    if (index, page, layers) != (other, other_page, other_layers):
        raise ValueError("pools must have the same layers and page size, on one device")
    status = _lib.lib().ts_kv_pages_copy(a, b, from_ptr, to_ptr, count, _raw_stream(index))
    if status:
        _lib.check(status, "ts_kv_pages_copy")


def kv_pages_fork(page_table, lens, index, refs, counters, *, page_size, table_out=None, lens_out=None):
    """Rows that share the pages of the rows ``index`` names: fork, beam reorder, and free (an entry of -1 leaves
    its row empty).  Returns ``(table, lens)`` with ``len(index)`` rows; ``refs`` and ``counters`` are updated."""
    device = page_table.get_device()
    if device < 0:
        raise ValueError("the B200 attention engine needs CUDA device tensors")
    table, stride, rows, slots = _page_table(page_table, device)
    n, pages = index.shape[0], refs.shape[0]
    if n == 0 or page_size <= 0:
        raise ValueError("fork needs at least one row and a positive page size")
    if table_out is None:
        table_out = page_table.new_empty((n, slots))
    if lens_out is None:
        lens_out = lens.new_empty((n,))
    out, out_stride, out_rows, out_slots = _page_table(table_out, device, written=True)
    if (out_rows, out_slots) != (n, slots):
        raise ValueError("table_out must be [len(index), slots]")
    status = _lib.lib().ts_kv_pages_fork(
        table, stride, _int32_vector(lens, "lens", rows, device), rows, _int32_vector(index, "index", n, device), out,
        out_stride, _int32_vector(lens_out, "lens_out", n, device), n, slots, page_size,
        _int32_vector(refs, "refs", pages, device), pages, _int32_vector(counters, "counters", 4, device),
        _raw_stream(device))
    if status:
        _lib.check(status, "ts_kv_pages_fork")
    return table_out, lens_out


def kv_pages_reserve(pool, page_table, lens, steps, refs, counters, *, page_size, workspace=None):
    """Give every row pages of its own for the next ``steps`` tokens (an int, or int32 per row on the device):
    free pages for empty slots, a copy of a partly filled page that other rows hold too.  Works in place; when the
    pool or the table is too small it sets an error bit of ``counters[2]`` and changes nothing."""
    packed, pages, device, _, _ = _page_pool(pool)
    table, stride, rows, slots = _page_table(page_table, device, written=True)
    row_steps = None
    if isinstance(steps, torch.Tensor):
        row_steps, steps = _int32_vector(steps, "steps", rows, device), 0
    if steps < 0 or page_size <= 0:
        raise ValueError("steps must not be negative and the page size must be positive")
    handle = _lib.lib()
    need = handle.ts_kv_pages_reserve_workspace_size(pages, rows)
    workspace = _workspace(workspace, need, page_table)
    status = handle.ts_kv_pages_reserve(
        packed, table, stride, _int32_vector(lens, "lens", rows, device), rows, slots, page_size, steps, row_steps,
        _int32_vector(refs, "refs", pages, device), _int32_vector(counters, "counters", 4, device),
        workspace.data_ptr(), need, _raw_stream(device))
    if status:
        _lib.check(status, "ts_kv_pages_reserve")


def kv_pages_compact(pool, page_table, refs, counters, *, table_out=None, refs_out=None, workspace=None):
    """Move the live pages to the start of the pool (the highest page into the lowest hole, and so on) and rewrite
    the tables and counts, in place unless ``table_out`` / ``refs_out`` are given.  Returns ``(table, refs)``."""
    packed, pages, device, _, _ = _page_pool(pool)
    table, stride, rows, slots = _page_table(page_table, device)
    table_out = page_table if table_out is None else table_out
    refs_out = refs if refs_out is None else refs_out
    out, out_stride, out_rows, out_slots = _page_table(table_out, device, written=True)
    if (out_rows, out_slots) != (rows, slots):
        raise ValueError("table_out must have the table's shape")
    handle = _lib.lib()
    need = handle.ts_kv_pages_compact_workspace_size(pages)
    workspace = _workspace(workspace, need, page_table)
    status = handle.ts_kv_pages_compact(
        packed, table, stride, out, out_stride, rows, slots, _int32_vector(refs, "refs", pages, device),
        _int32_vector(refs_out, "refs_out", pages, device), _int32_vector(counters, "counters", 4, device),
        workspace.data_ptr(), need, _raw_stream(device))
    if status:
        _lib.check(status, "ts_kv_pages_compact")
    return table_out, refs_out


_INV_FREQ: dict = {}


def rope_inv_freq(rotary_dim: int, base: float, device) -> torch.Tensor:
    """inv_freq[i] = base^(-2i/rotary_dim) in fp32, evaluated as the reference
    does it (float32 exponent array, nn/attention.py:274), cached per device."""
    import numpy as np

    key = (int(rotary_dim), float(base), str(device))
    if key not in _INV_FREQ:
        host = base ** (-np.arange(0, rotary_dim, 2).astype(np.float32) / rotary_dim)
        _INV_FREQ[key] = torch.from_numpy(np.ascontiguousarray(host.astype(np.float32))).to(device)
    return _INV_FREQ[key]


def rope(x, *, offset=0, base=10000.0, rotary_dim=None, positions=None, inverse=False, out=None):
    """Interleaved-pair rotary embedding of a [B, H, T, C] view at positions offset + t
    (or positions[b] + t, positions [B] or [B, 1]; or positions[b, t], as ``tree_positions`` gives them); ``inverse``
    applies the inverse rotation (the VJP)."""
    _require_cuda(x)
    dim = x.shape[3] if rotary_dim is None else int(rotary_dim)
    out = torch.empty_like(x) if out is None else out
    inv = rope_inv_freq(dim, base, x.device)
    pos = None
    if positions is not None:
        pos = positions if positions.dtype == torch.int32 else positions.to(torch.int32)
        if pos.get_device() != x.get_device() or pos.numel() < x.shape[0]:
            raise ValueError("positions must be one a row or one a token, on the input's device")
        if pos.shape == (x.shape[0], 1):  # a row's, as [B]
            pos = pos.reshape(-1).contiguous()
        if pos.dim() == 2:
            if pos.shape != (x.shape[0], x.shape[2]):
                raise ValueError("positions of every token must be [B, T] on the input's device")
            pos = pos.contiguous()
            with _on(x.get_device()):
                _lib.check(
                    _lib.lib().ts_rope_at(view4(x), view4(out), dtype_code(x.dtype), x.shape[0], x.shape[1],
                                          x.shape[2], x.shape[3], dim, pos.data_ptr(), inv.data_ptr(),
                                          1 if inverse else 0, _stream_handle(x.device)), "ts_rope_at")
            return out
    _lib.check(
        _lib.lib().ts_rope(view4(x), view4(out), dtype_code(x.dtype), x.shape[0], x.shape[1], x.shape[2],
                           x.shape[3], dim, int(offset), pos.data_ptr() if pos is not None else None,
                           inv.data_ptr(), 1 if inverse else 0, _stream_handle(x.device)),
        "ts_rope",
    )
    return out


def kv_append_rope(key, value, key_cache, value_cache, *, position=0, positions=None, positions_out=None,
                   base=10000.0, rotary_dim=None):
    """kv_append with the keys rotated at their cache positions in the same pass."""
    _require_cuda(key, value, key_cache, value_cache)
    dim = key.shape[3] if rotary_dim is None else int(rotary_dim)
    p = _lib.KvAppendParams()
    p.key, p.value = view4(key), view4(value)
    p.key_cache, p.value_cache = view4(key_cache), view4(value_cache)
    p.src_dtype = dtype_code(key.dtype)
    p.cache_dtype = dtype_code(key_cache.dtype)
    if value.dtype != key.dtype or value_cache.dtype != key_cache.dtype:
        raise TypeError("key/value and their caches must share a dtype each")
    p.batch, p.heads, p.steps = key.shape[0], key.shape[1], key.shape[2]
    p.head_dim, p.value_dim, p.capacity = key.shape[3], value.shape[3], key_cache.shape[2]
    p.position = int(position)
    p.positions = positions.data_ptr() if positions is not None else None
    p.positions_out = positions_out.data_ptr() if positions_out is not None else None
    inv = rope_inv_freq(dim, base, key.device)
    _lib.check(_lib.lib().ts_kv_append_rope(ctypes.byref(p), inv.data_ptr(), dim, _stream_handle(key.device)),
               "ts_kv_append_rope")


def device_status(device=None) -> tuple[int, int]:
    """(status, site) of the device fault word; clears it.  Synchronises the stream."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    info = ctypes.c_uint32(0)
    with torch.cuda.device(device):
        status = _lib.lib().ts_attn_device_status(_stream_handle(device), ctypes.byref(info))
    return status, info.value


def check_device_status(device=None) -> None:
    status, site = device_status(device)
    if status != _lib.OK:
        raise _lib.EngineError(status, f"device fault site 0x{site:x}")
