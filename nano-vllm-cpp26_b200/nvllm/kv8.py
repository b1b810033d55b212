"""The 8-bit paged KV cache (C ABI in include/nvllm.h, nvllm_kv8_*).

The paged geometry of the fp32 arenas with one byte per value and one power-of-two
scale per (token, KV head), for rows of fp32, bf16 or fp16 and grouped query
heads: :func:`kv8_write` quantises rows into the arenas, :func:`kv8_read` brings
rows back, :func:`kv8_attention` attends over them (single tokens, chunks, whole
prompts or a mix), with an optional sliding window and sink positions.

Rows are 2-d tensors whose last dimension is contiguous; their row stride is
free, so a slice of a fused QKV buffer is passed as it is. Calls run on the
device of their tensors (also when it is not the current one), on ``stream`` or
that device's current stream.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import nvllm as _nv

KV8_E4M3 = 0
KV8_INT8 = 1

_DTYPES = {}  # torch dtype -> nvllm_dtype, filled at the first call
_FORMATS = {}  # torch dtype of the codes -> nvllm_kv8_format
_INT32 = _RAW_STREAM = _CURRENT_DEVICE = None  # of torch, likewise


class _Arena(ctypes.Structure):
    """nvllm_kv8_arena."""

    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("k_exps", ctypes.c_void_p), ("v_exps", ctypes.c_void_p),
                ("format", ctypes.c_int32)]


_BOUND = None


def _lib():
    global _BOUND, _INT32, _RAW_STREAM, _CURRENT_DEVICE
    if _BOUND is not None:
        return _BOUND
    import torch
    L = _nv.lib()
    vp, i32, i64, f32, sz = (ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float,
                             ctypes.c_size_t)
    ap, lp = ctypes.POINTER(_Arena), ctypes.POINTER(_nv.KVLayout)
    for f in (L.nvllm_kv8_write, L.nvllm_kv8_read):
        f.restype = ctypes.c_int
        f.argtypes = [vp, vp, i32, i64, i64, ap, vp, i64, i32, lp, vp]
    L.nvllm_kv8_attention_workspace_size.restype = sz
    L.nvllm_kv8_attention_workspace_size.argtypes = [i32, i32, i32, i32, lp]
    L.nvllm_kv8_attention.restype = ctypes.c_int
    L.nvllm_kv8_attention.argtypes = [vp, i64, vp, i64, i32, ap, vp, i32, vp, vp, i32, i32, i32, i32,
                                      i32, f32, i32, i32, vp, sz, lp, vp]
    _INT32, _CURRENT_DEVICE = torch.int32, torch.cuda.current_device
    _RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream",
                          lambda index: torch.cuda.current_stream(index).cuda_stream)
    _DTYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    _FORMATS.update({torch.float8_e4m3fn: KV8_E4M3, torch.int8: KV8_INT8})
    _BOUND = L
    return L


class KV8Arena:
    """The arenas of one cache: codes ``k``, ``v`` [num_blocks, num_layers, block_size,
    num_heads * head_dim] (torch.float8_e4m3fn or torch.int8, which is the format)
    and exponents ``k_exp``, ``v_exp`` [num_blocks, num_layers, num_heads, block_size]
    int8; a cached value is code * 2**exponent. Made once and kept; it holds
    references to the tensors."""

    def __init__(self, layout: _nv.KVLayout, k, v, k_exp, v_exp):
        _lib()
        codes = layout.arena_shape()
        exps = (layout.num_blocks, layout.num_layers, layout.num_heads, layout.block_size)
        if k.dtype not in _FORMATS:
            raise ValueError(f"k must be float8_e4m3fn or int8, got {k.dtype}")
        for t, n, shape, dtype in ((k, "k", codes, k.dtype), (v, "v", codes, k.dtype),
                                   (k_exp, "k_exp", exps, None), (v_exp, "v_exp", exps, None)):
            if dtype is not None and t.dtype != dtype:
                raise ValueError(f"{n} must be {dtype}, got {t.dtype}")
            if dtype is None and str(t.dtype) != "torch.int8":
                raise ValueError(f"{n} must be int8, got {t.dtype}")
            if tuple(t.shape) != shape:
                raise ValueError(f"{n} must have shape {shape}, got {tuple(t.shape)}")
            if not t.is_contiguous():
                raise ValueError(f"{n} must be contiguous")
        if not k.is_cuda or any(t.device != k.device for t in (v, k_exp, v_exp)):
            raise ValueError("the arenas must be CUDA tensors on one device")
        self.layout, self.k, self.v, self.k_exp, self.v_exp = layout, k, v, k_exp, v_exp
        self.device, self.index = k.device, k.get_device()
        self._c = _Arena(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(),
                         _FORMATS[k.dtype])
        self._ref, self._lay = ctypes.byref(self._c), ctypes.byref(layout)

    @classmethod
    def alloc(cls, layout: _nv.KVLayout, fmt: int = KV8_E4M3, device="cuda") -> "KV8Arena":
        """New arenas (zeros)."""
        import torch
        if fmt not in (KV8_E4M3, KV8_INT8):
            raise ValueError(f"unknown format {fmt}")
        code = torch.float8_e4m3fn if fmt == KV8_E4M3 else torch.int8
        k, v = (torch.zeros(layout.arena_shape(), dtype=torch.uint8, device=device).view(code)
                for _ in range(2))
        exps = (layout.num_blocks, layout.num_layers, layout.num_heads, layout.block_size)
        ke, ve = (torch.zeros(exps, dtype=torch.int8, device=device) for _ in range(2))
        return cls(layout, k, v, ke, ve)


def _rows(t, name: str, width: int, arena: KV8Arena) -> int:
    """Checks a 2-d row tensor; its nvllm_dtype."""
    if t.get_device() != arena.index:
        raise ValueError(f"{name} must be on the arena's device {arena.device}, got {t.device}")
    kind = _DTYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] != width:
        raise ValueError(f"{name} must have shape [n, {width}], got {tuple(t.shape)}")
    if t.stride(1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return kind


def _ints(t, name: str, arena: KV8Arena, dim: int = 1):
    if t.get_device() != arena.index:
        raise ValueError(f"{name} must be on the arena's device {arena.device}, got {t.device}")
    if t.dtype != _INT32:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dim}-d tensor")


def _int32(*n: int) -> None:
    """Refuses arguments that the C ABI's int32 would cut."""
    if max(n) > 2147483647 or min(n) < -2147483648:
        raise ValueError("integer arguments must fit 32 bits")


def _stride(t) -> int:
    # the stride of a lone row means nothing
    return t.shape[1] if t.shape[0] <= 1 else t.stride(0)


def _call(arena: KV8Arena, stream, f, *args) -> int:
    """Calls f(*args, stream) with the arena's device current."""
    if stream is None:
        # the raw handle: a Stream object costs more than the launch
        stream = _RAW_STREAM(arena.index)
    elif not isinstance(stream, int):
        stream = stream.cuda_stream
    if arena.index == _CURRENT_DEVICE():
        return f(*args, stream)
    import torch
    with torch.cuda.device(arena.index):
        return f(*args, stream)


def _stream_scope(stream, device):
    """A context in which ``stream`` (None, a raw handle or a Stream) is current."""
    import torch
    if isinstance(stream, int):
        stream = (torch.cuda.ExternalStream(stream, device=device) if stream > 1  # (0, 1: legacy)
                  else torch.cuda.default_stream(device))
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def _move(what: str, f, key, value, arena: KV8Arena, slot_mapping, layer: int, stream,
          check: bool) -> int:
    width = arena.layout.hidden
    kind = _rows(key, "key", width, arena)
    if _rows(value, "value", width, arena) != kind:
        raise ValueError(f"key and value must have one type, got {key.dtype} and {value.dtype}")
    _ints(slot_mapping, "slot_mapping", arena)
    _int32(layer, 0)
    n = slot_mapping.numel()
    if key.shape[0] < n or value.shape[0] < n:
        raise ValueError(f"key and value must hold slot_mapping's {n} rows")
    st = _call(arena, stream, f, key.data_ptr(), value.data_ptr(), kind, _stride(key),
               _stride(value), arena._ref, slot_mapping.data_ptr(), n, layer, arena._lay)
    if check:
        _nv._check(st, what)
    return st


def kv8_write(key, value, arena: KV8Arena, slot_mapping, layer: int, stream=None,
              check: bool = True) -> int:
    """Quantises rows of key/value [n, KV heads * head_dim] into the arena's slots
    (negative: skipped). Slots must be distinct."""
    return _move("nvllm_kv8_write", _lib().nvllm_kv8_write, key, value, arena, slot_mapping, layer,
                 stream, check)


def kv8_read(key, value, arena: KV8Arena, slot_mapping, layer: int, stream=None,
             check: bool = True) -> int:
    """Fills rows of key/value with the values of the arena's slots; rows of
    negative slots stay as they are."""
    return _move("nvllm_kv8_read", _lib().nvllm_kv8_read, key, value, arena, slot_mapping, layer,
                 stream, check)


def kv8_workspace_size(num_seqs: int, max_query_len: int, max_context_len: int, num_heads: int,
                       layout: _nv.KVLayout) -> int:
    _int32(num_seqs, max_query_len, max_context_len, num_heads)
    return int(_lib().nvllm_kv8_attention_workspace_size(num_seqs, max_query_len, max_context_len,
                                                         num_heads, ctypes.byref(layout)))


def kv8_alloc_workspace(num_seqs: int, max_query_len: int, max_context_len: int, num_heads: int,
                        layout: _nv.KVLayout, device="cuda"):
    """A workspace for calls of kv8_attention within these maxima. Calls that may
    overlap on the GPU need one each."""
    import torch
    n = kv8_workspace_size(num_seqs, max_query_len, max_context_len, num_heads, layout)
    return torch.empty(max(n, 256), dtype=torch.uint8, device=device)


def kv8_attention(out, query, arena: KV8Arena, block_tables, cu_seqlens_q, context_lens,
                  max_query_len: int, max_context_len: int, layer: int,
                  num_heads: int | None = None, scale: float | None = None, window: int = 0,
                  sinks: int = 0, workspace=None, stream=None, check: bool = True) -> int:
    """Causal attention of each sequence's new rows over the 8-bit cache.

    ``query`` and ``out`` [rows, num_heads * head_dim] (``num_heads`` query heads, a
    multiple of the layout's KV heads; default: as many). Metadata as in
    :func:`nvllm.paged_attention`. ``window`` > 0 keeps, for the row at position
    p, the positions above p - window and the first ``sinks`` ones. Without a
    ``workspace`` the call allocates one on its stream."""
    layout = arena.layout
    if num_heads is None:
        num_heads = layout.num_heads
    width = num_heads * layout.head_dim
    kind = _rows(query, "query", width, arena)
    if _rows(out, "out", width, arena) != kind:
        raise ValueError(f"out must have query's type {query.dtype}, got {out.dtype}")
    if out.shape[0] < query.shape[0]:
        raise ValueError(f"out must hold query's {query.shape[0]} rows")
    _ints(block_tables, "block_tables", arena, 2)
    _ints(cu_seqlens_q, "cu_seqlens_q", arena)
    _ints(context_lens, "context_lens", arena)
    _int32(max_query_len, max_context_len, layer, window, sinks)
    num_seqs = context_lens.numel()
    if block_tables.shape[0] != num_seqs or cu_seqlens_q.numel() != num_seqs + 1:
        raise ValueError("block_tables, cu_seqlens_q and context_lens disagree on the sequences")
    if scale is None:
        scale = 1.0 / math.sqrt(layout.head_dim)
    if workspace is None:
        # on the call's stream: the allocator orders a block's uses on the stream it came from
        with _stream_scope(stream, arena.device):
            workspace = kv8_alloc_workspace(num_seqs, max_query_len, max_context_len, num_heads, layout,
                                            arena.device)
    elif workspace.get_device() != arena.index:
        raise ValueError(f"workspace must be on the arena's device {arena.device}")
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    st = _call(arena, stream, _lib().nvllm_kv8_attention, out.data_ptr(), _stride(out),
               query.data_ptr(), _stride(query), kind, arena._ref, block_tables.data_ptr(),
               block_tables.shape[1], cu_seqlens_q.data_ptr(), context_lens.data_ptr(), num_seqs,
               max_query_len, max_context_len, num_heads, layer, scale, window, sinks,
               workspace.data_ptr(), workspace.numel() * workspace.element_size(), arena._lay)
    if check:
        _nv._check(st, "nvllm_kv8_attention")
    return st
