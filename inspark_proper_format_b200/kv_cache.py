"""Paged key-value cache of one attention layer (torch-level wrappers over
``isp_kv_append`` / ``isp_kv_gather``).

K and V rows are quantised as they are written (E4M3 or INT8 with one FP32 scale per
(token, head) row, or plain BF16 / FP16) and read by ``attention.paged_decode_attention``
in that form; ``kv_gather`` reads rows back, e.g. a cached prefix as the keys of
``attention.prompt_attention``.

The reference appends to contiguous 16-bit caches inside its engines
(``ops/triton/target_kv_write.py``); pages and 8-bit rows are this library's.

One triple names the same tokens to every call: ``page_table`` (int32 [B, width], the pool
pages of each sequence in order), ``lengths`` (int32 [B], its tokens including those of
the call) and ``cu_seqlens`` (int32 [B + 1], the call's packed tokens of each sequence:
the last ``cu[b + 1] - cu[b]`` positions below ``lengths[b]``).  They are device tensors,
read by the kernels only, so a decode loop needs no host synchronisation; an entry that
points outside the pool is skipped and recorded in ``_lib.read_device_error()``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

FORMATS = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32,
          torch.float8_e4m3fn: _lib.E4M3, torch.int8: _lib.I8}

# the current stream's handle without the Python stream object (2 us of a 15 us call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class PagedKVCache:
    """K and V pools [pages, kv_heads, page_size, head_dim], with FP32 scales
    [pages, kv_heads, page_size] for the 8-bit formats."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, fmt: str = "e4m3",
                 device="cuda"):
        if fmt not in FORMATS:
            raise ValueError(f"unknown cache format {fmt!r}")
        if min(pages, kv_heads, page_size) < 1 or head_dim not in (64, 128):
            raise ValueError("pages, kv_heads and page_size must be positive and head_dim 64 or 128")
        shape = (pages, kv_heads, page_size, head_dim)
        size = FORMATS[fmt].itemsize
        kind = torch.uint8 if size == 1 else torch.int16

        def pool():
            return torch.zeros(shape, device=device, dtype=kind).view(FORMATS[fmt])
        scales = [torch.zeros(shape[:3], device=device) if size == 1 else None for _ in range(2)]
        self._take(pool(), pool(), *scales)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache over existing pools (no copy)."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, k_scale, v_scale):
        if k.dtype not in FORMATS.values() or v.dtype != k.dtype or k.ndim != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim] pools of one cache format")
        if min(k.shape[:3]) < 1 or k.shape[3] not in (64, 128):
            raise ValueError("pages, kv_heads and page_size must be positive and head_dim 64 or 128")
        scaled = k.dtype.itemsize == 1
        for s in (k_scale, v_scale):
            if scaled != (s is not None):
                raise ValueError("8-bit pools need k_scale and v_scale, 16-bit pools take none")
            if scaled and (s.dtype != torch.float32 or s.shape != k.shape[:3]):
                raise ValueError("scales must be FP32 [pages, kv_heads, page_size]")
        for t in (k, v, k_scale, v_scale):
            if t is not None and (not t.is_contiguous() or t.device != k.device or t.data_ptr() % 16):
                raise ValueError("cache tensors must be contiguous, 16-byte aligned and on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.fmt = next(name for name, dtype in FORMATS.items() if dtype == k.dtype)
        self.device = k.device
        self.dtype = k.dtype
        self._struct = _lib.KVCache(_lib.ptr(k), _lib.ptr(v), _lib.ptr(k_scale), _lib.ptr(v_scale), self.pages,
                                    _TYPES[k.dtype], self.page_size, self.kv_heads, self.head_dim)
        self.struct = ctypes.byref(self._struct)          # the C ABI's description of this cache


def index_array(t: torch.Tensor, name: str, device, size=None) -> int:
    """The pointer of an int32 CUDA index array (1-D, contiguous, of ``size`` elements)."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be an int32 CUDA tensor on the operands' device")
    shape = t.shape
    if len(shape) != 1 or (size is not None and shape[0] != size) or (t.stride(0) != 1 and shape[0] > 1):
        raise ValueError(f"{name} must be contiguous with {size if size is not None else 'its'} elements")
    return t.data_ptr()


def table_args(page_table: torch.Tensor, lengths: torch.Tensor, device):
    """((pointer, row stride, width, lengths pointer, batch), table) of a page table and its lengths.
    The kernels step from row to row by at least the width, so a view whose rows overlap (an
    expanded one) is copied; the caller keeps ``table`` until the call."""
    if (not isinstance(page_table, torch.Tensor) or page_table.dtype is not torch.int32 or not page_table.is_cuda
            or page_table.device != device or page_table.ndim != 2):
        raise ValueError("page_table must be an int32 CUDA tensor [batch, pages per sequence]")
    batch, width = page_table.shape
    stride, last = page_table.stride()
    if width < 1 or (last != 1 and width > 1):
        raise ValueError("page_table must be an int32 CUDA tensor [batch, pages per sequence]")
    if stride < width and batch > 1:
        page_table = page_table.contiguous()
    args = (page_table.data_ptr(), max(page_table.stride(0), width), width,
            index_array(lengths, "lengths", device, batch), batch)
    return args, page_table


def call(device, name: str, *args) -> None:
    """Run a C entry point on the device's current stream (its last argument) and raise on an
    error status.  The current device is switched only where it is another one."""
    fn = getattr(_lib.load(), name)
    stream = _raw_stream(device.index) if _raw_stream is not None else _lib.stream_handle(device)
    if torch.cuda.current_device() == device.index:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream)
    if status:
        _lib.check(status, name)


def rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [tokens, heads, dim] with strides the kernels take: itself where the last
    dimension is contiguous and its rows are apart, at multiples of 16 bytes; else a copy."""
    unit = 16 // t.element_size()
    tokens, heads, dim = t.shape
    token, head, last = t.stride()
    if (last == 1 and token % unit == 0 and head % unit == 0 and t.data_ptr() % 16 == 0
            and (token >= dim or tokens <= 1) and (head >= dim or heads == 1)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def kv_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, cu_seqlens: torch.Tensor | None = None) -> None:
    """Write the rows ``k``, ``v`` [T, kv_heads, head_dim] (BF16, FP16 or FP32, any strides) of
    packed tokens into the cache.  Without ``cu_seqlens`` there is one token per sequence
    (a decode step); a token whose sequence has length 0 is not written."""
    if not k.is_cuda or k.device != cache.device or v.device != cache.device:
        raise ValueError("k, v and the cache must be on one CUDA device")
    if k.shape != v.shape or k.ndim != 3 or k.shape[1:] != (cache.kv_heads, cache.head_dim):
        raise ValueError("k and v must both be [tokens, kv_heads, head_dim] of the cache")
    if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("k and v must both be BF16, FP16 or FP32")
    table, page_table = table_args(page_table, lengths, cache.device)
    cu = None
    if cu_seqlens is not None:
        cu = index_array(cu_seqlens, "cu_seqlens", cache.device, table[-1] + 1)
    elif k.shape[0] != table[-1]:
        raise ValueError("without cu_seqlens there is one token per sequence")
    if k.shape[0] == 0:
        return
    k, v = rows(k), rows(v)
    call(cache.device, "isp_kv_append", k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], k.shape[0], k.stride(0),
         k.stride(1), v.stride(0), v.stride(1), cu, *table, cache.struct)


def kv_gather(cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor,
              cu_seqlens: torch.Tensor | None = None, *, tokens: int | None = None,
              dtype: torch.dtype = torch.bfloat16):
    """Read rows back as (k, v), each [tokens, kv_heads, head_dim] in ``dtype``: the inverse of
    ``kv_append`` with the same arguments.  ``tokens`` is ``cu_seqlens[-1]``, given by the
    caller so that nothing has to be copied to the host; rows that no sequence claims, and
    positions before a sequence's start, are zeros."""
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("rows are read back as BF16, FP16 or FP32")
    table, page_table = table_args(page_table, lengths, cache.device)
    batch = table[-1]
    cu = None
    if cu_seqlens is None:
        if tokens not in (None, batch):
            raise ValueError("without cu_seqlens there is one token per sequence")
        tokens = batch
    else:
        cu = index_array(cu_seqlens, "cu_seqlens", cache.device, batch + 1)
        if tokens is None or tokens < 0:
            raise ValueError("tokens must give the number of packed rows")
    k, v = torch.empty((2, tokens, cache.kv_heads, cache.head_dim), device=cache.device, dtype=dtype).unbind(0)
    if tokens:
        call(cache.device, "isp_kv_gather", cache.struct, cu, *table, tokens, _TYPES[dtype], k.data_ptr(), v.data_ptr())
    return k, v
