"""Serving attention (torch-level wrappers over ``isp_prompt_attention`` and
``isp_paged_decode``).

``prompt_attention`` computes the attention of packed prompts of different lengths,
``paged_decode_attention`` that of one new token per sequence over a
``kv_cache.PagedKVCache``.  Both take grouped heads (query head h reads key-value head
``h // (heads // kv_heads)``), BF16 or FP16 queries and head dimensions 64 and 128.  The
reference leaves both to its engines' closed attention; forward only, as every op of this
package.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .kv_cache import PagedKVCache, call, index_array, rows, table_args

_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _softmax_scale(scale, dim):
    value = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not (0.0 < value < math.inf):
        raise ValueError("the softmax scale must be positive and finite")
    return value


def _check_out(out, q):
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have the queries' shape, type and device")
    if out.stride(2) != 1 or (out.stride(0) * 2) % 16 or (out.stride(1) * 2) % 16 or out.data_ptr() % 16:
        raise ValueError("out needs a contiguous last dimension and 16-byte aligned rows")
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                     cu_seqlens_k: torch.Tensor | None = None, causal: bool = True, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed sequences: ``q`` [tokens, heads, dim], ``k``, ``v`` [keys, kv_heads, dim]
    (views of a fused projection are taken as they are), sequence b in rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` of q and those of ``cu_seqlens_k`` (default:
    the same) of k and v.

    Causal attention is aligned at the end: query i of n sees keys ``j <= i + m - n`` of m,
    so the queries may follow a cached prefix.  A query that sees no key, or only keys with a
    score of -inf, gives zeros; rows that no sequence claims are undefined.  ``scale`` defaults
    to ``1 / sqrt(dim)``."""
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError("expected q [tokens, heads, dim] and k, v [keys, kv_heads, dim]")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must all be BF16 or all FP16")
    if not q.is_cuda or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one CUDA device")
    dim, heads, kv_heads = q.shape[2], q.shape[1], k.shape[1]
    if dim not in (64, 128) or kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError("dim must be 64 or 128 and heads a multiple of kv_heads")
    cu = index_array(cu_seqlens, "cu_seqlens", q.device)
    batch = cu_seqlens.shape[0] - 1
    if batch < 0:
        raise ValueError("cu_seqlens holds one more entry than there are sequences")
    if cu_seqlens_k is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError("cu_seqlens_k is needed where queries and keys differ in number")
        cu_k = cu
    else:
        cu_k = index_array(cu_seqlens_k, "cu_seqlens_k", q.device, batch + 1)
    value = _softmax_scale(scale, dim)
    out = _check_out(out, q)
    if q.shape[0] == 0 or batch == 0:
        return out
    if k.shape[0] == 0:
        return out.zero_()
    q, k, v = rows(q), rows(k), rows(v)
    call(q.device, "isp_prompt_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), _TYPES[q.dtype], q.shape[0],
         k.shape[0], cu, cu_k, batch, heads, kv_heads, dim, *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], value,
         int(bool(causal)), out.data_ptr(), *out.stride()[:2])
    return out


class DecodeWorkspace:
    """Scratch of ``paged_decode_attention`` on one device: the partial results of sequences
    whose cache is read by several blocks.  Calls that may run at the same time (on two
    streams) need one each."""

    def __init__(self, device="cuda"):
        size = ctypes.c_int64(0)
        with torch.cuda.device(device):
            _lib.check(_lib.load().isp_paged_decode_workspace(ctypes.byref(size)), "isp_paged_decode_workspace")
        self.buffer = torch.zeros(size.value, device=device, dtype=torch.uint8)


def paged_decode_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                           scale: float | None = None, out: torch.Tensor | None = None,
                           workspace: DecodeWorkspace | None = None) -> torch.Tensor:
    """Attention of one token per sequence, ``q`` [batch, heads, dim], over the first
    ``lengths[b]`` positions of each sequence's pages (``kv_append`` has written the token's
    own row).  Length 0 gives zeros.  A 16-bit cache must have q's type.

    A decode loop keeps a ``DecodeWorkspace``; without one a fresh one is made for the call."""
    if q.ndim != 3 or q.dtype not in _TYPES:
        raise ValueError("q must be a BF16 or FP16 tensor [batch, heads, dim]")
    if not q.is_cuda or q.device != cache.device:
        raise ValueError("q and the cache must be on one CUDA device")
    if q.shape[2] != cache.head_dim or q.shape[1] < 1 or q.shape[1] % cache.kv_heads:
        raise ValueError("q does not fit the cache's head_dim and kv_heads")
    if cache.k_scale is None and cache.dtype != q.dtype:
        raise ValueError("a 16-bit cache must have the queries' type")
    table, page_table = table_args(page_table, lengths, q.device)
    if table[-1] != q.shape[0]:
        raise ValueError("page_table and lengths must have one row per query")
    value = _softmax_scale(scale, q.shape[2])
    out = _check_out(out, q)
    if q.shape[0] == 0:
        return out
    q = rows(q)
    if workspace is None:
        workspace = DecodeWorkspace(q.device)
    buffer = workspace.buffer
    if buffer.device != q.device:
        raise ValueError("the workspace is on another device")
    call(q.device, "isp_paged_decode", q.data_ptr(), _TYPES[q.dtype], *q.stride()[:2], cache.struct, *table, q.shape[1],
         value, out.data_ptr(), *out.stride()[:2], buffer.data_ptr(), buffer.numel())
    return out
