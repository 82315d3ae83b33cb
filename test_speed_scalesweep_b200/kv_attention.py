"""Attention over an NVFP4 KV cache (:mod:`.kv_cache`): single tokens, chunks
of prompts and batches that mix both, in one call.

Keys and values stay in 4 bits until they are in registers or shared memory;
a scale times a code has 6 significant bits, so 16-bit floats hold it exactly
and the only roundings are those of the softmax weights and of the result."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kv_cache import cache_struct, check_distinct, heads_struct


def _check_int32(name: str, t: torch.Tensor, shape: tuple[int, ...], device: torch.device) -> None:
    if t.dtype != torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)} on {device}")


def nvfp4_paged_attention(query: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                          kv_input_scale: torch.Tensor, block_table: torch.Tensor,
                          seq_lens: torch.Tensor, query_start: torch.Tensor, max_query_len: int,
                          max_seq_len: int, *, softmax_scale: float | None = None,
                          causal: bool = True, window: int | None = None,
                          out: torch.Tensor | None = None, return_lse: bool = False,
                          status: torch.Tensor | None = None):
    """Attention of ``query`` [T, Hq, D] (bf16 or f16; the heads may be slices
    of a qkv output) over the cache.

    ``seq_lens`` int32 [B]: each sequence's keys, its new tokens' included (they
    are written first).  ``query_start`` int32 [B + 1]: sequence b has the query
    rows ``query_start[b]:query_start[b + 1]``.  ``block_table`` int32 [B, P]:
    its pages; an entry outside the cache (-1) holds no keys.
    ``max_query_len`` and ``max_seq_len`` bound the lengths from above; they size
    the launch, so that nothing is read back.

    ``causal``: a query sees the keys up to its own position, its sequence's
    queries being the last of its keys.  ``window``: only those at most
    ``window`` positions before it.  ``softmax_scale`` defaults to D ** -0.5.
    A row that sees no key gives zeros (log-sum-exp -inf).

    Returns ``out`` [T, Hq, D] of the query's type (rows of no sequence are left
    as they were; without ``out`` a new tensor, those rows undefined), with
    ``return_lse`` also the float32 [T, Hq] natural log-sum-exp of the scores.
    ``status``: optional int32 device tensor, set to 1 if a bounded wait inside
    the kernel gave up."""
    cache = cache_struct(codes, scales, kv_input_scale)
    if kv_input_scale is None:
        raise ValueError("kv_input_scale is required")
    dev = codes.device
    if query.dim() != 3:
        raise ValueError(f"query must be [T, heads, head_size], got shape {tuple(query.shape)}")
    tokens, hq, d = query.shape
    if d != cache.head_size:
        raise ValueError(f"query has head size {d}, the cache {cache.head_size}")
    dtype = _lib.dtype_code(query)
    q = heads_struct("query", query, (tokens, hq, d), query.dtype, dev)
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != dev:
        raise ValueError(f"block_table must be an int32 tensor [sequences, pages] on {dev}")
    seqs, columns = block_table.shape
    if columns and block_table.stride(1) != 1 and columns > 1:
        raise ValueError("block_table's rows must be contiguous")
    _check_int32("seq_lens", seq_lens, (seqs,), dev)
    _check_int32("query_start", query_start, (seqs + 1,), dev)
    if status is not None and (status.device != dev or status.dtype != torch.int32):
        raise ValueError(f"status must be an int32 tensor on {dev}")
    if window is not None and window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    if out is None:
        out = torch.empty((tokens, hq, d), dtype=query.dtype, device=dev)
    o = heads_struct("out", out, (tokens, hq, d), query.dtype, dev)
    check_distinct("out", out)
    lse = torch.empty((tokens, hq), dtype=torch.float32, device=dev) if return_lse else None
    args = _lib.KVAttention(
        block_table.data_ptr(), block_table.stride(0) if seqs > 1 else columns,
        seq_lens.data_ptr(), query_start.data_ptr(), lse.data_ptr() if return_lse else None,
        status.data_ptr() if status is not None else None, tokens, seqs, columns, hq,
        max_query_len, max_seq_len, bool(causal), -1 if window is None else min(window, (1 << 31) - 1),
        d ** -0.5 if softmax_scale is None else softmax_scale)
    h = _lib.lib()
    pc, pa = ctypes.byref(cache), ctypes.byref(args)
    with _lib.on_device(dev):
        need = h.ssw_nvfp4_paged_attention_workspace_bytes(pc, pa, dtype)
        if need < 0:
            _lib.check(_lib.SSW_ERR_INVALID_ARGUMENT)
        workspace = torch.empty(need // 4, dtype=torch.float32, device=dev) if need else None
        st = h.ssw_nvfp4_paged_attention(
            pc, pa, dtype, ctypes.byref(q), ctypes.byref(o),
            workspace.data_ptr() if need else None, need, _lib.stream_handle(dev))
    _lib.check(st)
    return (out, lse) if return_lse else out
