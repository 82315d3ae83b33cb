"""Attention over an NVFP4 KV cache (:mod:`.kv_cache`): single tokens, chunks
of prompts and batches that mix both, in one call.

Keys and values stay in 4 bits until they are in registers or shared memory;
a scale times a code has 6 significant bits, so 16-bit floats (f16) hold it
exactly.  What is rounded to 16 bits: a bf16 query to f16, the softmax weights
(f16, in units that keep full precision down to 2^-24 of the largest) and the
result.  f16 holds bf16 values from 2^-17 to 2^16 exactly.  Single tokens and
short queries are scaled by a power of two per row first, so that only elements
below 2^-17 of the row's largest are rounded; rows of longer queries only where
their largest lies outside 2^-6 .. 2^15, so that otherwise elements below 2^-17
are rounded, by at most 2^-19 of the largest.  Sums are float32."""
from __future__ import annotations

import torch

from . import _lib


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
    the launch, so that nothing is read back.  Queries and keys past them may be
    passed over.

    ``causal``: a query sees the keys up to its own position, its sequence's
    queries being the last of its keys.  ``window``: only those at most
    ``window`` positions before it.  ``softmax_scale`` defaults to D ** -0.5.
    A row that sees no key gives zeros (log-sum-exp -inf); NaN or an infinity in
    a query row that sees one gives NaN, in that row alone.  Scores are float32
    in units of log 2: a row whose largest lies past 2^23 may not be finite, past
    2^28 it is NaN.  (The cache's scales
    are finite, as the write leaves them: a foreign NaN scale of a key that some
    query sees makes NaN of rows that share work with that query's.)

    Returns ``out`` [T, Hq, D] of the query's type (rows of no sequence are left
    as they were; without ``out`` a new tensor, those rows undefined), with
    ``return_lse`` also the float32 [T, Hq] natural log-sum-exp of the scores.
    ``status``: optional int32 device tensor, set to 1 if a bounded wait inside
    the kernel gave up; the rows that it left unfinished are NaN.

    There is no backward pass: a query that requires a gradient is refused outside
    ``torch.no_grad()``."""
    return _lib.kv_binding().attend(query, codes, scales, kv_input_scale, block_table, seq_lens,
                                    query_start, max_query_len, max_seq_len, softmax_scale, causal,
                                    window, out, return_lse, status)
