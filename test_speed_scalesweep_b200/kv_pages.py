"""Pages of an NVFP4 KV cache (:mod:`.kv_cache`): taking, forking, freeing,
compacting and copying them, with the tables on the device.

Every call is a launch or two on the current stream: nothing is read back, so a
scheduler's step can run ahead of the GPU or be captured in a CUDA graph."""
from __future__ import annotations

import torch

from . import _lib

_STATUS = {1: "not enough free pages",
           2: "a sequence index is out of range or named twice, a child is not empty, or new tokens "
              "are negative or do not add up to their total",
           3: "a sequence is longer than its row of the block table"}


class NVFP4KVPages:
    """Page tables of one cache.

    ``codes`` and ``scales``: one layer's cache or, with a leading layer axis,
    all layers' (they share the tables).  ``block_table`` int32
    ``[max_seqs, columns]``, ``seq_lens`` int32 ``[max_seqs]`` and ``refcount``
    int32 ``[num_pages]`` are the caller's tensors, updated in place: attention
    reads rows of the first two as they are.  :meth:`empty` makes them.

    Pages are taken lowest first, in the order of the requests.  A request that
    cannot be served changes nothing and leaves a code in ``status`` (int32
    ``[1]``), which :meth:`check` reads.  A part-filled page must belong to one
    sequence alone; :meth:`fork` keeps it so.  :meth:`copy` is no request on the
    tables and leaves no code."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, refcount: torch.Tensor,
                 status: torch.Tensor | None = None):
        self.codes, self.scales = codes, scales
        self.block_table, self.seq_lens, self.refcount = block_table, seq_lens, refcount
        self._kv = _lib.kv_binding()
        self._pages, self.status = self._kv.pages(codes, scales, block_table, seq_lens, refcount, status)

    @classmethod
    def empty(cls, codes: torch.Tensor, scales: torch.Tensor, max_seqs: int,
              max_pages_per_seq: int) -> "NVFP4KVPages":
        """Tables of ``max_seqs`` empty sequences over a free pool."""
        dev = codes.device
        pages = codes.shape[-5] if codes.dim() >= 5 else 0  # the constructor refuses other shapes
        return cls(codes, scales,
                   torch.full((max_seqs, max_pages_per_seq), -1, dtype=torch.int32, device=dev),
                   torch.zeros(max_seqs, dtype=torch.int32, device=dev),
                   torch.zeros(pages, dtype=torch.int32, device=dev))

    def extend(self, seqs: torch.Tensor, new_tokens: torch.Tensor, total_tokens: int) -> torch.Tensor:
        """Pages for ``new_tokens[i]`` more tokens of each sequence ``seqs[i]``
        (int32; distinct), and the slots of the new tokens, sequence by sequence:
        int64 ``[total_tokens]``, the sum of ``new_tokens``."""
        return self._kv.pages_extend(self._pages, seqs, new_tokens, total_tokens)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Make each empty sequence ``children[i]`` a copy of ``parents[i]``
        (int32): full pages are shared, a part-filled last page is copied, so
        that each can be extended on its own."""
        self._kv.pages_fork(self._pages, parents, children)

    def free(self, seqs: torch.Tensor) -> None:
        """Empty the sequences ``seqs`` (int32; one named twice is freed once).
        Pages that no other sequence shares become free; their bytes stay until
        they are taken again."""
        self._kv.pages_free(self._pages, seqs)

    def compact(self) -> None:
        """Move the used pages to the front: with L in use, those numbered L and
        above take the free numbers below, in order; the tables follow."""
        self._kv.pages_compact(self._pages)

    def copy(self, source: torch.Tensor, target: torch.Tensor) -> None:
        """Copy page ``source[i]`` to ``target[i]`` (int32) in every layer.
        Targets are distinct, and none is a source; a pair with a page outside
        the cache is passed over.  The tables do not change."""
        self._kv.pages_copy(self._pages, source, target)

    def check(self) -> None:
        """Wait for the tables and raise for the first request that was not
        served since the last check."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError(f"KV pages: {_STATUS.get(code, code)}; the request changed nothing")
