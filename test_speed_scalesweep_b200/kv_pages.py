"""Pages of an NVFP4 KV cache (:mod:`.kv_cache`): taking, forking, freeing,
compacting and copying them, with the tables on the device.

Every call is a launch or two on the current stream: nothing is read back, so a
scheduler's step can run ahead of the GPU or be captured in a CUDA graph."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kv_cache import PAGE_SIZES

_STATUS = {1: "not enough free pages",
           2: "a sequence index is out of range, named twice, or a child that is not empty",
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
    sequence alone; :meth:`fork` keeps it so."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, refcount: torch.Tensor,
                 status: torch.Tensor | None = None):
        if codes.dim() not in (5, 6) or scales.dim() != codes.dim():
            raise ValueError("codes and scales must be [(layers,) num_pages, 2, kv_heads, page_size, ..]")
        if codes.dtype != torch.uint8 or scales.dtype != torch.float8_e4m3fn:
            raise ValueError("codes must be uint8 and scales float8_e4m3fn, got "
                             f"{codes.dtype} and {scales.dtype}")
        pages, two, heads, page, half = codes.shape[-5:]
        if two != 2 or page not in PAGE_SIZES or half % 8 or scales.shape != codes.shape[:-1] + (half // 8,):
            raise ValueError("codes must be [.., num_pages, 2, kv_heads, page_size, head_size/2] and "
                             f"scales [.., head_size/16], got {tuple(codes.shape)} and {tuple(scales.shape)}")
        dev = codes.device
        if dev.type != "cuda":
            raise ValueError("codes must be a CUDA tensor (there is no CPU implementation)")
        sc, ss = codes.stride(), scales.stride()
        nc, ns = 2 * heads * page * half, 2 * heads * page * (half // 8)
        if (sc[-4:] != (heads * page * half, page * half, half, 1)
                or ss[-4:] != (heads * page * (half // 8), page * (half // 8), half // 8, 1)):
            raise ValueError("codes and scales must be contiguous within a page")
        if block_table.dim() != 2 or block_table.stride(1) != 1:
            raise ValueError("block_table must be [max_seqs, columns] with contiguous rows")
        seqs, columns = block_table.shape
        for name, t, shape in (("block_table", block_table, (seqs, columns)),
                               ("seq_lens", seq_lens, (seqs,)), ("refcount", refcount, (pages,)),
                               ("status", status, (1,))):
            if t is None:
                continue
            if t.dtype != torch.int32 or t.device != dev or t.shape != shape:
                raise ValueError(f"{name} must be an int32 tensor of shape {list(shape)} on {dev}")
            if t is not block_table and not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        if scales.device != dev:
            raise ValueError(f"scales must be on {dev}, got {scales.device}")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.codes, self.scales, self.device = codes, scales, dev
        self.block_table, self.seq_lens, self.refcount, self.status = block_table, seq_lens, refcount, status
        layered = codes.dim() == 6
        self._pool = _lib.KVPool(codes.data_ptr(), scales.data_ptr(), sc[0] if layered else 0,
                                 ss[0] if layered else 0, sc[-5] if pages > 1 else nc,
                                 ss[-5] if pages > 1 else ns, nc, ns, pages,
                                 codes.shape[0] if layered else 1)
        self._tables = _lib.KVPages(refcount.data_ptr(), block_table.data_ptr(),
                                    block_table.stride(0) if seqs > 1 else columns,
                                    seq_lens.data_ptr(), status.data_ptr(), pages, seqs, columns, page)

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

    def _index(self, name: str, t: torch.Tensor, n: int) -> int:
        if t.dtype != torch.int32 or t.shape != (n,) or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape [{n}] on {self.device}")
        return t.data_ptr()

    def _workspace(self, n: int, tokens: int, pages: int) -> torch.Tensor:
        size = _lib.lib().ssw_kv_pages_workspace_bytes(n, tokens, self._tables.page_size, pages)
        return torch.empty(size // 4, dtype=torch.int32, device=self.device)

    def extend(self, seqs: torch.Tensor, new_tokens: torch.Tensor, total_tokens: int) -> torch.Tensor:
        """Pages for ``new_tokens[i]`` more tokens of each sequence ``seqs[i]``
        (int32; distinct), and the slots of the new tokens, sequence by sequence:
        int64 ``[total_tokens]``, the sum of ``new_tokens``."""
        n = seqs.numel()
        ps, pn = self._index("seqs", seqs, n), self._index("new_tokens", new_tokens, n)
        slots = torch.empty(total_tokens, dtype=torch.int64, device=self.device)
        ws = self._workspace(n, total_tokens, 0)
        with _lib.on_device(self.device):
            st = _lib.lib().ssw_kv_pages_extend(
                ctypes.byref(self._tables), n, ps, pn, total_tokens, slots.data_ptr(), ws.data_ptr(),
                ws.numel() * 4, _lib.stream_handle(self.device))
        _lib.check(st)
        return slots

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Make each empty sequence ``children[i]`` a copy of ``parents[i]``
        (int32): full pages are shared, a part-filled last page is copied, so
        that each can be extended on its own."""
        n = parents.numel()
        pp, pc = self._index("parents", parents, n), self._index("children", children, n)
        ws = self._workspace(n, 0, 0)
        with _lib.on_device(self.device):
            st = _lib.lib().ssw_kv_pages_fork(
                ctypes.byref(self._tables), ctypes.byref(self._pool), n, pp, pc, ws.data_ptr(),
                ws.numel() * 4, _lib.stream_handle(self.device))
        _lib.check(st)

    def free(self, seqs: torch.Tensor) -> None:
        """Empty the sequences ``seqs`` (int32).  Pages that no other sequence
        shares become free; their bytes stay until they are taken again."""
        n = seqs.numel()
        ps = self._index("seqs", seqs, n)
        with _lib.on_device(self.device):
            st = _lib.lib().ssw_kv_pages_free(ctypes.byref(self._tables), n, ps,
                                              _lib.stream_handle(self.device))
        _lib.check(st)

    def compact(self) -> None:
        """Move the used pages to the front: with L in use, those numbered L and
        above take the free numbers below, in order; the tables follow."""
        pages = self._tables.num_pages
        ws = self._workspace(0, 0, pages)
        with _lib.on_device(self.device):
            st = _lib.lib().ssw_kv_pages_compact(
                ctypes.byref(self._tables), ctypes.byref(self._pool), ws.data_ptr(), ws.numel() * 4,
                _lib.stream_handle(self.device))
        _lib.check(st)

    def copy(self, source: torch.Tensor, target: torch.Tensor) -> None:
        """Copy page ``source[i]`` to ``target[i]`` (int32) in every layer.
        Targets are distinct, and none is a source; the tables do not change."""
        n = source.numel()
        ps, pt = self._index("source", source, n), self._index("target", target, n)
        with _lib.on_device(self.device):
            st = _lib.lib().ssw_kv_pages_copy(ctypes.byref(self._pool), n, ps, pt,
                                              _lib.stream_handle(self.device))
        _lib.check(st)

    def check(self) -> None:
        """Wait for the tables and raise for the first request that was not
        served since the last check."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError(f"KV pages: {_STATUS.get(code, code)}; the request changed nothing")
