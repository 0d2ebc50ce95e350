"""Tensor-level host API of the sequences' pages over the CUDA C ABI: which pages of a paged cache each sequence has, kept on
the device, and one call a step that says where its new tokens go.

  KvPages               block table, lengths and free pages of a batch's sequences
  KvStep                where a step's tokens go: slots, positions, offsets
  kv_pages_step         cuts and grows the sequences by a step

kv_cache_write takes a step's slots and positions, attention_prefill and kv_cache_read its offsets, attention_decode the block
table and the lengths. Nothing is synchronised; a step can be captured in a CUDA graph with the calls that use it.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import _call, _indices
from .iq2_matmul import _bail


class KvPages:
    """The pages of `sequences` sequences: block_table int32 [sequences, width], whose first columns are the pages of
    sequence b's seq_lens[b] tokens (int32 [sequences]; the other columns are not read), and free_pages int32 [num_pages], whose
    first free_count[0] (int32 [1]) entries are the free pages, the next one to be taken last. A page belongs to one sequence
    or is free. The tensors cannot be replaced, and calls refuse ones whose memory has moved."""

    def __init__(self, block_table: torch.Tensor, seq_lens: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                 page_size: int):
        op = "KvPages"
        if not block_table.is_cuda:
            _bail(_lib.IQ2_ERR_DEVICE, f"{op} requires a CUDA device")
        index = block_table.get_device()
        for name, t, dims in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("free_pages", free_pages, 1),
                              ("free_count", free_count, 1)):
            if _indices(op, index, name, t, dims) is not t:
                _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op} expects contiguous layouts")
        if seq_lens.shape[0] != block_table.shape[0] or free_count.shape[0] != 1:
            _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: block_table has {block_table.shape[0]} sequences, seq_lens "
                                                 f"{seq_lens.shape[0]}, free_count {free_count.shape[0]} entries")
        if page_size <= 0:
            _bail(_lib.IQ2_ERR_ZERO_DIM, f"{op} expects non-zero dimensions")
        self._tensors = (block_table, seq_lens, free_pages, free_count)
        self.sequences, self.table_width = block_table.shape
        self.num_pages, self.page_size = free_pages.shape[0], page_size
        self.device, self._index = block_table.device, index
        self._addresses = self._now()
        self._struct = _lib.KvPagesStruct(*self._addresses, self.sequences, self.table_width, self.num_pages, page_size)
        self._ptr = ctypes.addressof(self._struct)

    block_table = property(lambda self: self._tensors[0])
    seq_lens = property(lambda self: self._tensors[1])
    free_pages = property(lambda self: self._tensors[2])
    free_count = property(lambda self: self._tensors[3])

    def _now(self) -> tuple:
        return tuple([t.data_ptr() for t in self._tensors])

    @classmethod
    def empty(cls, num_pages: int, page_size: int, sequences: int, table_width: int, device="cuda") -> "KvPages":
        """Sequences without tokens over `num_pages` free pages, taken from page 0 on."""
        i32 = {"dtype": torch.int32, "device": device}
        return cls(torch.zeros((sequences, table_width), **i32), torch.zeros(sequences, **i32),
                   torch.arange(num_pages - 1, -1, -1, **i32), torch.full((1,), num_pages, **i32), page_size)


class KvStep:
    """Where the tokens of a step go, int32: slots [total] (page * page_size + row; -1: no place), positions [total],
    cu_seqlens_q [sequences + 1] (the first of each sequence's rows), cu_seqlens_k [sequences + 1] (the sums of the lengths
    after the step), granted [sequences] (the new tokens, or 0 where there was no place for them). `empty` makes one that
    steps of these sizes can be written to again and again."""

    __slots__ = ("slots", "positions", "cu_seqlens_q", "cu_seqlens_k", "granted", "_held", "_total", "_sequences", "_index",
                 "_addresses")

    @classmethod
    def empty(cls, pages: KvPages, total: int) -> "KvStep":
        self, n = cls(), pages.sequences
        room, rows = -(-total // 4) * 4, -(-(n + 1) // 4) * 4  # (each starts on 16 bytes)
        held = pages.seq_lens.new_empty(2 * room + 2 * rows + n)
        slots, positions, cu_q, cu_k, self.granted = held.split((room, room, rows, rows, n))
        self.slots, self.positions = (slots, positions) if room == total else (slots[:total], positions[:total])
        self.cu_seqlens_q, self.cu_seqlens_k = (cu_q, cu_k) if rows == n + 1 else (cu_q[:n + 1], cu_k[:n + 1])
        at = held.data_ptr()
        self._held = held  # (the addresses below stay good whatever becomes of the views)
        self._total, self._sequences, self._index = total, n, pages._index
        self._addresses = (at, at + 4 * room, at + 8 * room, at + 8 * room + 4 * rows, at + 8 * room + 8 * rows)
        return self


def kv_pages_step(pages: KvPages, new_lens: torch.Tensor, total_tokens: int, *, keep: torch.Tensor | None = None,
                  out: KvStep | None = None) -> KvStep:
    """A step of the sequences, in place: with `keep` (int32 [sequences]) sequence b keeps at most keep[b] of its tokens (0: it
    has ended; drafted tokens that were not taken go the same way), and the pages behind are free again; then it gets
    new_lens[b] (int32 [sequences]) more. Returns where these go, as `total_tokens` rows packed in the order of the sequences:
    `out` (a KvStep of these sizes) or a new KvStep. All of a sequence's new tokens get a place or none: none where they
    pass the rows or the table's width, and none from the first sequence on that needs more new pages than are left (but for
    those that need none). Such a sequence keeps what it had, granted is 0 and its rows have slot -1 and position 0, as have
    rows of no sequence."""
    op = "kv_pages_step"
    index, n = pages._index, pages.sequences
    new = _indices(op, index, "new_lens", new_lens, 1)
    if keep is not None:
        keep = _indices(op, index, "keep", keep, 1)
    if new.shape[0] != n or (keep is not None and keep.shape[0] != n):
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: block_table has {n} sequences, new_lens {new.shape[0]}"
                                             f"{'' if keep is None else f', keep {keep.shape[0]}'}")
    if not 0 <= total_tokens < 2 ** 31 - 1:
        _bail(_lib.IQ2_ERR_OVERFLOW, f"{op}: total_tokens={total_tokens} is negative or too large")
    if out is None:
        out = KvStep.empty(pages, total_tokens)
    elif out._total != total_tokens or out._sequences != n or out._index != index:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: out has {out._total} rows of {out._sequences} sequences on cuda:{out._index}, "
                                             f"expected {total_tokens} of {n} on cuda:{index}")
    if pages._now() != pages._addresses:
        _bail(_lib.IQ2_ERR_INVALID_ARGUMENT, f"{op}: the pages' tensors have moved since the KvPages was made")
    args = _lib.KV_STEP.pack(0 if keep is None else keep.data_ptr(), new.data_ptr(), total_tokens, *out._addresses)
    _call(index, _lib.load().iq2_kv_pages_step, pages._ptr, args)
    return out
