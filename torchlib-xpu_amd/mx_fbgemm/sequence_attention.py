"""Attention over the rows of sequence features, and its cache for serving.

A sequence lookup (PoolingMode NONE) gives one row per event and the batch's
offsets; ``torch.ops.mx_fbgemm.jagged_attention`` attends within each list of
such rows, with gradients, and ``torch.ops.mx_fbgemm.jagged_rotary`` tells it
the events' positions (by the angles of ``rotary_table``).
``PagedSequenceCache`` keeps the keys and values of served sequences in pages, so
that a new event costs one row appended and one pass over its own history; it
may hold them in 4 bits, and rotate them on their way in.
"""

from __future__ import annotations

import itertools
from typing import Optional, Sequence

import torch

__all__ = ["PagedSequenceCache", "rotary_table"]


def rotary_table(positions: int, dim: int, base: float = 10000.0,
                 device: Optional[torch.device] = None) -> torch.Tensor:
    """Cosines and sines of the angles ``p * base ** (-2 i / dim)`` of positions
    p < ``positions`` and pairs i < ``dim / 2``: fp32 [positions, dim / 2, 2],
    rounded from 64 bits (far positions lose their angles in 32).  ``dim``, the
    values of a head that turn, is a multiple of 8.  Any other table of that
    shape (scaled positions, other frequencies) serves as well."""
    if positions < 0 or dim < 8 or dim % 8:
        raise ValueError(f"positions {positions} must not be negative, dim {dim} a positive multiple of 8")
    if not base > 0:
        raise ValueError(f"base {base} must be positive")
    device = torch.device(device) if device is not None else torch.device(
        "cuda", torch.cuda.current_device())
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * i / dim)
    return torch.stack([angles.cos(), angles.sin()], -1).float()


class PagedSequenceCache:
    """Keys and values of up to ``max_sequences`` sequences of up to
    ``max_length`` events each, in ``pages`` pages of ``page_size`` events
    ([pages, page_size, heads, head_dim] fp16 or bf16, the heads' widths a
    multiple of 8 up to 128).

    With ``bits=4`` a head's values are a row of head_dim / 2 bytes of codes, fp16
    scale and fp16 bias, as the 4-bit codec writes it (uint8 [pages, page_size,
    heads, head_dim / 2 + 4], a page's rows of one head next to each other): 3.8
    times the events in the same memory.  Rows come and queries go in ``dtype`` as
    before; a row with a value below fp16's range, or one that is no number, is NaN whole.

    With ``rotary`` (a table as ``rotary_table`` makes it, of ``max_length``
    positions at least) keys turn by their positions on the way in, and so do the
    queries given to ``append``; ``interleaved`` pairs neighbours instead of halves.

    The host keeps lengths and free pages, and what it tells the device goes through
    pinned memory, so no call waits for the device.  Nor can a call be captured in
    a graph, as its numbers are the host's: ``paged_cache_append`` and
    ``paged_cache_attention`` with numbers on the device can.
    Sequences are named by the number ``add`` gives; calls take any of them in
    any order, each at most once."""

    def __init__(self, pages: int, page_size: int, heads: int, head_dim: int,
                 max_sequences: int, max_length: int,
                 dtype: torch.dtype = torch.bfloat16,
                 device: Optional[torch.device] = None, bits: int = 16,
                 rotary: Optional[torch.Tensor] = None, interleaved: bool = False) -> None:
        if min(pages, page_size, heads, max_sequences, max_length) < 1:
            raise ValueError("pages, page_size, heads, max_sequences and max_length must be positive")
        if head_dim < 8 or head_dim > 128 or head_dim % 8:
            raise ValueError(f"head_dim {head_dim} must be a multiple of 8 up to 128")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype {dtype} must be float16 or bfloat16")
        device = torch.device(device) if device is not None else torch.device(
            "cuda", torch.cuda.current_device())
        if bits not in (4, 16):
            raise ValueError(f"bits {bits} must be 4 or 16")
        if rotary is not None:
            if rotary.dtype != torch.float32 or rotary.dim() != 3 or rotary.size(2) != 2:
                raise ValueError("rotary must be float32 [positions, pairs, 2]")
            if rotary.size(1) < 4 or rotary.size(1) % 4 or 2 * rotary.size(1) > head_dim:
                raise ValueError(f"{rotary.size(1)} pairs of rotary: a multiple of 4, at most half of head_dim")
            if rotary.size(0) < max_length:
                raise ValueError(f"rotary has {rotary.size(0)} positions for sequences of {max_length}")
        self.page_size, self.max_length, self.dtype, self.bits = page_size, max_length, dtype, bits
        # A view along the pairs is laid out here once, not in every call.
        self._rotary = rotary.contiguous() if rotary is not None else None
        self._interleaved = interleaved

        def tensor() -> torch.Tensor:
            if bits == 16:
                return torch.empty((pages, page_size, heads, head_dim), dtype=dtype, device=device)
            return torch.empty((pages, heads, page_size, head_dim // 2 + 4), dtype=torch.uint8,
                               device=device).transpose(1, 2)

        self.k, self.v = tensor(), tensor()
        if rotary is not None and rotary.device != self.k.device:
            raise ValueError(f"rotary is on {rotary.device}, the cache on {self.k.device}")
        width = -(-max_length // page_size)
        self._table = torch.full((max_sequences, width), -1, dtype=torch.int32, device=device)
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._free_pages = list(range(pages - 1, -1, -1))
        self._free_names = list(range(max_sequences - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    def length(self, sequence: int) -> int:
        """Events of a sequence."""
        return self._lengths[self._known(sequence)]

    def add(self) -> int:
        """A new, empty sequence."""
        if not self._free_names:
            raise RuntimeError(f"all {self._table.size(0)} sequences are in use")
        name = self._free_names.pop()
        self._pages[name], self._lengths[name] = [], 0
        return name

    def remove(self, sequence: int) -> None:
        """Ends a sequence; its pages are free again."""
        self._free_pages.extend(reversed(self._pages.pop(self._known(sequence))))
        del self._lengths[sequence]
        self._free_names.append(sequence)

    def append(self, sequences: Sequence[int], counts: Sequence[int], k: torch.Tensor,
               v: torch.Tensor, q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Adds ``counts[i]`` events to ``sequences[i]``: the rows of k and v
        ([sum(counts), heads, head_dim]) in that order.  Returns ``q`` ([sum(counts),
        H, head_dim], the same events' queries) turned by their positions, or as it
        is where the cache has no ``rotary``."""
        if len(counts) != len(sequences) or any(n < 0 for n in counts):
            raise ValueError("counts must hold one non-negative number per sequence")
        if k.size(0) != sum(counts):
            raise ValueError(f"k has {k.size(0)} rows for {sum(counts)} events")
        if q is not None and q.size(0) != k.size(0):
            raise ValueError(f"q has {q.size(0)} rows, k {k.size(0)}")
        if self.bits == 4 and k.dtype != self.dtype:  # (16-bit rows are checked against the cache itself)
            raise ValueError(f"k is {k.dtype}, the cache's rows are {self.dtype}")
        self._distinct(sequences)
        if not sequences:
            return q
        self._not_captured()
        starts = [self._lengths[s] for s in sequences]
        self._reserve(sequences, [a + n for a, n in zip(starts, counts)])
        # Offsets and starts in one copy to the device.
        both = self._to_device([0, *itertools.accumulate(counts), *starts])
        B = len(sequences)
        args = (k, v, both[: B + 1], both[B + 1:])
        if self._rotary is None:
            torch.ops.mx_fbgemm.paged_cache_append(*args, self.k, self.v, self._rows(sequences))
        else:
            turned = torch.ops.mx_fbgemm.paged_cache_append_rotary(
                q, *args, self._rotary, self.k, self.v, self._rows(sequences), self._interleaved)
            q = turned if q is not None else None
        for s, n in zip(sequences, counts):
            self._lengths[s] += n
        return q

    def attend(self, sequences: Sequence[int], q: torch.Tensor,
               scale: Optional[float] = None) -> torch.Tensor:
        """Attention of one query per sequence (q [len(sequences), H, head_dim],
        H a multiple of ``heads``) over all its events: [len(sequences), H,
        head_dim]."""
        self._distinct(sequences)
        if q.size(0) != len(sequences):
            raise ValueError(f"q has {q.size(0)} rows for {len(sequences)} sequences")
        self._not_captured()
        lengths = self._to_device([self._lengths[s] for s in sequences])
        return torch.ops.mx_fbgemm.paged_cache_attention(q, self.k, self.v, self._rows(sequences),
                                                         lengths, scale)

    def gather(self, sequences: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The sequences' keys and values, packed in that order ([events, heads,
        head_dim] of ``dtype``), and their offsets: what ``jagged_attention`` takes
        as k, v and k_offsets for several new events behind a cached history."""
        self._distinct(sequences)
        self._not_captured()
        lengths = [self._lengths[s] for s in sequences]
        offsets = self._to_device([0, *itertools.accumulate(lengths)])
        k, v = torch.ops.mx_fbgemm.paged_cache_gather(self.k, self.v, self._rows(sequences), offsets,
                                                      sum(lengths), self.dtype)
        return k, v, offsets

    # -- host side ----------------------------------------------------------

    def _known(self, sequence: int) -> int:
        if sequence not in self._lengths:
            raise KeyError(f"no sequence {sequence}")
        return sequence

    def _distinct(self, sequences: Sequence[int]) -> None:
        for s in sequences:
            self._known(s)
        if len(set(sequences)) != len(sequences):
            raise ValueError("a sequence is named twice")

    def _not_captured(self) -> None:
        """A replay would copy from pinned memory that holds other numbers by then."""
        if self._table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedSequenceCache's calls cannot be captured in a graph")

    def _to_device(self, numbers: list[int]) -> torch.Tensor:
        """The numbers on the device, enqueued: from pinned memory, which torch's host
        allocator keeps until the copy has run (one from pageable memory would wait
        for all work of the stream)."""
        device = self._table.device
        pinned = device.type == "cuda"
        return torch.tensor(numbers, dtype=torch.int32, pin_memory=pinned).to(device, non_blocking=pinned)

    def _rows(self, sequences: Sequence[int]) -> torch.Tensor:
        """The table's rows of the sequences, as wide as their longest."""
        width = max(1, max((len(self._pages[s]) for s in sequences), default=0))
        table = self._table[:, :width]
        if list(sequences) == list(range(len(sequences))):
            return table[: len(sequences)]
        return table.index_select(0, self._to_device(list(sequences)))

    def _reserve(self, sequences: Sequence[int], lengths: list[int]) -> None:
        """Pages for the sequences to grow to `lengths`; all of them, or none."""
        grow = [-(-n // self.page_size) - len(self._pages[s]) for s, n in zip(sequences, lengths)]
        if any(n > self.max_length for n in lengths):
            raise RuntimeError(f"a sequence would exceed max_length {self.max_length}")
        need = sum(g for g in grow if g > 0)
        if need > len(self._free_pages):
            raise RuntimeError(f"{need} pages needed, {len(self._free_pages)} free")
        rows, columns, pages = [], [], []
        for s, g in zip(sequences, grow):
            for _ in range(g):
                page = self._free_pages.pop()
                rows.append(s), columns.append(len(self._pages[s])), pages.append(page)
                self._pages[s].append(page)
        if pages:
            at = self._to_device([*rows, *columns, *pages]).view(3, -1)
            self._table[at[0].long(), at[1].long()] = at[2]
