"""Paged KV cache: pages of a fixed number of slots, and per sequence a table of them.

Beside the static layout of ``memory/kv_layout.py`` (one ``[max_seq, head_dim]`` block per layer, head, k | v and
sequence, reserved in full) this one gives a sequence pages as it grows, so its memory follows its length, and lets
sequences hold the same page.  A page id stands for that page in every layer: one table serves all of them.

``PagedKVSpec`` describes the pool, ``PageAllocator`` hands out page ids on the host, and ``PagedKVCache`` holds the
device tensors that ``backend/cuda_paged.py``'s operators work on, with host copies of table and lengths for the
bookkeeping (which rows need another page); nothing is read back from the device for it.
"""

from __future__ import annotations

from collections import Counter
from dataclasses import dataclass

import numpy as np

PAGE_SIZES = (8, 16, 32, 64, 128, 256)
HEAD_DIMS = (32, 64, 128)
_ITEM = {"float32": 4, "bfloat16": 2}


@dataclass(frozen=True)
class PagedKVSpec:
    layers: int
    kv_heads: int
    head_dim: int
    dtype: str          # "float32" or "bfloat16"
    page_size: int      # slots of a page
    num_pages: int      # of the pool, per layer and k | v
    rows: int           # sequences
    max_pages: int      # table entries of a row

    def validate(self) -> None:
        if self.dtype not in _ITEM:
            raise ValueError(f"unsupported dtype {self.dtype}")
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {self.page_size}")
        if self.head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {self.head_dim}")
        for name in ("layers", "kv_heads", "num_pages", "rows", "max_pages"):
            if getattr(self, name) <= 0:
                raise ValueError(f"{name} must be positive")

    @property
    def slots(self) -> int:
        """Slots that a row can hold."""
        return self.max_pages * self.page_size

    @property
    def nbytes(self) -> int:
        return 2 * self.layers * self.num_pages * self.kv_heads * self.page_size * self.head_dim * _ITEM[self.dtype]


class PageAllocator:
    """Free pages of a pool; taken lowest first, so a run is reproducible.  A page may have several holders (``share``) and
    is free again when the last one gave it back."""

    def __init__(self, num_pages: int) -> None:
        self._free = list(range(num_pages - 1, -1, -1))
        self._holders: dict[int, int] = {}

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self, count: int) -> list[int]:
        if count > len(self._free):
            raise MemoryError(f"{count} pages wanted, {len(self._free)} free")
        got = [self._free.pop() for _ in range(count)]
        self._holders.update((p, 1) for p in got)
        return got

    def holders(self, page: int) -> int:
        return self._holders.get(page, 0)

    def share(self, pages) -> None:
        """One holder more for each page."""
        for p in pages:
            if p not in self._holders:
                raise ValueError(f"page {p} is not taken")
        for p in pages:
            self._holders[p] += 1

    def give(self, pages) -> None:
        """One holder less for each page (all of them or, on an error, none)."""
        count = Counter(pages)
        for p, n in count.items():
            if n > self.holders(p):
                raise ValueError(f"page {p} is not taken" + (" as often" if p in self._holders else ""))
        for p, n in count.items():
            self._holders[p] -= n
            if not self._holders[p]:
                del self._holders[p]
        self._free = sorted(self._free + [p for p in count if p not in self._holders], reverse=True)


class PagedKVCache:
    """Device tensors of a paged cache, and the host's account of them.

    ``pages`` [layers, 2, num_pages, kv_heads, page_size, head_dim]; ``table`` [rows, max_pages] int32; with
    ``track`` the eviction state ``weights`` / ``slot_positions`` [layers, rows, kv_heads, slots].
    """

    def __init__(self, spec: PagedKVSpec, device="cuda", track: bool = False) -> None:
        import torch

        spec.validate()
        self.spec, self._torch = spec, torch
        dt = {"float32": torch.float32, "bfloat16": torch.bfloat16}[spec.dtype]
        self.pages = torch.zeros(spec.layers, 2, spec.num_pages, spec.kv_heads, spec.page_size, spec.head_dim, dtype=dt,
                                 device=device)
        self.table = torch.zeros(spec.rows, spec.max_pages, dtype=torch.int32, device=device)
        self.weights = self.slot_positions = None
        if track:
            shape = (spec.layers, spec.rows, spec.kv_heads, spec.slots)
            self.weights = torch.zeros(shape, dtype=torch.float32, device=device)
            self.slot_positions = torch.zeros(shape, dtype=torch.int32, device=device)
        self.allocator = PageAllocator(spec.num_pages)
        self.held: list[list[int]] = [[] for _ in range(spec.rows)]  # each row's pages, in the order of its table
        self._host_table = np.zeros((spec.rows, spec.max_pages), np.int32)

    def k(self, layer: int):
        return self.pages[layer, 0]

    def v(self, layer: int):
        return self.pages[layer, 1]

    def reserve(self, slots) -> bool:
        """Pages for ``slots[row]`` slots of every row (more than it holds already are kept); whether any was added.
        All or nothing: on MemoryError no row has changed.  The caller uploads the table (``upload``)."""
        spec = self.spec
        need = []
        for row, n in enumerate(slots):
            if n > spec.slots:
                raise ValueError(f"row {row}: {n} slots, the table holds {spec.slots}")
            need.append(max(-(-int(n) // spec.page_size) - len(self.held[row]), 0))
        got = self.allocator.take(sum(need))
        for row, count in enumerate(need):
            at = len(self.held[row])
            mine, got = got[:count], got[count:]
            self._host_table[row, at:at + count] = mine
            self.held[row] += mine
        return any(need)

    def upload(self) -> None:
        """The host's table to the device, on the current stream."""
        self.table.copy_(self._torch.from_numpy(self._host_table))

    def release(self, row: int) -> None:
        """Gives a row's pages back (the work that reads them must be enqueued before whatever takes them next)."""
        self.allocator.give(self.held[row])
        self.held[row] = []

    def trim(self, slots) -> None:
        """Gives back the pages behind ``slots[row]`` slots of every row.  A row cannot end inside a page that other rows
        hold too: its next token would be written there."""
        ps = self.spec.page_size
        for row, n in enumerate(slots):
            if n % ps and n // ps < len(self.held[row]) and self.allocator.holders(self.held[row][n // ps]) > 1:
                raise ValueError(f"row {row}: slot {n} lies in a page that other rows hold")
        for row, n in enumerate(slots):
            keep = -(-int(n) // ps)
            if len(self.held[row]) > keep:
                self.allocator.give(self.held[row][keep:])
                self.held[row] = self.held[row][:keep]

    def share_prompt(self, slots: int) -> None:
        """Every row's first full pages become row 0's (of ``slots`` slots that row 0 has); what the rows had in their place
        is given back.  Rows need not have any pages yet: a ``reserve`` behind it takes their tails."""
        full = slots // self.spec.page_size
        if full > len(self.held[0]):
            raise ValueError(f"{slots} slots fill {full} pages, row 0 has {len(self.held[0])} pages")
        shared = self.held[0][:full]
        for row in range(1, self.spec.rows):
            self.allocator.share(shared)
            self.allocator.give(self.held[row][:full])
            self.held[row] = shared + self.held[row][full:]
            self._host_table[row, :full] = shared
