"""A pool of cache pages shared by many sequences: who holds which page, on the GPU.

`PagePool` keeps the tensors that the page operations of `ops` work on (table, lens, refs; include/omnikv_hip.h,
okv_page_pool_t) and the list of arrays whose pages move together: the pools of `ops.PagedKV` and the codes and scales of
a paged `ops.KV8`, which read and write through the same `table`.  Sequence numbers and token counts are int32 tensors on the
GPU or lists of Python numbers.  With tensors nothing here waits for the GPU except `status()`, and a step of page operations
can be captured in a HIP graph; a list is copied to the GPU first, which waits for the stream and cannot be captured.

An 8-bit cache's open buffers belong to the sequences, not to the pages: `fork` copies a child's from its parent's, for
every cache that `add_cache` named.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Union

import torch

from . import ops

Numbers = Union[torch.Tensor, Sequence[int]]


class PagePool:
    def __init__(self, num_seqs: int, max_pages: int, num_pages: int, page_size: int, device="cuda"):
        if min(num_seqs, max_pages, num_pages, page_size) < 1:
            raise ValueError("a pool has at least one sequence, page per sequence, page and token per page")
        self.page_size = page_size
        self.table = torch.full((num_seqs, max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(num_seqs, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device=device)
        self.used = torch.zeros(1, dtype=torch.int32, device=device)  # pages in use, as of the last compact()
        self._status = torch.zeros(2, dtype=torch.int32, device=device)
        self._sum = torch.zeros(2, dtype=torch.int32, device=device)
        self._arrays: List[torch.Tensor] = []
        self._buffers: Optional[ops.PageBuffers] = None
        self._open: List[torch.Tensor] = []
        self._rows: Optional[ops.PageBuffers] = None

    def add(self, *arrays: torch.Tensor) -> None:
        """Arrays (num_pages, ...) whose pages move with the pool's (the pools of a PagedKV)."""
        both = ops.PageBuffers(self._arrays + list(arrays))
        if both.num_pages != self.refs.numel() or both.device != self.table.device:
            raise ValueError(f"arrays must hold {self.refs.numel()} pages on {self.table.device}")
        self._arrays, self._buffers = both.tensors, both

    def add_cache(self, cache: ops.KV8) -> None:
        """A paged 8-bit cache that goes through this pool's table: codes, scales, and its open buffers for fork."""
        if (cache.page_table is None or cache.page_table.data_ptr() != self.table.data_ptr()
                or cache.page_table.shape != self.table.shape or cache.page_size != self.page_size):
            raise ValueError("the cache must be paged through this pool's table")
        rows = ops.PageBuffers(self._open + [cache.open_k, cache.open_v]) if cache.open_k is not None else self._rows
        self.add(cache.k, cache.v, cache.k_scale, cache.v_scale)
        if rows is not None:
            self._open, self._rows = rows.tensors, rows

    def _numbers(self, x: Numbers) -> torch.Tensor:
        return x if isinstance(x, torch.Tensor) else torch.tensor(list(x), dtype=torch.int32, device=self.table.device)

    def _require_buffers(self) -> ops.PageBuffers:
        if self._buffers is None:
            raise ValueError("the pool has no arrays yet: add() or add_cache() first")
        return self._buffers

    def extend(self, seqs: Numbers, more: Numbers) -> None:
        """Sequences grow by `more` tokens each: pages for them (ops.pages_extend)."""
        ops.pages_extend(self.table, self.lens, self.refs, self._numbers(seqs), self._numbers(more), self.page_size, self._status)
        self._sum += self._status

    def fork(self, parents: Numbers, children: Numbers) -> None:
        """Children continue their parents (ops.pages_fork)."""
        ops.pages_fork(self.table, self.lens, self.refs, self._numbers(parents), self._numbers(children), self.page_size,
                       self._require_buffers(), self._status, self._rows)
        self._sum += self._status

    def free(self, seqs: Numbers) -> None:
        """Sequences end (ops.pages_free)."""
        ops.pages_free(self.table, self.lens, self.refs, self._numbers(seqs), self.page_size, self._status)
        self._sum += self._status

    def compact(self) -> None:
        """Used pages move to the lowest ones, in place (ops.pages_compact); `used` receives how many there are."""
        _, _, used = ops.pages_compact(self.table, self.refs, self._require_buffers(), self.table, self.refs)
        self.used.copy_(used)

    def status(self):
        """(pages the pool was short of, entries refused), summed over the calls since the last status(); waits for the GPU."""
        short, refused = self._sum.tolist()
        self._sum.zero_()
        return short, refused
