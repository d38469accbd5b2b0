"""Pages of a paged cache on the device: copying, forking, growing, freeing and compacting rows.

The reference is handed its block tables by the serving engine
(diffspec/runtime.py:869-875), whose allocator works on the host.  ``PagePool``
keeps the reference counts on the device, so that a step can fork requests
from a common prompt, grow their tables for draft tokens and cut them back
after rejection without a host round trip.  The tables are those that
``prefix_attention``, ``kernels`` and ``step`` read: int32 ``[rows, width]``, a
row's pages in order and -1 behind its last one.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _lib

__all__ = ["PagePool", "MAX_ROWS"]

STATUS_BAD_ROW = 1
STATUS_NO_PAGES = 2
STATUS_BAD_PAGE = 4
MAX_ROWS = 4096  # entries of a call's lists, and rows of a table


class PagePool:
    """Reference counts of the pages that a set of cache tensors share.

    ``caches``: tensors ``[num_pages, block_size, ...]`` of one device with
    the same first two dimensions, each page contiguous (the key and value
    caches of every layer).  ``ref_counts`` (int32 ``[num_pages]``, adopted,
    not copied) says how many rows hold each page; None starts with all
    pages free.  Free pages are taken in ascending order, for the rows of a
    call in their order.

    Row lists and lengths are sequences or int32 device tensors.  Sequences
    are checked here (``ValueError``); entries of device tensors that a call
    cannot take are left out and set bits of ``status`` (int32 device word):
    ``STATUS_BAD_ROW``, ``STATUS_NO_PAGES``, ``STATUS_BAD_PAGE``
    (include/ds355.h).  Calls on one pool run in order on the current stream,
    without host synchronisation when their lists are device tensors; a
    caller that changes streams orders them, from the second call on.
    """

    def __init__(self, caches: Sequence[torch.Tensor], ref_counts: torch.Tensor | None = None) -> None:
        caches = list(caches)
        if not caches:
            raise ValueError("a page pool needs at least one cache tensor")
        first = caches[0]
        if any(c.ndim < 2 or c.shape[:2] != first.shape[:2] for c in caches):
            raise ValueError("cache tensors must share [num_pages, block_size]")
        if min(first.shape[:2]) <= 0:
            raise ValueError("page counts and sizes must be positive")
        if any(not c[0].is_contiguous() for c in caches):
            raise ValueError("each page must be contiguous")
        if first.shape[0] > 1 and any(c.stride(0) < c[0].numel() for c in caches):
            raise ValueError("cache pages overlap")
        self.device = _lib.require_gpu(*caches, ref_counts)
        self.num_pages, self.block_size = first.shape[:2]
        if ref_counts is None:
            ref_counts = torch.zeros(self.num_pages, dtype=torch.int32, device=self.device)
        elif ref_counts.dtype != torch.int32 or ref_counts.shape != (self.num_pages,) or not ref_counts.is_contiguous():
            raise ValueError("ref_counts must be a contiguous int32 [num_pages] tensor")
        self.caches, self.ref_counts = caches, ref_counts
        pages = []
        for c in caches:
            at, step, size = c.data_ptr(), c.stride(0) * c.element_size(), c[0].numel() * c.element_size()
            pages += [at, step, size, 0 if (at | step | size) % 16 else 1]
        self._list = torch.tensor(pages, dtype=torch.int64, device=self.device)
        self._cache_args = (self._list.data_ptr(), len(caches), max(pages[2::4]), self.num_pages)
        size = int(_lib.load().ds_pages_workspace_bytes(self.num_pages))
        self._workspace = torch.zeros(size, dtype=torch.uint8, device=self.device)
        self._workspace_args = (self._workspace.data_ptr(), size)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        # Where the last compaction put each page; -1 for pages that were free.
        self.page_map = torch.arange(self.num_pages, dtype=torch.int32, device=self.device)
        # The first call may be on another stream than the one that fills these.
        torch.cuda.current_stream(self.device).synchronize()

    def _call(self, function: str, *args) -> None:
        with _lib.on_device(self.device):
            _lib.check(getattr(_lib.load(), function)(_lib.stream_handle(self.device), *args, self.status.data_ptr()))

    def _table(self, block_table: torch.Tensor) -> tuple:
        if block_table.dtype != torch.int32 or block_table.ndim != 2 or (block_table.shape[1] > 1
                                                                         and block_table.stride(1) != 1):
            raise ValueError("block_table must be int32 [rows, width] with unit last stride")
        if block_table.device != self.device:
            raise ValueError("block_table must be on the pool's device")
        if block_table.shape[0] > MAX_ROWS:
            raise _lib.UnsupportedShapeError(f"at most {MAX_ROWS} block table rows")
        return (self.ref_counts.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[0],
                block_table.shape[1])

    def _ints(self, values, name: str, limit: int | None, distinct: bool = False, count: int | None = None):
        """``values`` as an int32 device tensor; sequences are checked against [0, limit)."""
        if isinstance(values, torch.Tensor):
            if values.dtype != torch.int32 or values.ndim != 1 or not values.is_contiguous():
                raise ValueError(f"{name} must be a contiguous one-dimensional int32 tensor")
            if values.device != self.device:
                raise ValueError(f"{name} must be on the pool's device")
            tensor = values
        else:
            values = [int(v) for v in values]
            if any(v < 0 or (limit is not None and v >= limit) for v in values):
                raise ValueError(f"{name} must be between zero and {'the end' if limit is None else limit - 1}")
            if distinct and len(set(values)) != len(values):
                raise ValueError(f"{name} must be distinct")
            tensor = torch.tensor(values, dtype=torch.int32, device=self.device)
        if count is not None and tensor.numel() != count:
            raise ValueError(f"{name} needs one entry per row")
        return tensor

    def _lens(self, lens, count: int, width: int, name: str = "lens"):
        return self._ints(lens, name, width * self.block_size + 1, count=count)

    def copy(self, src, dst) -> None:
        """Pages ``dst[i]`` of every cache get the contents of pages ``src[i]``.

        Destinations are distinct, and none is the source of another entry
        (device tensors: the caller sees to it); counts and tables stay.
        """
        source = self._ints(src, "source pages", self.num_pages)
        target = self._ints(dst, "destination pages", self.num_pages, distinct=True, count=source.numel())
        if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
            moving = {int(s) for s, d in zip(src, dst) if int(s) != int(d)}
            if moving & {int(d) for d in dst}:
                raise ValueError("a destination page is also a source")
        elif _lib.DEBUG_CHECKS:
            pairs = [(s, d) for s, d in zip(source.tolist(), target.tolist())]
            if len({d for _, d in pairs}) != len(pairs) or {s for s, d in pairs if s != d} & {d for _, d in pairs}:
                raise ValueError("destination pages must be distinct and no source")
        self._call("ds_pages_copy", *self._cache_args, source.data_ptr(), target.data_ptr(), source.numel())

    def fork(self, block_table: torch.Tensor, parents, children, lens) -> None:
        """Rows ``children`` become the first ``lens`` tokens of rows ``parents``.

        A child first gives back the pages it holds; it then shares the
        parent's full pages, and a last partial page is copied, in every
        cache, to a page of its own.  Children are distinct and no parents.
        """
        table = self._table(block_table)
        rows = block_table.shape[0]
        p = self._ints(parents, "parents", rows)
        c = self._ints(children, "children", rows, distinct=True, count=p.numel())
        if not isinstance(parents, torch.Tensor) and not isinstance(children, torch.Tensor):
            if {int(x) for x in parents} & {int(x) for x in children}:
                raise ValueError("a child row is also a parent")
        n = self._lens(lens, p.numel(), block_table.shape[1])
        self._call("ds_pages_fork", *self._cache_args, *table, p.data_ptr(), c.data_ptr(), n.data_ptr(), p.numel(),
                   self.block_size, *self._workspace_args)

    def extend(self, block_table: torch.Tensor, rows, lens) -> None:
        """Rows get the free pages they lack for ``lens`` tokens; they never lose any."""
        table = self._table(block_table)
        r = self._ints(rows, "rows", block_table.shape[0], distinct=True)
        n = self._lens(lens, r.numel(), block_table.shape[1])
        self._call("ds_pages_extend", self.num_pages, *table, r.data_ptr(), n.data_ptr(), r.numel(), self.block_size)

    def free(self, block_table: torch.Tensor, rows, keep_lens=None) -> None:
        """Rows give back the pages behind their first ``keep_lens`` tokens (None: all pages)."""
        table = self._table(block_table)
        r = self._ints(rows, "rows", block_table.shape[0], distinct=True)
        n = None if keep_lens is None else self._ints(keep_lens, "keep_lens", None, count=r.numel())
        self._call("ds_pages_free", self.num_pages, *table, r.data_ptr(), _lib.ptr(n), r.numel(), self.block_size)

    def compact(self, block_table: torch.Tensor) -> torch.Tensor:
        """Moves held pages to the front of the pool: with n held pages, the
        k-th held page at or past n moves to the k-th free page below n, in
        every cache, the counts and ``block_table`` (which must hold every
        use of the pages).  Returns ``page_map``: int32 ``[num_pages]``, each
        page's new place, -1 where it was free."""
        table = self._table(block_table)
        self._call("ds_pages_compact", *self._cache_args, *table, self.page_map.data_ptr(), *self._workspace_args)
        return self.page_map
