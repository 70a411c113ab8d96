"""Pages of a paged KV cache: copied between pools, shared by forked sequences, moved together, given back (etxb_pages_update).

The layout is the programs': keys [layers][pages][NKV][HD / 8][16][8], values [layers][pages][NKV][HD][16]; a page is 16 positions of every layer and
tensor.  Nothing here looks inside a page, so any tensors [layers][pages][...] serve.  No counterpart in the reference, whose requests each own their
blocks (examples/vllm_llm/model.py:194-211)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import lib as L
from ._call import cuda_tensor, same_device, stream_handle


def _pool(name, tensors):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not 1 <= len(tensors) <= 4:
        raise ValueError(f"{name}: 1 to 4 tensors, got {len(tensors)}")
    for i, t in enumerate(tensors):
        cuda_tensor(f"{name}[{i}]", t, (t.dtype,) if isinstance(t, torch.Tensor) else (), inner=False)
        if t.dim() < 3 or t.shape[:2] != tensors[0].shape[:2] or not t[0, 0].is_contiguous() or t.numel() == 0:
            raise ValueError(f"{name}[{i}]: shape {tuple(t.shape)}, expected [layers][pages][...] with {tuple(tensors[0].shape[:2])} and pages without gaps")
    same_device(tensors[0].device, **{f"{name}[{i}]": t for i, t in enumerate(tensors)})
    return tensors


def _ids(name, v, n=None):
    a = np.ascontiguousarray(v, np.int32).reshape(-1)
    if not np.array_equal(a, np.asarray(v).reshape(-1)) or (n is not None and a.size != n):
        raise ValueError(f"{name}: {'whole numbers' if n is None else f'{n} whole numbers'}")
    return a


def _update(src, dst, src_ids=(), dst_ids=(), tables=None, sets=((), (), ()), share=((), 0, 0), remap=((), ()), stream=None):
    a, keep = L.PagesArgs(), []

    def lst(field, v):
        v = _ids(field, v)
        keep.append(v)
        setattr(a, field, v.ctypes.data if v.size else None)
        return v.size
    a.n_tensors, a.layers, a.src_pages, a.dst_pages = len(src), src[0].shape[0], src[0].shape[1], dst[0].shape[1]
    for i, (s, d) in enumerate(zip(src, dst)):
        z = s.element_size()
        a.t[i] = L.PageTensor(s.data_ptr(), d.data_ptr(), s.stride(0) * z, s.stride(1) * z, d.stride(0) * z, d.stride(1) * z, s[0, 0].numel() * z)
    a.n_copy = lst("src_ids", src_ids)
    if lst("dst_ids", dst_ids) != a.n_copy:
        raise ValueError(f"{a.n_copy} pages to copy to {len(dst_ids)}")
    if tables is not None:
        a.tables, a.table_stride, a.table_rows, a.table_width = tables.data_ptr(), tables.stride(0), tables.shape[0], tables.shape[1]
    a.n_set = lst("set_rows", sets[0])
    lst("set_cols", sets[1]), lst("set_pages", sets[2])
    a.n_share, a.share_from, a.shared = lst("share_rows", share[0]), share[1], share[2]
    a.n_remap = lst("remap_rows", remap[0])
    lst("remap_entries", remap[1])
    dev = src[0].device
    handle = stream_handle(dev, stream, [*src, *dst, tables])
    L.check(L.load().etxb_pages_update(dev.index, C.byref(a), C.sizeof(a), C.c_void_p(handle)))


def copy_pages(src, dst, src_ids, dst_ids, stream=None) -> None:
    """Page dst_ids[i] of the pool `dst` becomes page src_ids[i] of the pool `src`, in every layer and tensor (src and dst: lists of tensors, or one;
    the same pool, or two with pages of one size).  Within one pool no page may be both read and written; no page is written twice."""
    src, dst = _pool("src", src), _pool("dst", dst)
    if len(src) != len(dst) or src[0].shape[0] != dst[0].shape[0] or any(s.shape[2:] != d.shape[2:] or s.dtype != d.dtype for s, d in zip(src, dst)):
        raise ValueError("copy_pages: pools of the same tensors, layers and pages")
    same_device(src[0].device, dst=dst[0])
    _update(src, dst, _ids("src_ids", src_ids), _ids("dst_ids", dst_ids), stream=stream)


class PagePool:
    """The pages of a cache and the sequences that hold them.

    A sequence is a row of `tables` (int32 [max_seqs][max_pages] on the device: the block table its attention reads), with a length in positions.
    Forked sequences share the full pages of what they have in common; a page that is shared is never written, since only full pages are.  Pages are
    given out lowest first.  Which pages are whose is kept on the host; a call changes the tables and copies pages in one launch on its stream, so the
    steps that read them follow on the same stream (or wait for it).  A call that fails changes nothing."""

    def __init__(self, tensors, max_seqs: int, max_pages: int, tables=None, page_len: int = 16):
        self.tensors = _pool("tensors", tensors)
        dev = self.tensors[0].device
        if max_seqs < 1 or max_pages < 1 or page_len < 1:
            raise ValueError("PagePool: at least one sequence, page and position")
        if tables is None:
            tables = torch.zeros((max_seqs, max_pages), dtype=torch.int32, device=dev)
        self.tables = cuda_tensor("tables", tables, (torch.int32,), (max_seqs, max_pages))
        same_device(dev, tables=tables)
        self.page_len, self.n_pages = page_len, self.tensors[0].shape[1]
        self._users = np.zeros(self.n_pages, np.int32)          # sequences that hold a page
        self._pages = [None] * max_seqs                         # row -> its pages in order
        self._length = [0] * max_seqs

    # ---- what is where
    @property
    def free_pages(self) -> int:
        return int((self._users == 0).sum())

    def rows(self) -> list:
        return [r for r, p in enumerate(self._pages) if p is not None]

    def pages_of(self, row: int) -> list:
        return self._row(row).tolist()

    def length_of(self, row: int) -> int:
        self._row(row)
        return self._length[row]

    def _row(self, row):
        if not 0 <= row < len(self._pages) or self._pages[row] is None:
            raise ValueError(f"row {row} holds no sequence")
        return self._pages[row]

    def _need(self, length: int) -> int:
        if length < 0:
            raise ValueError(f"a length of {length} positions")
        n = -(-length // self.page_len)
        if n > self.tables.shape[1]:
            raise ValueError(f"{length} positions take {n} pages, a table has {self.tables.shape[1]}")
        return n

    def _take(self, n: int) -> np.ndarray:
        free = np.flatnonzero(self._users == 0)[:n]
        if free.size < n:
            raise RuntimeError(f"the pool has {free.size} free pages, {n} are needed")
        return free.astype(np.int32)

    def _free_rows(self, n: int) -> list:
        out = [r for r, p in enumerate(self._pages) if p is None][:n]
        if len(out) < n:
            raise RuntimeError(f"{len(out)} free rows in the tables, {n} are needed")
        return out

    # ---- calls
    def open(self, length: int, stream=None) -> int:
        """A new sequence with pages for `length` positions; returns its row."""
        n = self._need(length)
        row, pages = self._free_rows(1)[0], self._take(n)
        if n:
            _update(self.tensors, self.tensors, tables=self.tables, sets=(np.full(n, row), np.arange(n), pages), stream=stream)
        self._users[pages] += 1
        self._pages[row], self._length[row] = pages, length
        return row

    def extend(self, rows, length, stream=None) -> None:
        """Pages up to `length` positions (a number, or one per row) for each of `rows`; a length is never reduced."""
        rows = [int(rows)] if np.ndim(rows) == 0 else [int(r) for r in rows]
        lengths = [int(length)] * len(rows) if np.ndim(length) == 0 else [int(n) for n in length]
        if len(lengths) != len(rows) or len(set(rows)) != len(rows):
            raise ValueError("extend: each row once, with one length")
        for r, n in zip(rows, lengths):
            self._row(r)
            if n < self._length[r]:
                raise ValueError(f"row {r} has {self._length[r]} positions, not {n}")
        more = [self._need(n) - self._pages[r].size for r, n in zip(rows, lengths)]
        new = self._take(sum(more))
        if new.size:
            cols = np.concatenate([np.arange(self._pages[r].size, self._pages[r].size + m) for r, m in zip(rows, more)])
            _update(self.tensors, self.tensors, tables=self.tables, sets=(np.repeat(rows, more), cols, new), stream=stream)
        self._users[new] += 1
        at = 0
        for r, m, n in zip(rows, more, lengths):
            if m:
                self._pages[r] = np.concatenate([self._pages[r], new[at:at + m]])
                at += m
            self._length[r] = n

    def fork(self, row: int, n: int, length: int | None = None, stream=None) -> list:
        """n new sequences that continue `row` from `length` positions on (None: all of it): the full pages are shared, the last, partly filled one is
        copied for each.  Returns their rows."""
        pages = self._row(row)
        length = self._length[row] if length is None else int(length)
        if not 0 <= length <= self._length[row] or n < 0:
            raise ValueError(f"fork: {n} sequences from {length} positions of {self._length[row]}")
        full, part = divmod(length, self.page_len)
        rows, new = self._free_rows(n), self._take(n if part else 0)
        if n and (full or part):
            sets = (rows, np.full(n, full), new) if part else ((), (), ())
            _update(self.tensors, self.tensors, np.repeat(pages[full], n) if part else (), new, self.tables, sets, (rows, row, full), stream=stream)
        self._users[pages[:full]] += n
        self._users[new] += 1
        for i, r in enumerate(rows):
            self._pages[r] = np.concatenate([pages[:full], new[i:i + 1]]) if part else pages[:full].copy()
            self._length[r] = length
        return rows

    def close(self, rows) -> None:
        """The sequences end: pages that nobody else holds are free again (their contents and the rows' entries stay as they are)."""
        rows = [int(rows)] if np.ndim(rows) == 0 else [int(r) for r in rows]
        if len(set(rows)) != len(rows):
            raise ValueError("close: each row once")
        for r in rows:
            self._row(r)
        for r in rows:
            self._users[self._pages[r]] -= 1
            self._pages[r], self._length[r] = None, 0

    def compact(self, stream=None) -> int:
        """Moves pages until the ones in use are the lowest: the highest into the lowest hole, and so on.  Returns how many moved; the pool's pages from
        `n_pages - free_pages` on are then free."""
        used = np.flatnonzero(self._users)
        n = used.size
        high = used[used >= n][::-1]
        if high.size == 0:
            return 0
        low = np.flatnonzero(self._users[:n] == 0)
        rows = [r for r in self.rows() if self._pages[r].size]
        _update(self.tensors, self.tensors, high, low, self.tables, remap=(rows, [self._pages[r].size for r in rows]), stream=stream)
        to = np.arange(self.n_pages, dtype=np.int32)
        to[high] = low
        self._users[low] = self._users[high]
        self._users[high] = 0
        for r in rows:
            self._pages[r] = to[self._pages[r]]
        return int(high.size)
