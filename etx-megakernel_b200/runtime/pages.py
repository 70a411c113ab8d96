"""Pages of a paged KV cache: copied between pools, shared by forked sequences, moved together, given back (etxb_pages_update, etxb_pool_*).

The layout is the programs': keys [layers][pages][NKV][HD / 8][16][8], values [layers][pages][NKV][HD][16]; a page is 16 positions of every layer and
tensor.  Nothing here looks inside a page, so any tensors [layers][pages][...] serve.  No counterpart in the reference, whose requests each own their
blocks (examples/vllm_llm/model.py:194-211)."""
from __future__ import annotations

import ctypes as C
from array import array

import torch

from . import lib as L
from ._call import cuda_tensor, raw_stream, same_device, stream_handle

_BYTES = C.sizeof(L.PagesArgs)


def _pool(name, tensors):
    try:
        tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    except TypeError:
        raise ValueError(f"{name}: tensors, got {type(tensors).__name__}") from None
    if not 1 <= len(tensors) <= 4:
        raise ValueError(f"{name}: 1 to 4 tensors, got {len(tensors)}")
    for i, t in enumerate(tensors):
        cuda_tensor(f"{name}[{i}]", t, (t.dtype,) if isinstance(t, torch.Tensor) else (), inner=False)
        if t.dim() < 3 or t.shape[:2] != tensors[0].shape[:2] or t.numel() == 0 or not t[0, 0].is_contiguous():
            raise ValueError(f"{name}[{i}]: shape {tuple(t.shape)}, expected [layers][pages][...] with {tuple(tensors[0].shape[:2])} and pages without gaps")
    same_device(tensors[0].device, **{f"{name}[{i}]": t for i, t in enumerate(tensors)})
    return tensors


def _layout(src, dst):
    a = L.PagesArgs()
    a.n_tensors, a.layers, a.src_pages, a.dst_pages = len(src), src[0].shape[0], src[0].shape[1], dst[0].shape[1]
    for i, (s, d) in enumerate(zip(src, dst)):
        z = s.element_size()
        a.t[i] = L.PageTensor(s.data_ptr(), d.data_ptr(), s.stride(0) * z, s.stride(1) * z, d.stride(0) * z, d.stride(1) * z, s[0, 0].numel() * z)
    return a


def _ints(name, v):
    """`v` as a C array of 32-bit numbers (a number is one of them)."""
    if type(v) is not list:
        v = v.tolist() if hasattr(v, "tolist") else v
        v = v if isinstance(v, (list, tuple, range)) else (v,)
    try:
        out = array("i", v)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"{name}: whole numbers of 32 bits") from e
    return (C.c_int32 * len(out)).from_buffer(out)


def _int(name, v):
    """`v` as a 32-bit number (ctypes would cut a larger one)."""
    if type(v) is int and -2 ** 31 <= v < 2 ** 31:
        return v
    return _ints(name, [v])[0]


def _check(rc):
    """What the library refuses is the caller's error; a pool without room is not."""
    if rc:
        try:
            L.check(rc)
        except L.EtxbError as e:
            if e.status == "E_ARG":
                raise ValueError(str(e)) from None
            raise


def copy_pages(src, dst, src_ids, dst_ids, stream=None) -> None:
    """Page dst_ids[i] of the pool `dst` becomes page src_ids[i] of the pool `src`, in every layer and tensor (src and dst: lists of tensors, or one;
    the same pool, or two with pages of one size; pages of different tensors do not overlap).  Within one pool no page may be both read and written; no page is
    written twice."""
    src, dst = _pool("src", src), _pool("dst", dst)
    if len(src) != len(dst) or src[0].shape[0] != dst[0].shape[0] or any(s.shape[2:] != d.shape[2:] or s.dtype != d.dtype for s, d in zip(src, dst)):
        raise ValueError("copy_pages: pools of the same tensors, layers and pages")
    same_device(src[0].device, dst=dst[0])
    a, ids, to = _layout(src, dst), _ints("src_ids", src_ids), _ints("dst_ids", dst_ids)
    if len(ids) != len(to):
        raise ValueError(f"copy_pages: {len(ids)} pages to copy to {len(to)}")
    a.n_copy, a.src_ids, a.dst_ids = len(ids), C.addressof(ids), C.addressof(to)
    index = src[0].get_device()
    _check(L.load().etxb_pages_update(index, C.byref(a), _BYTES, stream_handle(index, stream, (*src, *dst))))


class _Books:
    """A pool of the library, given back with the last PagePool that refers to it (a copied object is a second one)."""

    def __init__(self, lib, handle):
        self.lib, self.handle = lib, handle

    def __del__(self):
        self.lib.etxb_pool_destroy(self.handle)


class PagePool:
    """The pages of a cache and the sequences that hold them.

    A sequence is a row of `tables` (int32 [max_seqs][max_pages] on the device: the block table its attention reads), with a length in positions.
    Forked sequences share the full pages of what they have in common; a page that is shared is never written, since only full pages are.  Pages are
    given out lowest first.  Which pages are whose is kept on the host; a call changes the tables and copies pages in one launch on its stream, so the
    steps that read them follow on the same stream (or wait for it).  A call that fails changes nothing: ValueError for what cannot be asked,
    EtxbError (E_FULL) where pages or rows run out.  Calls that change tables are not captured into a graph: a replay would change what is others' by then."""

    def __init__(self, tensors, max_seqs: int, max_pages: int, tables=None, page_len: int = 16):
        self.tensors = _pool("tensors", tensors)
        dev = self.tensors[0].device
        if max_seqs < 1 or max_pages < 1 or page_len < 1:
            raise ValueError("PagePool: at least one sequence, page and position")
        if tables is None:
            tables = torch.zeros((max_seqs, max_pages), dtype=torch.int32).to(dev)      # (there when the pool is: its calls may come on any stream)
        self.tables = cuda_tensor("tables", tables, (torch.int32,), (max_seqs, max_pages))
        same_device(dev, tables=tables)
        if max_seqs > 1 and tables.stride(0) < max_pages:
            raise ValueError(f"tables: rows overlap (stride {tables.stride(0)} below {max_pages})")
        self.page_len, self.n_pages, self._index = page_len, self.tensors[0].shape[1], self.tensors[0].get_device()
        a = _layout(self.tensors, self.tensors)
        a.tables, a.table_stride, a.table_rows, a.table_width = tables.data_ptr(), tables.stride(0) if max_seqs > 1 else max_pages, max_seqs, max_pages
        self._lib, self._h = L.load(), C.c_void_p()
        _check(self._lib.etxb_pool_create(self._index, C.byref(a), _BYTES, page_len, self._carrier(), C.byref(self._h)))
        self._books = _Books(self._lib, self._h)

    def _carrier(self):
        return None                                             # (the library's own etxb_pages_update)

    def _stream(self, stream):
        if stream is None:
            return raw_stream(self._index)
        return stream_handle(self._index, stream, (*self.tensors, self.tables))

    # ---- what is where
    @property
    def free_pages(self) -> int:
        n = C.c_int32()
        _check(self._lib.etxb_pool_free(self._h, C.byref(n)))
        return n.value

    def rows(self) -> list:
        n = C.c_int32()
        out = []
        for r in range(self.tables.shape[0]):
            _check(self._lib.etxb_pool_row(self._h, r, C.byref(n), None, 0, None))
            if n.value >= 0:
                out.append(r)
        return out

    def pages_of(self, row: int) -> list:
        n, buf = C.c_int32(), (C.c_int32 * self.tables.shape[1])()
        self.length_of(row)
        _check(self._lib.etxb_pool_row(self._h, row, None, buf, len(buf), C.byref(n)))
        return buf[:n.value]

    def length_of(self, row: int) -> int:
        n = C.c_int32()
        _check(self._lib.etxb_pool_row(self._h, _int("row", row), C.byref(n), None, 0, None))
        if n.value < 0:
            raise ValueError(f"row {row} holds no sequence")
        return n.value

    # ---- calls
    def open(self, length: int, stream=None) -> int:
        """A new sequence with pages for `length` positions; returns its row."""
        row = C.c_int32()
        _check(self._lib.etxb_pool_open(self._h, _int("length", length), C.byref(row), self._stream(stream)))
        return row.value

    def extend(self, rows, length, stream=None) -> None:
        """Pages up to `length` positions (a number, or one per row) for each of `rows`; a length is never reduced."""
        rows = _ints("rows", rows)
        length = length.tolist() if hasattr(length, "tolist") else length
        lengths = _ints("length", length if isinstance(length, (list, tuple, range)) else [length] * len(rows))
        if len(lengths) != len(rows):
            raise ValueError("extend: each row with one length")
        _check(self._lib.etxb_pool_extend(self._h, rows, lengths, len(rows), self._stream(stream)))

    def fork(self, row: int, n: int, length: int | None = None, stream=None) -> list:
        """n new sequences that continue `row` from `length` positions on (None: all of it; positions that are written by then): the full pages are shared, the last, partly filled one is
        copied for each.  Returns their rows."""
        if length is not None and length < 0:
            raise ValueError(f"fork: from {length} positions")
        row, n, length = _int("row", row), _int("n", n), -1 if length is None else _int("length", length)
        rows = (C.c_int32 * max(n, 0))()
        _check(self._lib.etxb_pool_fork(self._h, row, n, length, rows, self._stream(stream)))
        return rows[:]

    def close(self, rows) -> None:
        """The sequences end: pages that nobody else holds are free again (their contents and the rows' entries stay as they are)."""
        rows = _ints("rows", rows)
        _check(self._lib.etxb_pool_close(self._h, rows, len(rows)))

    def compact(self, stream=None) -> int:
        """Moves pages until the ones in use are the lowest: the highest into the lowest hole, and so on.  Returns how many moved; the pool's pages from
        `n_pages - free_pages` on are then free."""
        moved = C.c_int32()
        _check(self._lib.etxb_pool_compact(self._h, C.byref(moved), self._stream(stream)))
        return moved.value
