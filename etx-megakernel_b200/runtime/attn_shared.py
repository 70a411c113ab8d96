"""Decode attention for sequences that share prefixes (etxb_attn_shared): keys and values of a prefix are read once for all its sequences.

A call of its own, beside the tiles of the step (ops/attn.py), which the programs use and which read every sequence's whole context.  No counterpart in the
reference."""
from __future__ import annotations

import ctypes as C
import struct
from array import array
from functools import lru_cache
from itertools import accumulate

import torch

from . import lib as L
from ._call import cuda_tensor, lend, other_stream, raw_stream, same_device

MAX_SEQS = 1024
_BF16, _I32 = (torch.bfloat16,), (torch.int32,)
_T, _BYTES = torch.Tensor, C.sizeof(L.AttnSharedArgs)
_pack = struct.Struct("11PN6q8ifi").pack                           # (the structure's fields in order, quicker than through ctypes)


@lru_cache(maxsize=1024)
def _work_bytes(index, first, seqs, groups, NH, NKV, HD, pages, width, prefix_width):
    """What the library asks for; it depends on nothing but these sizes (first: the groups' beginnings, as bytes)."""
    n = C.c_size_t()
    rc = L.load().etxb_attn_shared_work(index, _pack(*[0] * 8, C.cast(C.c_char_p(first), C.c_void_p).value, *[0] * 9, seqs, groups, NH, NKV, HD, pages, width, prefix_width, 1.0, 0), _BYTES, C.byref(n))
    if rc:
        L.check(rc)
    return n.value
_BAD = {1: "a table names a page outside the cache", 2: "a length lies outside its table", 4: "a wait inside the kernel ran past two seconds"}


def _check(q, kc, vc, tables, lens, prefix_tables, prefix_lens, out, status):
    """Raises what is wrong with the tensors."""
    cuda_tensor("kc", kc, _BF16, (None, None, None, 16, 8), inner=False)
    pages, NKV, hd8 = kc.shape[:3]
    HD = 8 * hd8
    if not HD or not NKV:
        raise ValueError(f"kc: {NKV} heads of {HD}")
    cuda_tensor("vc", vc, _BF16, (pages, NKV, HD, 16), inner=False)
    if kc.stride()[1:] != (hd8 * 128, 128, 8, 1) or vc.stride()[1:] != (HD * 16, 16, 1):
        raise ValueError("kc, vc: a page has no gaps")
    cuda_tensor("q", q, _BF16)
    shape = q.shape
    if len(shape) == 3 and (shape[2] != HD or (shape[1] > 1 and q.stride(1) != HD)) or len(shape) not in (2, 3) or (len(shape) == 2 and shape[1] % HD):
        raise ValueError(f"q: shape {tuple(shape)} with strides {q.stride()}, expected [sequences][heads][{HD}] with adjoining heads")
    if out is not None:
        cuda_tensor("out", out, _BF16, shape)
        if len(shape) == 3 and shape[1] > 1 and out.stride(1) != HD:
            raise ValueError("out: the heads of a row adjoin")
    cuda_tensor("tables", tables, _I32, (shape[0], None))
    cuda_tensor("lens", lens, _I32, (shape[0],))
    cuda_tensor("prefix_tables", prefix_tables, _I32, (None, None))
    cuda_tensor("prefix_lens", prefix_lens, _I32, (prefix_tables.shape[0],))
    if status is not None:
        cuda_tensor("status", status, _I32, (1,))
    same_device(q.device, kc=kc, vc=vc, out=out, tables=tables, lens=lens, prefix_tables=prefix_tables, prefix_lens=prefix_lens, status=status)


def attn_shared(q, kc, vc, tables, lens, prefix_tables, prefix_lens, groups=None, scale=None, out=None, status=None, stream=None):
    """Attention of the new position of every sequence: over the prefix of its group, then over positions of its own.

    q            [seqs][NH][HD] bf16 (or [seqs][NH * HD]; rows may lie further apart)
    kc, vc       one layer of the paged caches: [pages][NKV][HD / 8][16][8] and [pages][NKV][HD][16] bf16
    tables, lens int32 [seqs][any], [seqs]: each sequence's own pages and positions (0: none); the new position is in the cache already, and counted
    prefix_tables, prefix_lens   int32 [groups][any], [groups]: pages and positions that the sequences of a group share
    groups       how many sequences each group has, in order (None: one group of all)
    scale        None: HD ** -0.5
    out          bf16, shaped like q; returned
    status       int32 tensor [1] or None.  A page outside the cache or a length outside its table makes the outputs of the sequences concerned NaN and
                 sets a bit there, which `attn_shared_check` turns into an error
    stream       a raw handle or torch stream; None is the current one.  What the call reads and is given to write has to be ready there; what it returns is
                 memory of that stream, also kept for what the current one still does with it when it is released

    Scores, statistics and sums are fp32.  A sequence without any position has the output 0.  Equal inputs give equal outputs."""
    # What usually comes passes here in a few microseconds, which is what small calls take; all else goes through _check, which says what is wrong.
    plain = out is None and status is None and isinstance(q, _T) and isinstance(kc, _T) and isinstance(vc, _T) and isinstance(tables, _T) and \
        isinstance(lens, _T) and isinstance(prefix_tables, _T) and isinstance(prefix_lens, _T)
    if plain:
        shape, k, v, t, p, index = q.shape, kc.shape, vc.shape, tables.shape, prefix_tables.shape, q.get_device()
        plain = len(shape) == 3 and len(k) == 5 and len(t) == 2 and len(p) == 2 and index >= 0 and \
            q.dtype is kc.dtype is vc.dtype is torch.bfloat16 and tables.dtype is lens.dtype is prefix_tables.dtype is prefix_lens.dtype is torch.int32 and \
            kc.get_device() == vc.get_device() == tables.get_device() == lens.get_device() == prefix_tables.get_device() == prefix_lens.get_device() == index and \
            q.is_contiguous() and kc.is_contiguous() and vc.is_contiguous() and tables.is_contiguous() and prefix_tables.is_contiguous() and lens.is_contiguous() and \
            prefix_lens.is_contiguous() and k[3] == 16 and k[4] == 8 and shape[2] == 8 * k[2] and v == (k[0], k[1], shape[2], 16) and t[0] == shape[0] and \
            lens.shape == (shape[0],) and prefix_lens.shape == (p[0],)
    if not plain:
        _check(q, kc, vc, tables, lens, prefix_tables, prefix_lens, out, status)
        shape, k, t, p, index = q.shape, kc.shape, tables.shape, prefix_tables.shape, q.get_device()
    seqs, pages, NKV, HD, n_groups = shape[0], k[0], k[1], 8 * k[2], p[0]
    NH = shape[1] if len(shape) == 3 else shape[1] // HD
    sizes = (seqs,) if groups is None else [int(n) for n in groups]
    if len(sizes) != n_groups or min(sizes, default=0) < 0 or sum(sizes) != seqs:
        raise ValueError(f"groups: {n_groups} sizes of {seqs} sequences altogether, got {list(sizes)}")
    if seqs > MAX_SEQS or n_groups > MAX_SEQS:
        raise ValueError(f"attn_shared: at most {MAX_SEQS} sequences and groups")
    first = array("i", (0, *accumulate(sizes)))
    page = HD * NKV * 16
    n = _work_bytes(index, first.tobytes(), seqs, n_groups, NH, NKV, HD, pages, t[1], p[1])
    other = None if stream is None else other_stream(index, stream)
    if other is None:
        if out is None:
            out = torch.empty_like(q) if plain else torch.empty(shape, dtype=torch.bfloat16, device=q.device)
        work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None  # of this call alone: torch keeps it from others until the stream has passed
        handle = raw_stream(index)
    else:
        lend(other, (q, out, kc, vc, tables, lens, prefix_tables, prefix_lens, status))
        with torch.cuda.stream(other):                            # (memory of the call's stream: the current one's may still be written there)
            made = torch.empty(shape, dtype=torch.bfloat16, device=q.device) if out is None else None
            work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        lend(torch.cuda.current_stream(index), (made,))
        out, handle = made if out is None else out, other.cuda_stream
    a = _pack(q.data_ptr(), out.data_ptr(), kc.data_ptr(), vc.data_ptr(), tables.data_ptr(), lens.data_ptr(), prefix_tables.data_ptr(), prefix_lens.data_ptr(),
              first.buffer_info()[0], 0 if status is None else status.data_ptr(), work.data_ptr() if n else 0, n,
              q.stride(0) if seqs > 1 else NH * HD, out.stride(0) if seqs > 1 else NH * HD, kc.stride(0) if pages > 1 else page, vc.stride(0) if pages > 1 else page,
              tables.stride(0), prefix_tables.stride(0), seqs, n_groups, NH, NKV, HD, pages, t[1], p[1], HD ** -0.5 if scale is None else float(scale), 0)
    rc = L.load().etxb_attn_shared(index, a, _BYTES, handle)
    if rc:
        L.check(rc)
    return out


def attn_shared_check(status) -> None:
    """Raises what `status` has recorded (waits for its device)."""
    v = int(status.item())
    if v:
        raise L.EtxbError(5 if v & 4 else 1, "attn_shared: " + "; ".join(text for bit, text in _BAD.items() if v & bit))
