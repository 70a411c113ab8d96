"""Decode attention for sequences that share prefixes (etxb_attn_shared): keys and values of a prefix are read once for all its sequences.

Beside the tiles of the step (ops/attn.py), which read every sequence's whole context; no counterpart in the reference."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import lib as L
from ._call import cuda_tensor, same_device, stream_handle

MAX_SEQS = 1024
_BAD = {1: "a table names a page outside the cache", 2: "a length lies outside its table", 4: "a wait inside the kernel ran past two seconds"}


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
    stream       a raw handle or torch stream; None is the current one

    Scores, statistics and sums are fp32.  A sequence without any position has the output 0.  Equal inputs give equal outputs."""
    cuda_tensor("kc", kc, (torch.bfloat16,), (None, None, None, 16, 8))
    pages, NKV, hd8 = kc.shape[:3]
    HD = 8 * hd8
    cuda_tensor("vc", vc, (torch.bfloat16,), (pages, NKV, HD, 16))
    if not kc[0].is_contiguous() or not vc[0].is_contiguous():
        raise ValueError("kc, vc: a page has no gaps")
    cuda_tensor("q", q, (torch.bfloat16,))
    if q.dim() == 3 and q.shape[2] != HD or q.dim() not in (2, 3) or (q.dim() == 2 and q.shape[1] % HD) or (q.dim() == 3 and q.shape[1] > 1 and q.stride(1) != HD):
        raise ValueError(f"q: shape {tuple(q.shape)} with strides {q.stride()}, expected [sequences][heads][{HD}] with adjoining heads")
    seqs, NH = q.shape[0], q.shape[1] if q.dim() == 3 else q.shape[1] // HD
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    cuda_tensor("out", out, (torch.bfloat16,), tuple(q.shape))
    if out.dim() == 3 and NH > 1 and out.stride(1) != HD:
        raise ValueError("out: the heads of a row adjoin")
    cuda_tensor("tables", tables, (torch.int32,), (seqs, None))
    cuda_tensor("lens", lens, (torch.int32,), (seqs,))
    cuda_tensor("prefix_tables", prefix_tables, (torch.int32,), (None, None))
    n_groups = prefix_tables.shape[0]
    cuda_tensor("prefix_lens", prefix_lens, (torch.int32,), (n_groups,))
    if status is not None:
        cuda_tensor("status", status, (torch.int32,), (1,))
    sizes = [seqs] if groups is None else [int(n) for n in groups]
    if len(sizes) != n_groups or any(n < 0 for n in sizes) or sum(sizes) != seqs:
        raise ValueError(f"groups: {n_groups} sizes of {seqs} sequences altogether, got {sizes}")
    if seqs > MAX_SEQS or n_groups > MAX_SEQS:
        raise ValueError(f"attn_shared: at most {MAX_SEQS} sequences and groups")
    same_device(q.device, kc=kc, vc=vc, out=out, tables=tables, lens=lens, prefix_tables=prefix_tables, prefix_lens=prefix_lens, status=status)
    first = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    a = L.AttnSharedArgs(q=q.data_ptr(), out=out.data_ptr(), kc=kc.data_ptr(), vc=vc.data_ptr(), tables=tables.data_ptr(), lens=lens.data_ptr(),
                         prefix_tables=prefix_tables.data_ptr(), prefix_lens=prefix_lens.data_ptr(), group_first=first.ctypes.data,
                         status=status.data_ptr() if status is not None else None,
                         q_stride=q.stride(0) if seqs > 1 else NH * HD, out_stride=out.stride(0) if seqs > 1 else NH * HD, k_stride=kc.stride(0) if pages > 1 else kc[0].numel(),
                         v_stride=vc.stride(0) if pages > 1 else vc[0].numel(), table_stride=tables.stride(0), prefix_stride=prefix_tables.stride(0),
                         seqs=seqs, groups=n_groups, NH=NH, NKV=NKV, HD=HD, pages=pages, table_width=tables.shape[1], prefix_width=prefix_tables.shape[1],
                         scale=HD ** -0.5 if scale is None else float(scale))
    lib, n, work = L.load(), C.c_size_t(), None
    L.check(lib.etxb_attn_shared_work(q.device.index, C.byref(a), C.sizeof(a), C.byref(n)))
    if n.value:                                                  # of this call alone: torch keeps it from others until the stream has passed
        work = torch.empty(n.value, dtype=torch.uint8, device=q.device)
        a.work, a.work_bytes = work.data_ptr(), n.value
    handle = stream_handle(q.device, stream, [q, out, kc, vc, tables, lens, prefix_tables, prefix_lens, status, work])
    L.check(lib.etxb_attn_shared(q.device.index, C.byref(a), C.sizeof(a), C.c_void_p(handle)))
    return out


def attn_shared_check(status) -> None:
    """Raises what `status` has recorded (waits for its device)."""
    v = int(status.item())
    if v:
        raise L.EtxbError(5 if v & 4 else 1, "attn_shared: " + "; ".join(text for bit, text in _BAD.items() if v & bit))
