"""Pages without a device: what the library refuses before its first CUDA call, and the pool's bookkeeping over random lives of sequences, with the
device's part played by numpy."""
import ctypes as C
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import PagePool, copy_pages, lib, pages  # noqa: E402

LISTS = ("src_ids", "dst_ids", "set_rows", "set_cols", "set_pages", "share_rows", "remap_rows", "remap_entries")


def call(nbytes=None, device=0, tensor=None, other=False, **f):
    """Two tensors of 3 layers and 10 pages of 64 bytes, in one pool (other: from one of 12 pages), tables of 4 rows of 6 entries."""
    import __graft_entry__ as ge
    ge.build()
    a, keep = lib.PagesArgs(n_tensors=2, layers=3, src_pages=10, dst_pages=10, tables=1 << 24, table_stride=8, table_rows=4, table_width=6), []
    for i in range(2):
        a.t[i] = lib.PageTensor((1 << 20) * (i + 1), (1 << 20) * (i + 1), 640, 64, 640, 64, 64)
        if other:
            a.t[i].src, a.t[i].src_layer = (1 << 22) * (i + 1), 768
    if other:
        a.src_pages = 12
    for k, v in (tensor or {}).items():
        setattr(a.t[1], k, v)
    counts = {"src_ids": "n_copy", "set_rows": "n_set", "share_rows": "n_share", "remap_rows": "n_remap"}
    for k, v in f.items():
        if k in LISTS and v is not None:
            arr = np.array(v, np.int32)
            keep.append(arr)
            setattr(a, k, arr.ctypes.data if arr.size else None)
            if k in counts:
                setattr(a, counts[k], arr.size)
        else:
            setattr(a, k, v)
    lib.check(lib.load().etxb_pages_update(device, C.byref(a), C.sizeof(a) if nbytes is None else nbytes, None))


COPY = dict(src_ids=[1, 1], dst_ids=[2, 3])
SET = dict(set_rows=[1], set_cols=[2], set_pages=[3])


@pytest.mark.parametrize("bad,text", [
    (dict(nbytes=8), "etxb_pages_args"), (dict(device=64), "device"), (dict(n_tensors=0), "tensors"), (dict(n_tensors=5), "tensors"), (dict(layers=0), "layers"),
    (dict(n_copy=-1), "negative"), (dict(n_copy=1), "null"), (dict(src_pages=0), "one page"), (dict(COPY, tensor=dict(src=None)), "null"),
    (dict(COPY, tensor=dict(dst=(1 << 21) + 8)), "multiples of 16"), (dict(COPY, tensor=dict(page_bytes=72, src_page=80, dst_page=80)), "multiples of 16"),
    (dict(COPY, tensor=dict(page_bytes=0)), "16 bytes"), (dict(COPY, tensor=dict(page_bytes=80)), "overlap"), (dict(COPY, tensor=dict(src_layer=624, dst_layer=624)), "overlap"),
    (dict(COPY, tensor=dict(src=(1 << 21) + 64)), "one pool or apart"), (dict(COPY, tensor=dict(src=1 << 23)), "every tensor"),
    (dict(src_ids=[10], dst_ids=[2]), "outside"), (dict(src_ids=[-1], dst_ids=[2]), "outside"), (dict(src_ids=[1], dst_ids=[10]), "outside"), (dict(src_ids=[1], dst_ids=[-1]), "outside"),
    (dict(src_ids=[1, 4], dst_ids=[2, 2]), "twice"), (dict(src_ids=[1, 2], dst_ids=[2, 3]), "read and written"), (dict(src_ids=[1], dst_ids=[1]), "read and written"),
    (dict(SET, tables=None), "tables"), (dict(SET, tables=(1 << 24) + 2), "tables"), (dict(SET, table_stride=5), "tables"),
    (dict(SET, set_rows=[4]), "outside"), (dict(SET, set_cols=[6]), "outside"), (dict(SET, set_pages=[10]), "outside"), (dict(SET, set_rows=[-1]), "outside"),
    (dict(set_rows=[1, 1], set_cols=[2, 2], set_pages=[3, 4]), "twice"), (dict(SET, share_rows=[1], share_from=0, shared=3), "shared and written"),
    (dict(SET, share_rows=[2], share_from=1, shared=3), "shared and written"), (dict(share_rows=[1], share_from=4, shared=1), "shared entries"),
    (dict(share_rows=[1], share_from=0, shared=7), "shared entries"), (dict(share_rows=[0], share_from=0, shared=1), "rows that share"), (dict(share_rows=[1, 1], share_from=0, shared=1), "rows that share"),
    (dict(COPY, remap_rows=[0], remap_entries=[3]), "one new number"), (dict(src_ids=[9], dst_ids=[0], remap_rows=[0], remap_entries=[7]), "renumbered rows"),
    (dict(src_ids=[9], dst_ids=[0], remap_rows=[0, 0], remap_entries=[2, 2]), "renumbered rows"), (dict(src_ids=[9], dst_ids=[0], remap_rows=[4], remap_entries=[2]), "renumbered rows"),
    (dict(src_ids=[9], dst_ids=[0], remap_rows=[0], remap_entries=[2], other=True), "one pool"), (dict(SET, src_ids=[9], dst_ids=[0], remap_rows=[0], remap_entries=[2]), "call of its own")])
def test_library_refuses(bad, text):
    with pytest.raises(lib.EtxbError, match=text) as e:
        call(**bad)
    assert e.value.status == "E_ARG"


def test_nothing_to_do_is_no_work():
    call()
    call(share_rows=[1, 2], share_from=0, shared=0)
    call(remap_rows=[1], remap_entries=[4])


class Device:
    """What etxb_pages_update does, on CPU tensors."""

    def __init__(self, monkeypatch):
        monkeypatch.setattr(pages, "cuda_tensor", lambda name, t, dt, shape=None, inner=True: t)
        monkeypatch.setattr(pages, "_update", self.update)

    def update(self, src, dst, src_ids=(), dst_ids=(), tables=None, sets=((), (), ()), share=((), 0, 0), remap=((), ()), stream=None):
        assert len(set(map(int, dst_ids))) == len(dst_ids) and not set(map(int, dst_ids)) & set(map(int, src_ids))
        for s, d in zip(src, dst):
            for a, b in zip(src_ids, dst_ids):
                d[:, int(b)] = s[:, int(a)]
        for r in share[0]:
            tables[r, :share[2]] = tables[share[1], :share[2]]
        for r, c, p in zip(*sets):
            tables[int(r), int(c)] = int(p)
        to = {int(a): int(b) for a, b in zip(src_ids, dst_ids)}
        for r, n in zip(*remap):
            for c in range(n):
                tables[r, c] = to.get(int(tables[r, c]), int(tables[r, c]))


@pytest.mark.parametrize("seed", range(6))
def test_pool_over_random_lives(monkeypatch, seed):
    """Every sequence keeps reading its own positions through its table whatever else happens: positions are written as (sequence, position) marks."""
    Device(monkeypatch)
    rng = random.Random(seed)
    P, N, ROWS, WIDTH = 4, 60, 9, 12
    t = torch.zeros((1, N, P), dtype=torch.int64)
    pool = PagePool([t], ROWS, WIDTH, page_len=P)
    want, stamp = {}, 0

    def write(row, i0, i1):
        nonlocal stamp
        for i in range(i0, i1):
            stamp += 1
            page = int(pool.tables[row, i // P])
            assert pool._users[page] == 1                          # a shared page is never written
            t[0, page, i % P] = stamp
            want[row].append(stamp)
    for _ in range(300):
        op, rows = rng.choice(["open", "fork", "extend", "extend", "close", "compact"]), pool.rows()
        before = (pool._users.copy(), [None if p is None else p.copy() for p in pool._pages], list(pool._length), pool.tables.clone())
        try:
            if op == "open":
                r = pool.open(rng.randint(0, 20))
                want[r] = []
                write(r, 0, pool.length_of(r))
            elif op == "fork" and rows:
                r = rng.choice(rows)
                n = rng.randint(0, pool.length_of(r))
                for c in pool.fork(r, rng.randint(0, 3), n if rng.random() < 0.5 else None):
                    want[c] = want[r][:pool.length_of(c)]
            elif op == "extend" and rows:
                some = rng.sample(rows, rng.randint(1, len(rows)))
                old = {r: pool.length_of(r) for r in some}
                pool.extend(some, [old[r] + rng.randint(0, 6) for r in some])
                for r in some:
                    write(r, old[r], pool.length_of(r))
            elif op == "close" and rows:
                some = rng.sample(rows, rng.randint(1, len(rows)))
                pool.close(some)
                for r in some:
                    del want[r]
            elif op == "compact":
                pool.compact()
                assert pool._users[:N - pool.free_pages].all()
        except (RuntimeError, ValueError):                         # no room: nothing has changed
            assert np.array_equal(before[0], pool._users) and before[2] == pool._length and torch.equal(before[3], pool.tables)
        for r in pool.rows():
            assert pool.pages_of(r) == pool.tables[r, :len(pool.pages_of(r))].tolist()
            assert [int(t[0, pool.tables[r, i // P], i % P]) for i in range(pool.length_of(r))] == want[r]
        held = np.zeros(N, int)
        for r in pool.rows():
            held[pool.pages_of(r)] += 1
        assert np.array_equal(held, pool._users)


def test_pool_refusals(monkeypatch):
    Device(monkeypatch)
    pool = PagePool([torch.zeros((1, 6, 4))], 3, 4, page_len=4)
    r = pool.open(7)
    for f, text in ((lambda: pool.open(17), "a table has 4"), (lambda: pool.open(-1), "length"), (lambda: pool.extend(r, 6), "not 6"), (lambda: pool.extend([r, r], 9), "once"),
                    (lambda: pool.extend(2, 9), "no sequence"), (lambda: pool.fork(r, 1, 8), "of 7"), (lambda: pool.fork(r, -1), "fork"), (lambda: pool.close([r, r]), "once"),
                    (lambda: pool.close(1), "no sequence"), (lambda: pool.pages_of(-1), "no sequence"), (lambda: pool.extend([r], [8, 9]), "one length")):
        with pytest.raises(ValueError, match=text):
            f()
    with pytest.raises(RuntimeError, match="free rows"):
        pool.fork(r, 3)
    pool.open(12)
    with pytest.raises(RuntimeError, match="free pages"):
        pool.extend(r, 16)
    assert pool.length_of(r) == 7


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA tensor"):
        copy_pages([torch.zeros(1, 2, 8)], [torch.zeros(1, 2, 8)], [0], [1])
    with pytest.raises(ValueError, match="CUDA tensor"):
        PagePool([torch.zeros(1, 2, 8)], 1, 1)
