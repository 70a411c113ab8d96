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


class HostPool(PagePool):
    """A pool over CPU tensors: numpy does what etxb_pages_update does, behind the library's checks of the lists."""

    def _carrier(self):
        def update(device, args, nbytes, stream):
            a = args.contents
            lst = lambda p, n: np.ctypeslib.as_array(C.cast(p, C.POINTER(C.c_int32)), (n,)).copy() if n else np.zeros(0, np.int32)  # noqa: E731
            src, dst = lst(a.src_ids, a.n_copy), lst(a.dst_ids, a.n_copy)
            assert len(set(dst)) == len(dst) and not set(dst) & set(src) and nbytes == C.sizeof(lib.PagesArgs)
            for t in self.tensors:
                for x, y in zip(src, dst):
                    t[:, int(y)] = t[:, int(x)]
            for r in lst(a.share_rows, a.n_share):
                self.tables[int(r), :a.shared] = self.tables[a.share_from, :a.shared]
            for r, c, p in zip(lst(a.set_rows, a.n_set), lst(a.set_cols, a.n_set), lst(a.set_pages, a.n_set)):
                self.tables[int(r), int(c)] = int(p)
            to = dict(zip(src.tolist(), dst.tolist()))
            for r, n in zip(lst(a.remap_rows, a.n_remap), lst(a.remap_entries, a.n_remap)):
                for c in range(n):
                    self.tables[int(r), c] = to.get(int(self.tables[int(r), c]), int(self.tables[int(r), c]))
            self.calls = getattr(self, "calls", 0) + 1
            return getattr(self, "answer", 0)
        self._fn = lib.PAGES_FN(update)
        return C.cast(self._fn, C.c_void_p)

    def _stream(self, stream):
        return None


@pytest.fixture
def on_host(monkeypatch):
    import __graft_entry__ as ge
    ge.build()
    monkeypatch.setattr(pages, "cuda_tensor", lambda name, t, dt, shape=None, inner=True: t)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)


def users(pool):
    held = np.zeros(pool.n_pages, int)
    for r in pool.rows():
        held[pool.pages_of(r)] += 1
    return held


@pytest.mark.parametrize("seed", range(6))
def test_pool_over_random_lives(on_host, seed):
    """Every sequence keeps reading its own positions through its table whatever else happens: positions are written as (sequence, position) marks."""
    rng = random.Random(seed)
    P, N, ROWS, WIDTH = 4, 60, 9, 12
    t = torch.zeros((1, N, P), dtype=torch.int64)
    pool = HostPool([t], ROWS, WIDTH, page_len=P)
    want, stamp = {}, 0

    def write(row, i0, i1):
        nonlocal stamp
        for i in range(i0, i1):
            stamp += 1
            page = int(pool.tables[row, i // P])
            assert users(pool)[page] == 1                          # a shared page is never written
            t[0, page, i % P] = stamp
            want[row].append(stamp)
    for _ in range(300):
        op, rows = rng.choice(["open", "fork", "extend", "extend", "close", "compact"]), pool.rows()
        before = ([(r, pool.pages_of(r), pool.length_of(r)) for r in rows], pool.tables.clone(), t.clone())
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
                assert users(pool)[:N - pool.free_pages].all()
        except (RuntimeError, ValueError):                         # no room: nothing has changed
            assert before[0] == [(r, pool.pages_of(r), pool.length_of(r)) for r in pool.rows()] and torch.equal(before[1], pool.tables) and torch.equal(before[2], t)
        for r in pool.rows():
            assert pool.pages_of(r) == pool.tables[r, :len(pool.pages_of(r))].tolist()
            assert [int(t[0, pool.tables[r, i // P], i % P]) for i in range(pool.length_of(r))] == want[r]
        assert int((users(pool) == 0).sum()) == pool.free_pages


def test_pool_refusals(on_host):
    pool = HostPool([torch.zeros((1, 6, 4))], 3, 4, page_len=4)
    r = pool.open(7)
    for f, text in ((lambda: pool.open(17), "a table has 4"), (lambda: pool.open(-1), "length"), (lambda: pool.extend(r, 6), "not 6"), (lambda: pool.extend([r, r], 9), "once"),
                    (lambda: pool.extend(2, 9), "no sequence"), (lambda: pool.fork(r, 1, 8), "of 7"), (lambda: pool.fork(r, -1), "fork"), (lambda: pool.close([r, r]), "once"),
                    (lambda: pool.close(1), "no sequence"), (lambda: pool.pages_of(-1), "row -1 of 3"), (lambda: pool.open(2 ** 32 + 4), "32 bits"), (lambda: pool.fork(r, 2 ** 32), "32 bits"), (lambda: pool.extend([r], [8, 9]), "one length"), (lambda: pool.extend([r], 2 ** 40), "32 bits"),
                    (lambda: pool.close(0.5), "whole"), (lambda: pool.length_of(3), "row 3 of 3"), (lambda: pool.fork(r, 1, -1), "from -1")):
        with pytest.raises(ValueError, match=text):
            f()
    with pytest.raises(RuntimeError, match="free rows"):
        pool.fork(r, 3)
    pool.open(12)
    with pytest.raises(RuntimeError, match="free pages"):
        pool.extend(r, 16)
    assert pool.length_of(r) == 7


def test_what_cannot_be_carried_out_changes_nothing(on_host):
    """The device refuses (a status that is not 0): the books stay as they were."""
    pool = HostPool([torch.zeros((1, 9, 4))], 4, 4, page_len=4)
    r = pool.open(7)
    other = pool.open(3)
    pool.close(r)
    pool.answer = 3
    state = (pool.rows(), pool.pages_of(other), pool.free_pages)
    for f in (lambda: pool.open(5), lambda: pool.extend(other, 9), lambda: pool.fork(other, 2), lambda: pool.compact()):
        with pytest.raises(lib.EtxbError):
            f()
        assert (pool.rows(), pool.pages_of(other), pool.free_pages) == state and pool.length_of(other) == 3
    pool.answer = 0
    assert pool.compact() == 1 and pool.pages_of(other) == [0]


def test_pool_library_refusals():
    import __graft_entry__ as ge
    ge.build()
    h, a = C.c_void_p(), lib.PagesArgs(dst_pages=4, table_rows=2, table_width=2)
    fn = lib.load()
    for args in ((0, None, 0, 16), (0, C.byref(a), 8, 16), (0, C.byref(a), C.sizeof(a), 0), (64, C.byref(a), C.sizeof(a), 16), (-1, C.byref(a), C.sizeof(a), 16)):
        assert fn.etxb_pool_create(*args, None, C.byref(h)) == 1
    assert fn.etxb_pool_create(0, C.byref(a), C.sizeof(a), 16, None, None) == 1
    n = C.c_int32()
    assert fn.etxb_pool_open(None, 1, C.byref(n), None) == 1 and fn.etxb_pool_free(None, C.byref(n)) == 1 and fn.etxb_pool_destroy(None) == 0
    assert fn.etxb_pool_create(0, C.byref(a), C.sizeof(a), 16, None, C.byref(h)) == 0
    assert fn.etxb_pool_open(h, 1, None, None) == 1 and fn.etxb_pool_extend(h, None, None, 1, None) == 1 and fn.etxb_pool_close(h, None, 1) == 1
    assert fn.etxb_pool_fork(h, 0, 1, -1, None, None) == 1 and fn.etxb_pool_row(h, 0, None, None, -1, None) == 1 and fn.etxb_pool_free(h, None) == 1
    assert fn.etxb_pool_open(h, 0, C.byref(n), None) == 0 and fn.etxb_pool_open(h, 2 ** 31 - 1, C.byref(n), None) == 1
    assert fn.etxb_pool_destroy(h) == 0


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA tensor"):
        copy_pages([torch.zeros(1, 2, 8)], [torch.zeros(1, 2, 8)], [0], [1])
    with pytest.raises(ValueError, match="CUDA tensor"):
        PagePool([torch.zeros(1, 2, 8)], 1, 1)


def test_a_copied_pool_is_the_same_pool(on_host):
    import copy
    import gc
    pool = HostPool([torch.zeros((1, 8, 4), dtype=torch.int64)], 3, 4, page_len=4)
    r = pool.open(6)
    other = copy.copy(pool)
    del pool
    gc.collect()
    assert other.rows() == [r] and other.open(4) == 1 and other.free_pages == 5
    with pytest.raises((TypeError, ValueError)):
        copy.deepcopy(other)


@pytest.mark.parametrize("tables", [lambda: torch.zeros((1, 4), dtype=torch.int32).expand(3, 4), lambda: torch.zeros(20, dtype=torch.int32).as_strided((3, 4), (2, 1)),
                                    lambda: torch.zeros(20, dtype=torch.int32).as_strided((3, 4), (3, 1))])
def test_tables_whose_rows_overlap_are_refused(on_host, tables):
    """The library is told where the rows lie: an expanded tensor has memory for one, and the others would be written behind it."""
    with pytest.raises(ValueError, match="rows overlap"):
        HostPool([torch.zeros((1, 6, 4))], 3, 4, tables=tables(), page_len=4)
    one = torch.zeros(4, dtype=torch.int32).as_strided((1, 4), (0, 1))    # a single row has no stride to speak of
    pool = HostPool([torch.zeros((1, 6, 4))], 1, 4, tables=one, page_len=4)
    assert pool.open(7) == 0 and one[0, :2].tolist() == [0, 1]


def test_the_library_refuses_tables_whose_rows_overlap():
    import __graft_entry__ as ge
    ge.build()
    h, fn = C.c_void_p(), lib.load()
    for stride in (0, 2, -3):
        a = lib.PagesArgs(dst_pages=4, tables=1 << 24, table_stride=stride, table_rows=2, table_width=3)
        assert fn.etxb_pool_create(0, C.byref(a), C.sizeof(a), 16, None, C.byref(h)) == 1 and b"overlap" in fn.etxb_last_error()
    a.table_rows = 1
    assert fn.etxb_pool_create(0, C.byref(a), C.sizeof(a), 16, None, C.byref(h)) == 0 and fn.etxb_pool_destroy(h) == 0


@pytest.mark.parametrize("case,text", [
    (dict(tensor=dict(dst=(1 << 22), dst_layer=768)), "tensors overlap"),                          # tensor 1 goes where tensor 0 is read
    (dict(tensor=dict(src=(1 << 22), src_layer=768, dst=1 << 20)), "tensors overlap"),            # both go to one place
    (dict(tensor=dict(dst=(1 << 20) + 640)), "tensors overlap"),                                    # a layer further on
    (dict(tensor=dict(dst=(1 << 20) + 32)), "tensors overlap")])
def test_copies_of_one_tensor_into_another_ones_are_refused(case, text):
    """Pages of all tensors are copied at once, in no order: what one reads or writes no other one writes."""
    with pytest.raises(lib.EtxbError, match=text):
        call(src_ids=[1], dst_ids=[2], other=True, **case)


def layout(t0, t1, layers=3, pages=10, page=64, n=64, layer=640):
    import __graft_entry__ as ge
    ge.build()
    a = lib.PagesArgs(n_tensors=2, layers=layers, src_pages=pages, dst_pages=pages, n_copy=1)
    ids = np.array([pages, 1], np.int32)                                # (a page outside its pool: what comes so far is refused for that)
    a.src_ids, a.dst_ids = ids.ctypes.data, ids.ctypes.data + 4
    for i, at in enumerate((t0, t1)):
        a.t[i] = lib.PageTensor(at, at, layer, page, layer, page, n)
    assert lib.load().etxb_pages_update(0, C.byref(a), C.sizeof(a), None) == 1
    return lib.load().etxb_last_error().decode()


@pytest.mark.parametrize("base", [1 << 20, (1 << 40) + 4096])
def test_keys_and_values_in_one_tensor(base):
    """Views of one tensor whose pages lie between each other's, or whose layers do, are apart."""
    assert "outside" in layout(base, base + 64, page=128, layer=1280)               # [layers][pages][2][..]
    assert "outside" in layout(base + 64, base, page=128, layer=1280)
    assert "outside" in layout(base, base + 640, layer=1280)                        # [layers][2][pages][..]
    assert "outside" in layout(base, base + 1280 + 64, page=128, layer=1280)        # (another tensor's next layer: its pages still lie between)
    assert "outside" in layout(base, base + 640, layers=1)
    assert "overlap" in layout(base, base + 48, page=128, layer=1280)
    assert "overlap" in layout(base, base + 80, page=128, layer=1280)
    assert "overlap" in layout(base, base + 576, layer=1280)
    assert "overlap" in layout(base, base + 704, layer=1280)
    assert "overlap" in layout(base, base + 64, page=128, layer=1216)               # (layers that end inside a page's distance)
    assert "overlap" in layout(base, base)


@pytest.mark.parametrize("seed", range(4))
def test_what_counts_as_apart_is_apart(seed):
    """Random small layouts, against the bytes themselves."""
    rng = random.Random(seed)
    seen = set()
    for _ in range(400):
        layers, pages, n = rng.randint(1, 3), rng.randint(1, 4), 16 * rng.randint(1, 3)
        page = n + 16 * rng.randint(0, 4)
        layer = page * (pages - 1) + n + 16 * rng.randint(0, 12)
        d = 16 * rng.randint(-30, 30)
        mine = {l * layer + p * page + i for l in range(layers) for p in range(pages) for i in range(0, n, 16)}
        apart = not mine & {d + x for x in mine}
        says = "overlap" not in layout(1 << 20, (1 << 20) + d, layers, pages, page, n, layer)
        assert apart or not says                                        # (never taken for apart; some that are may be refused)
        seen.add((apart, says))
    assert (True, True) in seen and (False, False) in seen


@pytest.mark.parametrize("bad", [5, None, torch.zeros((0, 3, 4)), torch.zeros((1, 0, 4)), torch.zeros((1, 3, 0)), [torch.zeros((1, 3, 4)), torch.zeros(0)], [torch.zeros((2, 3))]])
def test_what_is_no_pool_is_a_value_error(on_host, bad):
    for f in (lambda: HostPool(bad, 2, 2), lambda: copy_pages(bad, [torch.zeros((1, 3, 4))], [0], [1]), lambda: copy_pages([torch.zeros((1, 3, 4))], bad, [0], [1])):
        with pytest.raises(ValueError, match="tensors|src|dst"):
            f()


@pytest.mark.parametrize("number", [np.int64, np.int32, torch.tensor, int])
def test_a_length_for_all_rows_is_any_whole_number(on_host, number):
    pool = HostPool([torch.zeros((1, 12, 4))], 3, 4, page_len=4)
    rows = [pool.open(3) for _ in range(3)]
    pool.extend(rows, number(9))
    assert [pool.length_of(r) for r in rows] == [9, 9, 9]
    pool.extend(np.array(rows), np.array([10, 11, 12]))
    assert [pool.length_of(r) for r in rows] == [10, 11, 12]
    with pytest.raises(ValueError, match="one length"):
        pool.extend(rows, [13])
