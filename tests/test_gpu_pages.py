"""Pages on the device against the same moves made with torch, bit for bit."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import PagePool, copy_pages  # noqa: E402

DEV = "cuda:0"


def pool_tensors(L, n, shapes, seed, dtype=torch.int16, gap=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for s in shapes:
        t = torch.randint(-30000, 30000, (L, n + gap, *s), device=DEV, generator=g, dtype=torch.int16).to(dtype)
        out.append(t[:, :n])
    return out


@pytest.mark.parametrize("L,shapes", [(1, [(8,)]), (3, [(4, 16, 16, 8), (4, 128, 16)]), (48, [(2, 8, 16, 8), (2, 64, 16)]), (2, [(8, 32, 16, 8), (8, 256, 16), (24,), (1000,)])])
@pytest.mark.parametrize("n_copy", [1, 2, 37])
def test_copies_between_and_within_pools(L, shapes, n_copy):
    rng = random.Random(L * 100 + n_copy)
    src, dst = pool_tensors(L, 80, shapes, 1, gap=3), pool_tensors(L, 90, shapes, 2)
    a, b = [rng.randrange(80) for _ in range(n_copy)], rng.sample(range(90), n_copy)      # a source may come twice
    want = [d.clone() for d in dst]
    for s, w in zip(src, want):
        w[:, b] = s[:, a]
    keep = [s.clone() for s in src]
    copy_pages(src, dst, a, b)
    assert all(torch.equal(x, y) for x, y in zip(dst, want)) and all(torch.equal(x, y) for x, y in zip(src, keep))
    ids = rng.sample(range(80), 2 * n_copy)
    want = [s.clone() for s in src]
    for w, k in zip(want, keep):
        w[:, ids[n_copy:]] = k[:, ids[:n_copy]]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    copy_pages(src, src, ids[:n_copy], ids[n_copy:], stream=s)
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(src, want))


def test_more_pages_than_one_launch_lists():
    """Ten thousand pages: the lists go in several launches."""
    n = 10000
    src, dst = pool_tensors(1, n, [(8,)], 3), pool_tensors(1, n, [(8,)], 4)
    g = torch.Generator().manual_seed(1)
    a, b = torch.randperm(n, generator=g).tolist(), torch.randperm(n, generator=g).tolist()
    copy_pages(src, dst, a, b)
    want = torch.empty_like(dst[0])
    want[:, b] = src[0][:, a]
    assert torch.equal(dst[0], want)


def test_pool_past_32_bits():
    """A pool of more than 4 GB: its last pages."""
    t = torch.zeros((3, 1030, 1 << 20), dtype=torch.int16, device=DEV)
    t[:, 0] = 5
    t[2, 1028] = 9
    copy_pages([t], [t], [0, 1028], [1029, 1])
    assert bool((t[:, 1029] == 5).all()) and bool((t[2, 1] == 9).all()) and bool((t[:, 2:1028] == 0).all())


@pytest.mark.parametrize("seed", range(3))
def test_pool_over_random_lives(seed):
    """Opened, forked, grown, closed, moved: what each sequence reads through its table on the device stays what was written."""
    rng = random.Random(seed)
    P, N, ROWS, WIDTH = 16, 90, 12, 9
    k, v = pool_tensors(2, N, [(2, 16), (3, 16)], seed)
    pool = PagePool([k, v], ROWS, WIDTH)
    want, stamp = {}, 0

    def write(row, i0, i1):
        nonlocal stamp
        for i in range(i0, i1):
            stamp = stamp % 30000 + 1
            page = pool.pages_of(row)[i // P]
            k[:, page, :, i % P] = stamp
            v[:, page, :, i % P] = -stamp
            want[row].append(stamp)
    for _ in range(40):
        op, rows = rng.choice(["open", "fork", "extend", "close", "compact"]), pool.rows()
        try:
            if op == "open":
                r = pool.open(rng.randint(0, 60))
                want[r] = []
                write(r, 0, pool.length_of(r))
            elif op == "fork" and rows:
                r = rng.choice(rows)
                n = rng.randint(0, pool.length_of(r))
                for c in pool.fork(r, rng.randint(0, 4), n if rng.random() < 0.5 else None):
                    want[c] = want[r][:pool.length_of(c)]
            elif op == "extend" and rows:
                some = rng.sample(rows, rng.randint(1, len(rows)))
                old = {r: pool.length_of(r) for r in some}
                pool.extend(some, [old[r] + rng.randint(0, 30) for r in some])
                for r in some:
                    write(r, old[r], pool.length_of(r))
            elif op == "close" and rows:
                some = rng.sample(rows, rng.randint(1, len(rows) // 2 + 1))
                pool.close(some)
                for r in some:
                    del want[r]
            elif op == "compact":
                pool.compact()
        except (RuntimeError, ValueError):
            pass
        for r in pool.rows():
            n = pool.length_of(r)
            tab = pool.tables[r, :len(pool.pages_of(r))].long()
            assert tab.tolist() == pool.pages_of(r)
            if n:
                assert k[1][tab].transpose(0, 1).reshape(2, -1)[1, :n].tolist() == want[r] and v[0][tab].transpose(0, 1).reshape(3, -1)[2, :n].tolist() == [-x for x in want[r]]


def test_many_rows_and_captured_calls():
    """Hundreds of sequences (lists of several launches), and a copy that is captured and replayed."""
    k, = pool_tensors(1, 9000, [(8,)], 7)
    pool = PagePool([k], 1200, 12)
    r = pool.open(100)
    rows = pool.fork(r, 1100)
    pool.extend(rows, 190)
    pool.close(rows[::2])
    n = pool.compact()
    # (7 + 1100 pages at the fork, 5 more each; 3307 stay in use, and of the rows that go on those from 440 on hold 5 pages above: 330 rows)
    assert n == 1650 and pool.tables[rows[1::2][7], :12].tolist() == pool.pages_of(rows[1::2][7])
    assert all(pool.tables[x, :12].tolist() == pool.pages_of(x) for x in rows[1::50])
    held = k[0, pool.pages_of(r)[-1]].clone()
    assert torch.equal(k[0, pool.pages_of(rows[3])[6]], held)
    src, dst = pool_tensors(2, 9, [(16,)], 8), pool_tensors(2, 9, [(16,)], 9)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        copy_pages(src, dst, [1, 2], [8, 0])
    src[0][:, 1:3] = 123
    g.replay()
    assert bool((dst[0][:, [8, 0]] == 123).all())


def test_books_are_not_captured():
    k, = pool_tensors(1, 40, [(8,)], 12)
    pool = PagePool([k], 6, 5)
    r = pool.open(37)
    before, g = pool.tables.clone(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        x = k + 1
        for call in (lambda: pool.open(20), lambda: pool.fork(r, 2), lambda: pool.extend([r], 60)):
            with pytest.raises(ValueError, match="not captured"):
                call()
    g.replay()
    assert pool.rows() == [r] and pool.length_of(r) == 37 and pool.free_pages == 37 and torch.equal(pool.tables, before) and torch.equal(x, k + 1)
    assert pool.fork(r, 2) == [1, 2]


def test_renumbering_in_several_launches():
    """5000 moves (a launch lists 1975 of them beside the rows): every table entry is renumbered once."""
    k, = pool_tensors(1, 12000, [(8,)], 11)
    pool = PagePool([k], 1000, 10)
    rows = [pool.open(160) for _ in range(1000)]
    keep = {r: k[0, pool.pages_of(r)].clone() for r in rows[500::50]}
    pool.close(rows[:500])
    assert pool.compact() == 5000 and pool.free_pages == 7000
    tab = pool.tables.cpu()
    for r in rows[500:]:
        assert tab[r].tolist() == pool.pages_of(r) and max(pool.pages_of(r)) < 5000
    for r, c in keep.items():
        assert torch.equal(k[0, pool.pages_of(r)], c)


def test_refusals_change_nothing():
    src, dst = pool_tensors(2, 9, [(16,)], 8), pool_tensors(2, 9, [(16,)], 9)
    keep = dst[0].clone()
    for bad in (([0], [0, 1]), ([9], [0]), ([0, 1], [2, 2]), ([0.5], [1])):
        with pytest.raises((ValueError, RuntimeError)):
            copy_pages(src, dst, *bad)
    with pytest.raises(ValueError, match="pools of the same"):
        copy_pages(src, pool_tensors(2, 9, [(8,)], 1), [0], [1])
    with pytest.raises(ValueError, match="without gaps"):
        copy_pages([src[0][:, :, ::2]], [dst[0][:, :, ::2]], [0], [1])
    assert torch.equal(dst[0], keep)
