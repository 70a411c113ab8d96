"""A pool over random lives on the device, where only a pool or a table without room may refuse, and what is refused changes nothing."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import EtxbError, PagePool  # noqa: E402

DEV, P = "cuda:0", 16


@pytest.mark.parametrize("seed", range(4))
def test_only_what_has_no_room_is_refused(seed):
    rng = random.Random(seed)
    N, ROWS, WIDTH = 60, 10, 9
    k, v = (torch.zeros((2, N, *s), device=DEV, dtype=torch.int16) for s in ((2, P), (3, P)))
    pool = PagePool([k, v], ROWS, WIDTH)
    want, stamp, done, moved = {}, 0, {}, 0

    def write(row, i0, i1):
        nonlocal stamp
        for i in range(i0, i1):
            stamp = stamp % 30000 + 1
            page = pool.pages_of(row)[i // P]
            k[:, page, :, i % P] = stamp
            v[:, page, :, i % P] = -stamp
            want[row].append(stamp)
    for step in range(90):
        op, rows = ("open", "fork", "extend", "close", "compact")[step % 5 if step < 15 else rng.randrange(5)], pool.rows()
        if not rows and op in ("fork", "extend", "close"):
            continue
        before = ([(r, pool.pages_of(r), pool.length_of(r)) for r in rows], pool.free_pages, pool.tables.clone(), k.clone(), v.clone())
        try:
            if op == "open":
                n = rng.randint(0, 170)
                r = pool.open(n)
                want[r] = []
                write(r, 0, n)
            elif op == "fork":
                r = rng.choice(rows)
                n = rng.randint(0, pool.length_of(r))
                for c in pool.fork(r, rng.randint(1, 4), n if rng.random() < 0.5 else None):
                    want[c] = want[r][:pool.length_of(c)]
            elif op == "extend":
                some = rng.sample(rows, rng.randint(1, len(rows)))
                old = {r: pool.length_of(r) for r in some}
                pool.extend(some, [old[r] + rng.randint(0, 30) for r in some])
                for r in some:
                    write(r, old[r], pool.length_of(r))
            elif op == "close":
                some = rng.sample(rows, rng.randint(1, len(rows) // 2 + 1))
                pool.close(some)
                for r in some:
                    del want[r]
            else:
                moved += pool.compact()
            done[op] = done.get(op, 0) + 1
        except (EtxbError, ValueError) as e:
            assert e.status == "E_FULL" if isinstance(e, EtxbError) else "a table has 9" in str(e), e
            assert op in ("open", "fork", "extend")
            assert before[:2] == ([(r, pool.pages_of(r), pool.length_of(r)) for r in pool.rows()], pool.free_pages)
            assert torch.equal(before[2], pool.tables) and torch.equal(before[3], k) and torch.equal(before[4], v)
        assert sorted(want) == pool.rows()
        for r in pool.rows():
            n = pool.length_of(r)
            tab = pool.tables[r, :len(pool.pages_of(r))].long()
            assert n == len(want[r]) and tab.tolist() == pool.pages_of(r)
            if n:
                assert k[1][tab].transpose(0, 1).reshape(2, -1)[1, :n].tolist() == want[r] and v[0][tab].transpose(0, 1).reshape(3, -1)[2, :n].tolist() == [-x for x in want[r]]
    assert sorted(done) == ["close", "compact", "extend", "fork", "open"] and moved > 0
    pool.close(pool.rows())
    with pytest.raises(EtxbError) as e:                                 # and there is an end to the pages
        for _ in range(ROWS):
            pool.open(WIDTH * P)
    assert e.value.status == "E_FULL" and len(pool.rows()) == N // WIDTH and pool.free_pages == N % WIDTH


def test_renumbering_more_rows_than_a_launch_lists():
    """2600 rows of which 2500 go on, in lists of 1975 and the rest: pages move once, every entry is renumbered once."""
    n = 2600
    k = torch.randint(-30000, 30000, (2, 3 * n, 8), device=DEV, dtype=torch.int16)
    pool = PagePool([k], n, 3)
    rows = [pool.open(40) for _ in range(n)]
    held = {r: k[:, pool.pages_of(r)].clone() for r in rows[100:]}
    pool.close(rows[:100])
    assert pool.compact() == 300 and pool.free_pages == 300
    tab = pool.tables.cpu()
    assert all(tab[r].tolist() == pool.pages_of(r) for r in rows[100:]) and max(max(pool.pages_of(r)) for r in rows[100:]) == 3 * n - 301
    assert all(torch.equal(k[:, pool.pages_of(r)], c) for r, c in held.items())
