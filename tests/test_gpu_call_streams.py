"""Calls with `stream=`: what they return and work in is memory that nothing else is still going to write, and what the caller's stream still reads stays."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import PagePool, sample  # noqa: E402
from tests.test_gpu_attn_shared import Case  # noqa: E402

DEV = "cuda:0"
LATER = 60_000_000                                                  # clocks, some 30 ms: what is queued behind is written long after the call


def released_but_still_to_be_written(*likes):
    """Memory of the current stream's that is free again for torch, and that kernels which are queued on that stream will write."""
    torch.cuda._sleep(LATER)
    for like in likes:
        for t in [torch.empty_like(like) for _ in range(16)]:
            t.fill_(-5)


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_drawn_tokens(dtype, handle):
    g = torch.Generator(device=DEV).manual_seed(1)
    l, u = (torch.randn((7, 4001), device=DEV, generator=g) * 2).to(dtype), torch.rand(7, device=DEV, generator=g)
    want, s = sample(l, u, 0.8, 40, 0.9), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        released_but_still_to_be_written(*want)
        got = sample(l, u, 0.8, 40, 0.9, stream=s.cuda_stream if handle else s)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    # results that the current stream is still going to read, released on the host
    other, here = sample(l.flip(0), u, 0.8, 40, 0.9), torch.cuda.current_stream()
    torch.cuda.synchronize()
    r = sample(l, u, 0.8, 40, 0.9, stream=s)
    here.wait_stream(s)
    torch.cuda._sleep(LATER)
    copies = [x.clone() for x in r]
    del r
    with torch.cuda.stream(s):                                      # (ready on the call's stream)
        flipped = l.flip(0)
    more = [sample(flipped, u, 0.8, 40, 0.9, stream=s) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(copies, want)) and all(torch.equal(x, y) for m in more for x, y in zip(m, other))


def test_attention():
    c = Case(32, 4, 128, [6], [3000], [100, 3, 0, 50, 16, 77], seed=11)
    want, s = c.run(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(LATER)
        for n in (1 << 20, 4 << 20, 16 << 20, 64 << 20):            # the workspace's size and others
            for t in [torch.empty(n, dtype=torch.uint8, device=DEV) for _ in range(3)]:
                t.fill_(255)
        for t in [torch.empty_like(want) for _ in range(16)]:
            t.fill_(-5)
        got = c.run(stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_captured_on_another_stream():
    """A call on a stream that a capture has forked: its memory is the graph's."""
    c = Case(8, 2, 128, [2], [200], [40, 3], seed=2)
    l, u = torch.randn((5, 3001), device=DEV).bfloat16(), torch.rand(5, device=DEV)
    want, drawn, g, side = c.run(), sample(l, u), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        got, r = c.run(stream=side), sample(l, u, stream=side)
        here.wait_stream(side)
    junk = [torch.full((1 << 20,), 7.0, device=DEV) for _ in range(20)]
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(r, drawn)) and all(bool((j == 7).all()) for j in junk)


def test_a_pools_own_tables():
    """Tables that the pool makes are there when it is, whatever its stream still has to do: a call on another stream does not wait for that."""
    k, s = torch.zeros((1, 40, 8), device=DEV, dtype=torch.int16), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(LATER)
    pool = PagePool([k], 4, 6)
    row = pool.open(90, stream=s)
    forks = pool.fork(row, 2, stream=s)
    torch.cuda.synchronize()
    assert all(pool.tables[r, :6].tolist() == pool.pages_of(r) for r in (row, *forks)) and pool.pages_of(row) == [0, 1, 2, 3, 4, 5]
