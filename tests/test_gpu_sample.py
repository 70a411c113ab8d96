"""Drawing tokens (runtime.sample) against the definition in 64 bits, row by row on the CPU.

Tokens and numbers of kept tokens are whole numbers and have to be equal: the weights of the kernel are off by at most 2^-43 of the largest for
fp32 and by roundings of 64-bit numbers for 16 bits, and no border lies within 1e-11 of the sum from a random number or a share (checked for each row below).  A log-probability is the fp32 rounding of a sum of two
64-bit numbers; |value| < 64 gives an error of at most 2^-24 * 64 from the rounding and 1e-9 from the weights."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import EtxbError, sample  # noqa: E402,F401

DEV = "cuda:0"
NEG = float("-inf")


def oracle(l, u, T, k, p, mp):
    """(token, log-probability, kept, distance of u from the nearest border) of one row, in the order of the definition."""
    l = np.where(np.isnan(l), NEG, l.astype(np.float64))
    ids = np.nonzero(l > NEG)[0]
    if ids.size == 0:
        return -1, NEG, 0, 1.0
    ids = ids[np.argsort(-l[ids], kind="stable")]
    v = l[ids]
    if not T > 0:
        return int(ids[0]), 0.0, 1, 1.0
    d = np.where(v == v[0], 0.0, v - v[0] if np.isfinite(v[0]) else NEG)
    w = np.exp(d / np.float64(np.float32(T)))
    n = min(k, v.size) if k > 0 else v.size
    c = np.cumsum(w)
    margin = 1.0
    if p < 1:
        x = np.float64(np.float32(p)) * c[n - 1]
        before = np.concatenate([[0.0], c[:n - 1]])
        margin = min(margin, np.min(np.abs(before[1:] - x)) / c[n - 1]) if n > 1 else margin
        n = max(1, int((before < x).sum()))
    if mp > 0:
        n = max(1, min(n, int((w >= np.float64(np.float32(mp))).sum())))
    x = np.float64(np.float32(min(max(u, 0.0), 1 - 2.0 ** -24))) * c[n - 1]
    margin = min(margin, np.min(np.abs(c[:n] - x)) / c[n - 1])
    r = min(int((c[:n] <= x).sum()), n - 1)
    return int(ids[r]), float(d[r] / np.float64(np.float32(T)) - math.log(c[n - 1])), n, margin


def check(logits, u, T=1.0, k=0, p=1.0, mp=0.0, exact_margin=True, **kw):
    B, V = logits.shape
    as_list = lambda x: [x] * B if not isinstance(x, (list, tuple)) else list(x)  # noqa: E731
    ks, Ts, ps, mps = as_list(k), as_list(T), as_list(p), as_list(mp)
    args = {}
    for name, val, dt in (("temperature", T, torch.float32), ("top_k", k, torch.int32), ("top_p", p, torch.float32), ("min_p", mp, torch.float32)):
        args[name] = torch.tensor(val, dtype=dt, device=DEV) if isinstance(val, (list, tuple)) else val
    r = sample(logits, torch.tensor(u, dtype=torch.float32, device=DEV), **args, **kw)
    torch.cuda.synchronize()
    got = [x.cpu().tolist() for x in r]
    host = logits.float().cpu().numpy()
    for b in range(B):
        tok, lp, n, margin = oracle(host[b], u[b], Ts[b], ks[b], ps[b], mps[b])
        assert margin > 1e-11 or not exact_margin, f"row {b}: the case stands on a border ({margin})"
        assert (got[0][b], got[2][b]) == (tok, n), f"row {b}: token {got[0][b]} of {got[2][b]} kept, want {tok} of {n}"
        assert got[1][b] == lp or abs(got[1][b] - lp) <= 2 ** -18 + 1e-8, f"row {b}: log-probability {got[1][b]}, want {lp}"
    return r


def rows(B, V, dtype, seed, masked=0.0, std=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    l = torch.randn((B, V), device=DEV, generator=g) * std
    if masked:
        l[torch.rand((B, V), device=DEV, generator=g) < masked] = NEG
    return l.to(dtype)


ALL = [torch.bfloat16, torch.float16, torch.float32]
SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.3, 0, 0.95, 0.0), (0.9, 0, 1.0, 0.02), (2.0, 1000, 0.5, 0.001), (0.0, 7, 0.5, 0.5), (1.0, 1, 1.0, 0.0), (1.0, 0, 1e-9, 0.0)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 300, 1023, 5000, 32771, 151936])
def test_settings_and_sizes(V, dtype):
    B = len(SETTINGS)
    l = rows(B, V, dtype, V)
    u = np.random.default_rng(V).random(B).astype(np.float32).tolist()
    T, k, p, mp = (list(x) for x in zip(*SETTINGS))
    check(l, u, T, k, p, mp)


@pytest.mark.parametrize("dtype", ALL)
def test_largest_vocabulary_and_wide_batch(dtype):
    check(rows(2, 524288, dtype, 1), [0.3, 0.999], 1.0)
    l = rows(301, 1031, dtype, 2, masked=0.5)
    check(l, np.random.default_rng(3).random(301).astype(np.float32).tolist(), [0.5 + (i % 7) * 0.2 for i in range(301)], [(i * 13) % 200 for i in range(301)],
          [1.0 if i % 3 else 0.9 for i in range(301)], [0.0 if i % 4 else 0.05 for i in range(301)])


@pytest.mark.parametrize("dtype", ALL)
def test_first_and_last_numbers(dtype):
    """u = 0, the largest below 1, and what lies outside [0, 1): the first token of the order, and the last that has any weight."""
    l = rows(6, 999, dtype, 4)
    check(l, [0.0, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, float("nan")][:4] + [0.0, 0.0], 1.0, exact_margin=False)
    r = sample(l, torch.tensor([-1.0, float("nan"), float("-inf"), 0.0, 0.0, 0.0], device=DEV), temperature=1.0)
    assert r.tokens.tolist() == l.float().argmax(1).tolist()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("V", [37, 4099, 151936])
def test_masks_empty_rows_infinities_and_ties(V, dtype):
    lowest = torch.finfo(dtype).min
    l = rows(9, V, dtype, 5)
    l[0] = NEG                                                  # nothing is allowed
    l[1] = float("nan")                                         # nor here
    l[2] = NEG; l[2, V - 1] = -7.0                              # one token
    l[3] = lowest; l[3, V // 2] = lowest / 2                    # masked by the type's lowest value
    l[4] = lowest                                               # all of them: equal tokens
    l[5, V // 3] = float("inf"); l[5, V - 2] = float("inf")     # infinite logits share everything
    l[6, ::2] = float("nan")
    l[7] = 1.5                                                  # equal tokens everywhere
    l[8] = 0.0; l[8, ::3] = -0.0                                # zeros of both signs are equal
    u = [0.5, 0.5, 0.9, 0.2, 0.613, 0.7, 0.31, 0.777, 0.4001]
    for T, k, p, mp in ((1.0, 0, 1.0, 0.0), (0.8, 20, 1.0, 0.0), (1.0, 0, 0.8013, 0.0), (1.0, 0, 1.0, 0.5), (0.0, 0, 1.0, 0.0), (1e30, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0)):
        check(l, u, T, k, p, mp, exact_margin=False)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("off,V", [(0, 524288), (3, 524240)])
def test_values_that_occur_more_often_than_16_bits_hold(off, V, dtype):
    lowest = torch.finfo(dtype).min
    big = rows(12, 524288, dtype, 15)
    l = big[:, off:off + V]
    l[0] = lowest; l[0, 70001:200000] = 3.0
    l[1] = lowest
    l[2] = -0.0
    l[3] = 0.0; l[3, ::2] = -0.0
    l[4] = 2.5; l[4, 1::2] = -0.0; l[4, 3::4] = 0.0
    l[5] = NEG; l[5, V - 70000:] = -1.0
    l[6] = float("nan"); l[6, 123456:123460] = 4.0
    l[7] = float("inf"); l[7, :300000] = 1.0
    l[8] = 1.0; l[8, 32767:65535] = 2.0; l[8, 131071:196606] = 0.5
    l[9, 100:400000] = lowest
    l[10, 5000:77000] = 11.0
    u = [0.5, 0.4999, 0.9, 0.2, 0.613, 0.7, 0.31, 0.777, 0.4001, 0.55, 0.123, 0.987]
    for T, k, p, mp in ((1.0, 0, 1.0, 0.0), (0.8, 100001, 1.0, 0.0), (1.0, 0, 0.8013, 0.0), (0.0, 0, 1.0, 0.0), (3.0, 0, 1.0, 0.5)):
        check(l, u, T, k, p, mp, exact_margin=False)


@pytest.mark.parametrize("rows_, V", [(3, 65536), (90, 131072)])
@pytest.mark.parametrize("dtype,T", [(torch.bfloat16, 4e37), (torch.float16, 1.5e4)])
def test_every_value_occurs(dtype, T, rows_, V):
    """All 16-bit patterns but the infinite ones, in any order, NaN among them; blocks that share rows, and one for each."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    bits = torch.where(bits == float("inf"), torch.ones_like(bits), bits)
    g = torch.Generator().manual_seed(31)
    l = torch.stack([bits.repeat(V // 65536)[torch.randperm(V, generator=g)] for _ in range(3)]).to(DEV)
    l = l.repeat(rows_ // 3, 1)
    u = torch.rand(rows_, generator=g).tolist()
    for k, p, mp in ((0, 1.0, 0.0), (30001, 0.7, 0.0), (0, 0.6, 0.9)):
        if rows_ == 3:
            check(l, u, T, k, p, mp)
            continue
        r = sample(l, torch.tensor(u, device=DEV), T, k, p, mp)
        few = sample(l[3:6], torch.tensor(u[3:6], device=DEV), T, k, p, mp)
        assert torch.equal(r.tokens[3:6], few.tokens) and torch.equal(r.kept[3:6], few.kept) and torch.equal(r.logprobs[3:6], few.logprobs)
        tok, _, n, margin = oracle(l[0].float().cpu().numpy(), u[0], T, k, p, mp)
        assert margin > 1e-11 and (int(r.tokens[0]), int(r.kept[0])) == (tok, n)


@pytest.mark.parametrize("dtype", ALL)
def test_more_rows_than_blocks_at_once(dtype):
    """So many long rows that a block has a whole one; the same rows a few at a time are shared by several blocks."""
    B, V = 150, 66003
    l = rows(B, V, dtype, 16, masked=0.3)
    l[7] = l[7].abs().neg(); l[9] = torch.finfo(dtype).min; l[11] = NEG
    u = torch.rand(B, device=DEV, generator=torch.Generator(device=DEV).manual_seed(17))
    T = torch.tensor([(0.0, 0.7, 1.0, 2.5)[i % 4] for i in range(B)], device=DEV)
    k = torch.tensor([(0, 50, 30000)[i % 3] for i in range(B)], dtype=torch.int32, device=DEV)
    p = torch.tensor([(1.0, 0.9)[i % 2] for i in range(B)], device=DEV)
    m = torch.tensor([(0.0, 0.0, 0.0, 0.0, 0.01)[i % 5] for i in range(B)], device=DEV)
    r = sample(l, u, T, k, p, m)
    for b in range(0, B, 3):
        few = sample(l[b:b + 3], u[b:b + 3].clone(), T[b:b + 3], k[b:b + 3], p[b:b + 3], m[b:b + 3])
        assert torch.equal(r.tokens[b:b + 3], few.tokens) and torch.equal(r.kept[b:b + 3], few.kept)
        assert bool(((r.logprobs[b:b + 3] == few.logprobs) | ((r.logprobs[b:b + 3] - few.logprobs).abs() <= 2 ** -18)).all())
    for b in range(0, B, 10):
        tok, lp, n, margin = oracle(l[b].float().cpu().numpy(), float(u[b]), float(T[b]), int(k[b]), float(p[b]), float(m[b]))
        assert margin > 1e-11 and (int(r.tokens[b]), int(r.kept[b])) == (tok, n)


@pytest.mark.parametrize("dtype", ALL)
def test_settings_off_the_range(dtype):
    """Negative and not-a-number settings do what the documentation says: no cut, greedy for the temperature."""
    nan = float("nan")
    l = rows(8, 700, dtype, 6)
    u = [0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.8]
    r = sample(l, torch.tensor(u, device=DEV), torch.tensor([1, -1, nan, 1, 1, 1, 1, 1.0], device=DEV), torch.tensor([-5, 0, 0, 10 ** 9, 0, 0, 0, 0], dtype=torch.int32, device=DEV),
               torch.tensor([1, 1, 1, 2.0, nan, -1.0, 1, 1], device=DEV), torch.tensor([0, 0, 0, 0, 0, 0, -1.0, 3.0], device=DEV))
    plain = sample(l, torch.tensor(u, device=DEV), 1.0)
    top = l.float().argmax(1)
    for b in (0, 3, 4, 6):
        assert r.tokens[b] == plain.tokens[b] and r.kept[b] == 700
    for b in (1, 2, 5, 7):
        assert r.tokens[b] == top[b] and r.kept[b] == 1


@pytest.mark.parametrize("dtype", ALL)
def test_strides_offsets_and_streams(dtype):
    """Rows further apart, beginnings off every alignment, outputs of the caller's, another stream, and the next step's input."""
    big = rows(7, 1300, dtype, 7)
    u = torch.rand(7, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    for off, V in ((0, 1300), (1, 1001), (3, 517), (5, 1290), (7, 64)):
        view = big[:, off:off + V]
        check(view, u.tolist(), 0.9, 40, 0.95)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        tok, nxt = torch.full((9,), 77, dtype=torch.int32, device=DEV), torch.full((9,), 78, dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        a = sample(view, u, 0.9, 40, 0.95, tokens=tok[1:8], next_tokens=nxt[1:8], stream=s.cuda_stream)
        s.synchronize()
        b = sample(view.contiguous(), u, 0.9, 40, 0.95)
        assert torch.equal(a.tokens, b.tokens) and torch.equal(nxt[1:8], b.tokens) and torch.equal(a.logprobs, b.logprobs)
        assert tok[[0, 8]].tolist() == [77, 77] and nxt[[0, 8]].tolist() == [78, 78]      # nothing behind the rows is touched


@pytest.mark.parametrize("dtype", ALL)
def test_the_next_input_is_a_token(dtype):
    """A row without an allowed token gives -1; what goes to the next step, which looks it up, is 0."""
    l = rows(3, 700, dtype, 21)
    l[1] = float("nan")
    nxt = torch.full((3,), 78, dtype=torch.int32, device=DEV)
    r = sample(l, torch.full((3,), 0.5, device=DEV), next_tokens=nxt)
    t = r.tokens.tolist()
    assert t[1] == -1 and nxt.tolist() == [t[0], 0, t[2]]


def test_captured_replayed_and_repeated():
    l = rows(5, 151936, torch.bfloat16, 8)
    u = torch.rand(5, device=DEV)
    want = sample(l, u, 0.8, 0, 0.95)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = sample(l, u, 0.8, 0, 0.95)
    for seed in (1, 2, 3):
        u.copy_(torch.rand(5, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)))
        l.copy_(rows(5, 151936, torch.bfloat16, 100 + seed))
        g.replay()
        want = sample(l, u, 0.8, 0, 0.95)
        assert all(torch.equal(x, y) for x, y in zip(r, want))
    first = [sample(l, u, 1.0) for _ in range(20)]
    assert all(torch.equal(x, y) for r in first for x, y in zip(r, first[0]))


def test_frequencies_follow_the_probabilities():
    """20000 rows of one distribution: each token's share within 5 standard deviations."""
    n, V = 20000, 12
    l = torch.linspace(1.0, -2.0, V, device=DEV).bfloat16()
    r = sample(l.expand(n, V).contiguous(), torch.rand(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)), 0.9)
    p = torch.softmax(l.double() / 0.9, 0).cpu().numpy()
    got = torch.bincount(r.tokens.long(), minlength=V).cpu().numpy() / n
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / n))
