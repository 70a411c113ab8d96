"""Attention over shared prefixes (runtime.attn_shared) against softmax in 64 bits over each sequence's gathered positions.

Tolerance, derived: the kernel multiplies bf16 keys and queries exactly into fp32 sums (a score of magnitude s is off by at most about HD * 2^-24 of the sum
of its terms' magnitudes, here <= 2^-14 absolute), takes exp in fp32 (2^-22), and weights values with probabilities of at least 16 bits (2^-17 relative
each); every one of these moves the output by at most that share of the largest |value|, together below 2^-13.  The output is rounded once to bf16: half
a step, 2^-8 of its magnitude (bf16 has 8 significant bits: steps of 2^-7 between 1 and 2).  So |got - want| <= 2^-8 |want| + 2^-13 max|v|, taken with a factor of 2 on the second term for long sums."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import EtxbError, attn_shared, attn_shared_check  # noqa: E402

DEV = "cuda:0"


class Case:
    def __init__(self, NH, NKV, HD, sizes, plens, lens, seed=0, spare=3, fill=None, width=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        n = lambda x: -(-x // 16)  # noqa: E731
        need = sum(map(n, plens)) + sum(map(n, lens))
        pages = need + spare
        self.sizes, self.plens, self.lens_ = sizes, plens, lens
        self.NH, self.NKV, self.HD = NH, NKV, HD
        self.kc = torch.randn((pages, NKV, HD // 8, 16, 8), device=DEV, generator=g).bfloat16()
        self.vc = torch.randn((pages, NKV, HD, 16), device=DEV, generator=g).bfloat16()
        self.q = (torch.randn((len(lens), NH, HD), device=DEV, generator=g) * 1.5).bfloat16()
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        self.unused = order[need:]
        self.ptab = torch.full((len(plens), max([n(p) for p in plens] + [width])), -7, dtype=torch.int32, device=DEV)
        self.tab = torch.full((len(lens), max([n(x) for x in lens] + [width])), 1 << 30, dtype=torch.int32, device=DEV)   # entries behind a length are never looked at
        at = 0
        for tab, ls in ((self.ptab, plens), (self.tab, lens)):
            for i, ln in enumerate(ls):
                tab[i, :n(ln)] = order[at:at + n(ln)]
                if fill is not None and ln % 16:                  # what lies behind the last position
                    page = int(order[at + n(ln) - 1])
                    self.kc[page, :, :, ln % 16:] = fill
                    self.vc[page, :, :, ln % 16:] = fill
                at += n(ln)
        if fill is not None:
            self.kc[self.unused.long()] = fill
            self.vc[self.unused.long()] = fill
        self.pl = torch.tensor(plens, dtype=torch.int32, device=DEV)
        self.ln = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def run(self, **kw):
        return attn_shared(self.q, self.kc, self.vc, self.tab, self.ln, self.ptab, self.pl, groups=self.sizes, **kw)

    def rows(self, tab, n):
        p = tab[:-(-n // 16)].long()
        k = self.kc[p].permute(0, 3, 1, 2, 4).reshape(-1, self.NKV, self.HD)[:n]
        v = self.vc[p].permute(0, 3, 1, 2).reshape(-1, self.NKV, self.HD)[:n]
        return k, v

    def want(self, scale=None):
        G, b, out, vmax = self.NH // self.NKV, 0, [], []
        for g, size in enumerate(self.sizes):
            pk, pv = self.rows(self.ptab[g], self.plens[g])
            for i in range(b, b + size):
                k, v = self.rows(self.tab[i], self.lens_[i])
                k, v = torch.cat([pk, k]), torch.cat([pv, v])
                o = torch.zeros((self.NH, self.HD), dtype=torch.float64, device=DEV)
                for h in range(self.NKV):
                    if k.shape[0]:
                        s = self.q[i, h * G:(h + 1) * G].double() @ k[:, h].double().T * (scale or self.HD ** -0.5)
                        o[h * G:(h + 1) * G] = torch.softmax(s, 1) @ v[:, h].double()
                out.append(o)
                vmax.append(float(v.float().abs().max()) if v.numel() else 0.0)
            b += size
        return torch.stack(out), torch.tensor(vmax, device=DEV, dtype=torch.float64)[:, None, None]

    def check(self, out=None, **kw):
        out = self.run(**kw) if out is None else out
        assert out.shape[0] == len(self.lens_)
        want, vmax = self.want(kw.get("scale"))
        err = (out.double().view(want.shape) - want).abs()
        bound = want.abs() * 2.0 ** -8 + vmax * 2.0 ** -12
        assert bool((err <= bound).all()), f"worst {float((err - bound).max())} over the bound, error {float(err.max())} at {int(err.flatten().argmax())}"
        return out


@pytest.mark.parametrize("NH,NKV,HD", [(32, 4, 128), (8, 8, 128), (12, 2, 128), (16, 1, 64), (6, 3, 80), (4, 2, 256), (2, 1, 16), (10, 2, 96), (40, 8, 128)])
@pytest.mark.parametrize("lens", [([3], [100], [1, 17, 33]), ([1], [1], [0]), ([2, 1], [16, 300], [5, 0, 130]), ([5], [1037], [15, 16, 17, 31, 1])])
def test_shapes(NH, NKV, HD, lens):
    Case(NH, NKV, HD, *lens, seed=NH + HD).check()


@pytest.mark.parametrize("seqs", [1, 2, 15, 16, 17, 33, 64, 100])
def test_numbers_of_sequences(seqs):
    rng = np.random.default_rng(seqs)
    Case(32, 4, 128, [seqs], [700], [int(x) for x in rng.integers(0, 60, seqs)], seed=seqs).check()


@pytest.mark.parametrize("plen", [0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000, 5003, 40000])
def test_lengths_of_the_prefix(plen):
    Case(16, 2, 128, [4], [plen], [0, 1, 16, 200], seed=plen).check()


@pytest.mark.parametrize("own", [0, 1, 16, 100, 3000])
def test_nothing_shared(own):
    Case(8, 4, 64, [3], [0], [own, own // 2, own], seed=own).check()


@pytest.mark.parametrize("NH,NKV,HD,plen,own", [(8, 8, 64, 60001, [59, 422]), (16, 1, 128, 300011, [1, 40, 7]), (8, 2, 256, 30003, [5, 33]), (32, 8, 128, 9000, [4001, 5, 17, 3000, 900])])
def test_shares_of_many_tiles(NH, NKV, HD, plen, own):
    """Shares of tens of tiles that end inside a page and go on with short contexts."""
    c = Case(NH, NKV, HD, [len(own)], [plen], own, seed=plen)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.check(status=status)
    attn_shared_check(status)


def test_groups_of_all_sizes():
    """Empty groups, groups of one, groups without a prefix."""
    rng = np.random.default_rng(0)
    sizes = [0, 1, 7, 0, 20, 3, 1, 0]
    Case(12, 2, 128, sizes, [50, 400, 2003, 0, 77, 0, 16, 9], [int(x) for x in rng.integers(0, 90, 32)], seed=1).check()
    sizes = [1] * 40
    Case(8, 2, 64, sizes, [int(x) for x in rng.integers(0, 300, 40)], [int(x) for x in rng.integers(0, 40, 40)], seed=2).check()


def test_sequences_without_positions_are_zero():
    c = Case(8, 2, 128, [2, 2], [0, 40], [0, 5, 0, 0], seed=3)
    out = c.check()
    assert bool((out[0] == 0).all()) and not bool((out[2] == 0).all())


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -3e38])
def test_what_lies_behind_a_length_reaches_nothing(fill):
    Case(32, 4, 128, [3, 2], [1003, 45], [1, 0, 18, 130, 7], seed=4, fill=fill, width=80).check()
    Case(6, 3, 80, [3], [5], [1, 30, 15], seed=5, fill=fill).check()


def test_infinite_and_nan_values_where_they_count():
    """An infinite score, value or a NaN within the context reaches its own sequences and heads and no others."""
    c = Case(8, 2, 128, [2, 1], [300, 200], [40, 40, 40], seed=6)
    want = c.run()
    c.vc[int(c.tab[0, 1]), 1, 5, 3] = float("inf")                        # sequence 0, kv head 1, output element 5
    got = c.run()
    assert bool(torch.isinf(got[0, 4:, 5]).all())
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[0, 4:, 5] = False
    assert torch.equal(got[keep], want[keep])
    c.vc[int(c.tab[0, 1]), 1, 5, 3] = 0.0
    c.q[1, 2] = float("nan")
    got = c.run()
    assert bool(torch.isnan(got[1, 2]).all()) and not bool(torch.isnan(got[0]).any()) and not bool(torch.isnan(got[2]).any())


def test_large_scores_and_a_scale():
    """Scores of hundreds: the running maximum changes often and by much."""
    c = Case(16, 2, 128, [4], [900], [3, 90, 17, 44], seed=7)
    c.q *= 30
    # a score of up to 2500 has the rounding of its sum: 128 terms in fp32, at most 2^-13 here, which moves a probability by that share
    want, vmax = c.want()
    err = (c.run().double() - want).abs()
    assert bool((err <= want.abs() * 2.0 ** -8 + vmax * 2.0 ** -8).all())
    c.q /= 30
    c.check(scale=0.31)
    c.check(scale=1e-6)


def test_rising_scores():
    """Keys in the order of their scores: the maximum rises with every position."""
    c = Case(8, 2, 128, [2], [2000], [50, 50], seed=8)
    d = torch.zeros(128, device=DEV)
    d[0] = 1.0
    c.q.copy_(torch.randn_like(c.q) * 0.2)
    c.q[:, :, 0] = 8.0
    at = 0
    for page in c.ptab[0, :125].tolist():
        c.kc[page, :, 0, :, 0] = (torch.arange(at, at + 16, device=DEV).float() / 60.0).bfloat16()
        at += 16
    c.check()


def test_strides_and_outputs_in_place():
    """q inside a wider row (the qkv buffer), rows of the tables inside wider ones, caches of several layers, an output of the caller's."""
    c = Case(12, 2, 128, [3, 2], [333, 20], [9, 0, 48, 100, 1], seed=9)
    want = c.check()
    wide = torch.full((5, 12 * 128 + 512), 9.0, device=DEV).bfloat16()
    wide[:, :1536] = c.q.view(5, -1)
    kc = torch.zeros((4, *c.kc.shape), device=DEV).bfloat16(); kc[2] = c.kc
    vc = torch.zeros((4, *c.vc.shape), device=DEV).bfloat16(); vc[2] = c.vc
    tab = torch.zeros((9, 40), dtype=torch.int32, device=DEV); tab[2:7, 3:3 + c.tab.shape[1]] = c.tab
    out = torch.full((7, 1600), 5.0, device=DEV).bfloat16()
    got = attn_shared(wide[:, :1536], kc[2], vc[2], tab[2:7, 3:3 + c.tab.shape[1]], c.ln, c.ptab, c.pl, groups=[3, 2], out=out[1:6, :1536])
    assert torch.equal(got.reshape(5, 12, 128), want)
    assert bool((out[[0, 6]] == 5).all()) and bool((out[:, 1536:] == 5).all()) and bool((wide[:, 1536:] == 9).all())
    gapped = torch.zeros((c.kc.shape[0], 3, 16, 16, 8), device=DEV).bfloat16(); gapped[:, :2] = c.kc            # pages further apart
    got = attn_shared(c.q, gapped[:, :2], c.vc, c.tab, c.ln, c.ptab, c.pl, groups=[3, 2])
    assert torch.equal(got, want)


def test_cache_past_32_bits():
    """Pages beyond 4 GB of a cache."""
    c = Case(8, 8, 256, [2], [100], [20, 3], seed=10)
    pages = 45000                                                       # 65536 elements a page: 5.9 GB
    kc, vc = torch.zeros((pages, *c.kc.shape[1:]), device=DEV, dtype=torch.bfloat16), torch.zeros((pages, *c.vc.shape[1:]), device=DEV, dtype=torch.bfloat16)
    n = c.kc.shape[0]
    kc[pages - n:], vc[pages - n:] = c.kc, c.vc
    got = attn_shared(c.q, kc, vc, c.tab + (pages - n), c.ln, c.ptab + (pages - n), c.pl)
    c.check(out=got)


def test_streams_capture_and_repeats():
    c = Case(32, 4, 128, [6], [3000], [100, 3, 0, 50, 16, 77], seed=11)
    want = c.run()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = c.run(stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got, want)
    assert all(torch.equal(c.run(), want) for _ in range(10))
    graphs, outs = [], []
    for _ in range(2):                                                  # two graphs over the same inputs, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    c.pl.fill_(2500); c.ln.copy_(torch.tensor([1, 2, 3, 4, 5, 6], dtype=torch.int32)); c.q.mul_(-1)      # lengths are the device's
    c.plens, c.lens_ = [2500], [1, 2, 3, 4, 5, 6]
    c.tab[2, 0] = c.unused[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    c.check(out=outs[0])
    assert torch.equal(outs[0], outs[1])


def test_bad_pages_and_lengths():
    """They make the outputs they concern NaN and set the status; the other sequences are as before."""
    c = Case(8, 2, 128, [2, 2], [200, 100], [20, 33, 17, 5], seed=12)
    want = c.run()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert torch.equal(c.run(status=status), want)
    attn_shared_check(status)
    for what, where, value, rows, text in ((c.tab, (1, 2), -1, [1], "page"), (c.tab, (3, 0), c.kc.shape[0], [3], "page"), (c.ptab, (0, 5), 1 << 30, [0, 1], "page"),
                                           (c.ln, (2,), -1, [2], "length"), (c.ln, (0,), 49, [0], "length"), (c.pl, (1,), 16 * c.ptab.shape[1] + 1, [2, 3], "length")):
        old = what[where].clone()
        what[where] = value
        got = c.run(status=status)
        what[where] = old
        other = [r for r in range(4) if r not in rows]
        assert bool(torch.isnan(got[rows]).all()) and torch.equal(got[other], want[other])
        with pytest.raises(EtxbError, match=text):
            attn_shared_check(status)
        status.zero_()


def test_refusals():
    c = Case(8, 2, 128, [2], [20], [5, 3], seed=13)
    args = dict(q=c.q, kc=c.kc, vc=c.vc, tables=c.tab, lens=c.ln, prefix_tables=c.ptab, prefix_lens=c.pl)
    for bad, text in ((dict(q=c.q.float()), "dtype"), (dict(q=c.q[:, :, :64]), "q:"), (dict(q=c.q[:, :3].contiguous()), "multiple of NKV"), (dict(kc=c.kc[:, :, :8].contiguous()), "vc"),
                      (dict(vc=c.vc.transpose(2, 3)), "vc"), (dict(tables=c.tab[:1]), "tables"), (dict(tables=c.tab.long()), "dtype"), (dict(lens=c.ln[:1]), "lens"),
                      (dict(prefix_lens=c.pl[:0]), "prefix_lens"), (dict(groups=[1]), "groups"), (dict(groups=[3, -1]), "groups"), (dict(out=torch.empty_like(c.q).float()), "dtype"),
                      (dict(out=c.q[:1]), "out"), (dict(status=c.ln), "status"), (dict(tables=c.tab.cpu()), "CUDA")):
        with pytest.raises((ValueError, EtxbError), match=text):
            attn_shared(**{**args, **bad})
