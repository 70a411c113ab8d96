"""Several answers to one prompt, as a program draws them: a batch over pages, a prompt's cache adopted and forked, tokens drawn on the device, and attention
over what the sequences share.  Steps over pages do the same arithmetic as steps over blocks of their own: everything is compared bit for bit; drawn tokens
are compared with the definition in 64 bits on the logits the step left."""
import struct

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.models import batched as BT  # noqa: E402
from etx_megakernel_b200.models import decode as D  # noqa: E402
from etx_megakernel_b200.models import dsv2 as M  # noqa: E402
from etx_megakernel_b200.models import qwen as Q  # noqa: E402
from etx_megakernel_b200.ops import batch as op_batch  # noqa: E402
from etx_megakernel_b200.runtime import lib as L  # noqa: E402
from etx_megakernel_b200.runtime import EtxbError, Sampling, attn_shared  # noqa: E402
from tests.test_gpu_sample import oracle  # noqa: E402

DEV = "cuda:0"
SMALL = Q.Dims(name="small", H=512, NH=8, NKV=2, HD=128, INTER=0, L=3, V=1504, qk_norm=True, moe=True, E=16, TOPK=4, MI=128, norm_topk=True)


@pytest.fixture(scope="module")
def weights():
    w = D.random_packed_weights(SMALL, 256, torch.device(DEV), seed=4)
    w["embed"].mul_(30.0)
    w["lm_head"].mul_(8.0)                                              # a distribution that is not flat
    return w


def batch(weights, B, **kw):
    return BT.BatchProgram(SMALL, weights, B, device=0, maxlen=256, steps=64, **kw)


@pytest.mark.parametrize("B", [1, 5, 32])
def test_a_batch_over_pages_equals_one_over_blocks(weights, B):
    prompts = np.random.default_rng(B).integers(0, SMALL.V, (B, 21))
    a, b = batch(weights, B), batch(weights, B, pages=4 * B + 3)
    want, got = a.generate(prompts, 15), b.generate(prompts, 15)
    assert np.array_equal(got, want) and np.array_equal(a.read("logits"), b.read("logits")) and np.array_equal(a.read("attn_out"), b.read("attn_out"))
    got = b.generate(prompts[::-1], 9)                                  # again, over pages that others have held
    assert np.array_equal(got, a.generate(prompts[::-1], 9))
    assert b.cache.free_pages == 4 * B + 3 - 2 * B
    a.close(); b.close()


@pytest.mark.parametrize("B,engine", [(3, "tc"), (24, "tc"), (4, "mma")])
def test_long_contexts_over_scattered_pages(weights, B, engine):
    """Contexts of several partitions, in pages that lie in any order: as blocks one after the other, and a fork as a sequence that was fed all of it."""
    prompts = np.random.default_rng(B).integers(0, SMALL.V, (B, 170))
    kw = dict(device=0, maxlen=256, steps=224, engine=engine)
    a, b = BT.BatchProgram(SMALL, weights, B, **kw), BT.BatchProgram(SMALL, weights, B, pages=14 * B + 20, **kw)
    assert [b.cache.open(0) for _ in range(B)] == list(range(B))
    for t in range(169):                                                # a position at a time: the columns take their pages in turn
        b.decode(prompts[:, t], t, 1)
    want, got = a.generate(prompts, 30), b.decode(prompts[:, 169], 169, 30)
    assert b.cache.pages_of(1)[:3] == [1, 1 + B, 1 + 2 * B]
    assert np.array_equal(got, want) and np.array_equal(a.read("logits"), b.read("logits"))
    b.release(range(1, B))
    used = b.cache.length_of(0)                                         # column 0 goes on as two, the others as they would alone
    assert used == 199 and b.fork(0, 1) == [1]
    again = b.decode([5, 5] + [1] * (B - 2), used, 20)
    assert np.array_equal(again[0], again[1])
    a.close(); b.close()


def test_forked_sequences_equal_sequences_of_their_own(weights):
    """A context of 37 positions adopted once and forked, against adopted for every column: the same logits to the bit at every length, the shared pages
    untouched, though the columns go different ways."""
    B, P = 6, 37
    one = D.DecodeProgram(SMALL, weights, device=0, maxlen=256, steps=64)
    prompt = np.random.default_rng(7).integers(0, SMALL.V, P)
    one.generate(prompt, 1)
    a, b = batch(weights, B, pages=30), batch(weights, B, pages=40)
    c = a.adopt(one, P)
    assert a.fork(c, B - 1) == [1, 2, 3, 4, 5]
    assert [b.adopt(one, P) for _ in range(B)] == list(range(B))
    assert 30 - a.cache.free_pages == 3 + 5 and 40 - b.cache.free_pages == 18
    shared = a.buf["kc"][:, a.cache.pages_of(0)[:2]].clone()
    tokens = np.random.default_rng(8).integers(0, SMALL.V, B)
    x, y = a.decode(tokens, P, 14), b.decode(tokens, P, 14)
    assert np.array_equal(x, y) and np.array_equal(a.read("logits"), b.read("logits")) and len({tuple(r) for r in x.tolist()}) > 1
    assert torch.equal(shared, a.buf["kc"][:, a.cache.pages_of(0)[:2]])
    # three answers end, the rest moves together and goes on
    a.release([1, 3, 4]); b.release([1, 3, 4])
    a.cache.compact()
    x, y = a.decode(x[:, -1], P + 14, 8), b.decode(y[:, -1], P + 14, 8)
    assert np.array_equal(x[[0, 2, 5]], y[[0, 2, 5]])
    assert np.array_equal(a.read("logits")[[0, 2, 5]], b.read("logits")[[0, 2, 5]])
    # attention of one layer over what the three share, and over their own pages behind it
    rows, layer = [0, 2, 5], 1
    tab, n = a.buf["block_tables"][rows], a.cache.length_of(0)
    q = torch.randn((3, SMALL.NH, 128), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    kc, vc = a.buf["kc"][layer], a.buf["vc"][layer]
    lens = torch.full((3,), n - 32, dtype=torch.int32, device=DEV)
    got = attn_shared(q, kc, vc, tab[:, 2:].contiguous(), lens, tab[:1, :2].contiguous(), torch.tensor([32], dtype=torch.int32, device=DEV))
    for i, r in enumerate(rows):
        p = a.cache.pages_of(r)
        k = kc[p].permute(0, 3, 1, 2, 4).reshape(-1, SMALL.NKV, 128)[:n].double()
        v = vc[p].permute(0, 3, 1, 2).reshape(-1, SMALL.NKV, 128)[:n].double()
        for h in range(SMALL.NH):
            w = torch.softmax(k[:, h // 4] @ q[i, h].double() * 128 ** -0.5, 0) @ v[:, h // 4]
            assert bool(((got[i, h].double() - w).abs() <= w.abs() * 2.0 ** -8 + float(v.abs().max()) * 2.0 ** -12).all())
    one.close(); a.close(); b.close()


def test_a_closed_column_leaves_the_others_pages_alone(weights):
    """A sequence ended through the pool itself: its column's entries name pages that the next one holds by then, and steps still must not write there."""
    one = D.DecodeProgram(SMALL, weights, device=0, maxlen=256, steps=64)
    prog, alone = batch(weights, 2, pages=8), batch(weights, 2, pages=8)
    one.generate(np.random.default_rng(1).integers(0, SMALL.V, 20), 1)
    assert prog.adopt(one, 20) == 0 and prog.adopt(one, 20) == 1
    prog.cache.close([0, 1])
    assert prog.adopt(one, 20) == 0 and prog.cache.pages_of(0) == [0, 1]
    alone.adopt(one, 20)
    prog.buf["block_tables"][1] = torch.tensor(prog.cache.pages_of(0) + [0] * 14, dtype=torch.int32)
    assert np.array_equal(prog.decode([3, 9], 20, 10)[0], alone.decode([3, 4], 20, 10)[0])
    assert np.array_equal(prog.read("logits")[0], alone.read("logits")[0])
    one.close(); prog.close(); alone.close()


def test_answers_draw_their_own_tokens(weights):
    B, P, n = 8, 19, 12
    one = D.DecodeProgram(SMALL, weights, device=0, maxlen=256, steps=64)
    prog = batch(weights, B, pages=40)
    prompt = np.random.default_rng(3).integers(0, SMALL.V, P)
    s = Sampling(temperature=0.9, top_k=200, top_p=0.95, seed=11)
    got = prog.answers(one, prompt, n, s)
    lp = prog.logprobs.cpu().numpy()
    assert got.shape == (B, n) and len({tuple(r) for r in got.tolist()}) > 1 and lp.shape == (n, B) and (lp <= 0).all()
    # the first tokens come from the prompt's logits, the last ones from the logits the last step left
    u = s.numbers(n, B, DEV).cpu().numpy()
    for logits, i in ((one.read("logits").reshape(1, -1).repeat(B, 0), 0), (prog.read("logits"), n - 1)):
        for b in range(B):
            tok, logp, _, margin = oracle(logits[b], float(u[i, b]), 0.9, 200, 0.95, 0.0)
            assert margin > 1e-11 and got[b, i] == tok and abs(lp[i, b] - logp) <= 2 ** -18 + 1e-8
    again = prog.answers(one, prompt, n, s)
    assert np.array_equal(again, got) and np.array_equal(prog.logprobs.cpu().numpy(), lp)
    assert not np.array_equal(prog.answers(one, prompt, n, Sampling(temperature=0.9, top_k=200, top_p=0.95, seed=12)), got)
    assert prog.answers(one, prompt, 1, s).shape == (B, 1)
    greedy = prog.answers(one, prompt, n, Sampling(temperature=0.0))
    assert all(np.array_equal(greedy[b], greedy[0]) for b in range(B)) and greedy[0, 0] == one.generate(prompt, 1)[0]
    one.close(); prog.close()


def test_temperature_0_is_greedy(weights):
    prompt = np.random.default_rng(5).integers(0, SMALL.V, 9)
    one = D.DecodeProgram(SMALL, weights, device=0, maxlen=256, steps=64)
    assert np.array_equal(one.generate(prompt, 20, sampling=Sampling(temperature=0.0)), one.generate(prompt, 20))
    drawn = one.generate(prompt, 20, sampling=Sampling(temperature=1.5, seed=3), sync_every=3)
    assert np.array_equal(drawn, one.generate(prompt, 20, sampling=Sampling(temperature=1.5, seed=3))) and one.logprobs.shape == (20, 1)
    assert not np.array_equal(drawn, one.generate(prompt, 20))
    one.close()
    prog = batch(weights, 4)
    prompts = np.random.default_rng(6).integers(0, SMALL.V, (4, 9))
    assert np.array_equal(prog.generate(prompts, 11, sampling=Sampling(temperature=0.0)), prog.generate(prompts, 11))
    mixed = Sampling(temperature=torch.tensor([0.0, 1.0, 0.0, 2.0], device=DEV), top_k=torch.tensor([0, 1, 9, 0], dtype=torch.int32, device=DEV), seed=1)
    got, greedy = prog.generate(prompts, 11, sampling=mixed), prog.generate(prompts, 11)
    assert np.array_equal(got[:3], greedy[:3]) and not np.array_equal(got[3], greedy[3])
    prog.close()
    d = M.MlaDims(name="t", H=512, NH=4, C=512, DN=128, DR=64, DV=128, MI=128, E=8, TOPK=2, NS=1, DENSE_LAYERS=1, DENSE_INTER=512, L=2, V=512)
    mla = M.MlaProgram(d, M.random_weights(d, 64, torch.device(DEV), seed=2), device=0, maxlen=64)
    prompt = np.random.default_rng(9).integers(0, d.V, 7)
    assert np.array_equal(mla.generate(prompt, 9, sampling=Sampling(temperature=0.0)), mla.generate(prompt, 9))
    assert np.array_equal(mla.generate(prompt, 9, sampling=Sampling(seed=1)), mla.generate(prompt, 9, sampling=Sampling(seed=1)))
    mla.close()


def test_refusals(weights):
    one = D.DecodeProgram(SMALL, weights, device=0, maxlen=256, steps=64)
    plain, prog = batch(weights, 2), batch(weights, 2, pages=5)
    one.generate([1, 2, 3], 1)
    with pytest.raises(ValueError, match="without pages"):
        plain.adopt(one, 3)
    with pytest.raises(ValueError, match="over pages"):
        prog.load_kv(0, 0, np.zeros((1, 2, 128), np.float32), np.zeros((1, 2, 128), np.float32))
    with pytest.raises(EtxbError, match="free pages"):
        prog.adopt(one, 81)
    prog.adopt(one, 3)
    with pytest.raises(ValueError, match="positions at position 4"):
        prog.decode([1, 2], 4, 3)
    with pytest.raises(EtxbError, match="free pages"):
        prog.cache.extend([0], 90)
    with pytest.raises(ValueError, match="one GPU"):
        one.generate([1], 2, unfused=True, sampling=Sampling())
    with pytest.raises(ValueError, match="outside the vocabulary"):
        prog.decode([1, SMALL.V], 3, 3)
    with pytest.raises(ValueError, match="temperature"):
        prog.decode([1, 2], 3, 3, sampling=Sampling(temperature=torch.ones(3, device=DEV)))
    with pytest.raises(ValueError, match="random numbers"):
        prog.decode([1, 2], 3, 3, sampling=Sampling(given=torch.zeros((2, 2), device=DEV)))
    with pytest.raises(ValueError, match="in 5 pages"):
        prog.generate([[1, 2], [3, 4]], 60)
    with pytest.raises(ValueError, match="temperature"):
        plain.generate([[1, 2], [3, 4]], 5, sampling=Sampling(temperature=torch.ones(3, device=DEV)))
    assert plain.generate([[1, 2], [3, 4]], 5).shape == (2, 5)           # and goes on
    assert prog.cache.rows() == [0] and prog.cache.length_of(0) == 3     # nothing that was refused grew or ended a sequence
    assert prog.decode([5, 6], 3, 4).shape == (2, 4)                     # a column without a sequence runs along
    with pytest.raises(ValueError, match="pages"):
        batch(weights, 2, pages=0)
    one.close(); plain.close(); prog.close()


def test_prologue_blocks_that_are_refused():
    """Refused on the host, by the checks in front of a launch."""
    lib = L.load()

    def status(nb, span, tables):
        blk = struct.pack("<2iQ3I", nb, span, tables, nb & 255, 1, 1) + bytes(4)
        return lib.etxb_op_launch(0, L.BODY["prologue_nb"], blk, len(blk), 1, None, None), lib.etxb_last_error().decode()
    t = op_batch.COLS_TABLES
    for nb, span, tables in ((4 | t, 64, 0), (4 | t, 0, 4096), (4 | t, 40, 4096), (t, 64, 4096), (65 | t, 64, 4096), (4 | 2 * t, 64, 4096)):
        code, text = status(nb, span, tables)
        assert L.STATUS[code] == "E_UNSUPPORTED" and "per-column prologue" in text, (nb, span, tables, code, text)
