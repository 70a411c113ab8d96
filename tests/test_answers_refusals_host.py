"""What a batch over pages refuses, on the host: the program's device part is left out (steps are recorded), its pool keeps its books in the library over CPU
tensors.  A call that is refused runs no step and leaves rows, lengths and tables as they were."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.models import batched as BT  # noqa: E402
from etx_megakernel_b200.models import drawing  # noqa: E402
from etx_megakernel_b200.models import qwen as Q  # noqa: E402
from etx_megakernel_b200.runtime import Sampling, copy_pages  # noqa: E402
from tests.test_pages_host import HostPool, on_host  # noqa: E402,F401

DIMS = Q.Dims(name="small", H=512, NH=8, NKV=2, HD=128, INTER=0, L=3, V=1504, qk_norm=True, moe=True, E=16, TOPK=4, MI=128, norm_topk=True)


class Program(BT.BatchProgram):
    def __init__(self, B=3, pages=20, maxlen=128, steps=64):
        nblk = -(-maxlen // BT.BS)
        self.d, self.B, self.pages, self.maxlen, self.steps, self.dev = DIMS, B, pages, maxlen, steps, torch.device("cpu")
        self.buf = {"token_in": torch.zeros((steps, B), dtype=torch.int32), "block_tables": torch.full((B, nblk), pages, dtype=torch.int32),
                    "logits": torch.zeros((B, DIMS.V)), "kc": torch.zeros((2, pages + 1, 8)), "vc": torch.zeros((2, pages + 1, 8))}
        self.cache = HostPool([self.buf["kc"][:, :pages], self.buf["vc"][:, :pages]], B, nblk, tables=self.buf["block_tables"], page_len=BT.BS)
        self.runs = []

    def _run(self, fed, pos, n_gen, sync_every, sampling):
        self.runs.append((fed.tolist(), pos, n_gen))
        return np.zeros((self.B, n_gen), np.int32)

    def state(self):
        return [(r, self.cache.length_of(r), self.cache.pages_of(r)) for r in self.cache.rows()], self.buf["block_tables"].tolist(), self.runs


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("pos", [-1, -16, -(2 ** 31)])
def test_decode_refuses_positions_below_0(on_host, rows, pos):  # noqa: F811
    """Without a sequence nothing else names the position: tables would be read before their beginning, and the slot found there written."""
    prog = Program()
    for _ in range(rows):
        prog.cache.open(5)
    before = prog.state()
    with pytest.raises(ValueError, match="position"):
        prog.decode([1, 2, 3], pos, 4)
    assert prog.state() == before
    assert prog.decode([1, 2, 3], 5, 4).shape == (3, 4) and prog.runs == [([[1, 2, 3]], 5, 4)]


BAD_NUMBERS = [torch.zeros((4, 3), dtype=torch.float64), torch.zeros((4, 3), device="meta"), torch.zeros((4, 6))[:, ::2], torch.zeros((3, 4)), [[0.5] * 3] * 4]


@pytest.mark.parametrize("given", BAD_NUMBERS)
def test_decode_refuses_random_numbers_before_sequences_grow(on_host, monkeypatch, given):  # noqa: F811
    monkeypatch.setattr(drawing, "sample", lambda *a, **k: None)        # (settings are looked at on the device)
    prog = Program()
    prog.cache.open(5)
    before = prog.state()
    with pytest.raises(ValueError, match="random numbers"):
        prog.decode([1, 2, 3], 5, 4, sampling=Sampling(given=given))
    assert prog.state() == before
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        prog.decode([1, 2, 3], 5, 4, sampling=Sampling(seed="seven"))
    assert prog.state() == before
    prog.decode([1, 2, 3], 5, 4, sampling=Sampling(given=torch.zeros((4, 3))))
    assert prog.cache.length_of(0) == 9


def no_such_setting(*a, **k):
    raise ValueError("temperature: shape (4,), expected (3,)")


@pytest.mark.parametrize("what", ["setting", "numbers", "pages", "long", "no prompt", "less than none", "fails"])
def test_generate_over_pages_ends_no_sequence_for_nothing(on_host, monkeypatch, what):  # noqa: F811
    """Refused calls leave the sequences; a run that fails ends the ones it opened, whose positions nobody has written."""
    prog = Program()
    monkeypatch.setattr(drawing, "sample", no_such_setting if what == "setting" else lambda *a, **k: None)
    prog.cache.open(21)
    prog.cache.open(40)
    before = prog.state()
    prompts, n, s = np.ones((3, 7), int), 5, Sampling()
    if what == "numbers":
        s = Sampling(given=torch.zeros((4, 3)))
    elif what == "pages":
        prompts = np.ones((3, 100), int)
        prog.buf["token_in"] = torch.zeros((200, 3), dtype=torch.int32)
        n = 29                                                          # 8 pages a sequence of 20
    elif what == "long":
        n = 70
    elif what == "no prompt":
        prompts = np.ones((3, 0), int)
    elif what == "less than none":
        prompts, n = np.ones((3, 1), int), -1
    elif what == "fails":
        def failing(*a):
            raise RuntimeError("E_TIMEOUT")
        prog._run = failing
    with pytest.raises((ValueError, RuntimeError)) as e:
        prog.generate(prompts, n, sampling=s)
    if what == "fails":
        assert "E_TIMEOUT" in str(e.value) and prog.cache.rows() == [] and prog.cache.free_pages == 20 and bool((prog.buf["block_tables"] == 20).all())
    else:
        assert isinstance(e.value, ValueError) and prog.state() == before
    prog.__dict__.pop("_run", None)
    assert prog.generate(np.ones((3, 7), int), 0).shape == (3, 0) and prog.cache.rows() == [0, 1, 2] and prog.cache.length_of(2) == 6


class One:
    """What adopt and answers take of a one-sequence program."""

    def __init__(self, kc=(2, 9, 8), dims=DIMS, maxlen=128):
        self.d, self.maxlen, self.dev = dims, maxlen, torch.device("cpu")
        self.buf = {"kc": torch.zeros(kc), "vc": torch.zeros(kc), "logits": torch.zeros(dims.V)}
        self.fed = []

    def generate(self, prompt, n_gen):
        self.fed.append(list(prompt))


@pytest.mark.parametrize("what", ["shape", "copy", "negative", "long", "pages"])
def test_adopt_that_fails_opens_no_sequence(on_host, monkeypatch, what):  # noqa: F811
    """A cache of another layout (a shard's, say) is refused by the copy, behind the opening of a column."""
    def failing(*a, **k):
        raise RuntimeError("E_CUDA")
    monkeypatch.setattr(BT, "copy_pages", failing if what == "copy" else copy_pages)
    prog = Program(pages=8)
    prog.cache.open(21)
    before = prog.state()[0]
    with pytest.raises((ValueError, RuntimeError)):
        prog.adopt(One((2, 9, 4) if what == "shape" else (2, 9, 8)), {"negative": -1, "long": 129, "pages": 100}.get(what, 20))
    assert prog.state()[0] == before and prog.cache.free_pages == 6 and bool((prog.buf["block_tables"][1:] == 8).all())


@pytest.mark.parametrize("what", ["setting", "numbers", "no setting", "none asked", "no prompt", "long", "steps", "pages", "other model", "other layers", "other layout", "fails"])
def test_answers_end_no_sequence_for_nothing(on_host, monkeypatch, what):  # noqa: F811
    """Sizes, pages, settings and the other program are looked at before anything ends or runs; what fails behind that ends the sequences it opened."""
    class First:
        tokens, logprobs = torch.tensor([3, 4, 5], dtype=torch.int32), torch.zeros(3)
    monkeypatch.setattr(drawing, "sample", no_such_setting if what == "setting" else lambda *a, **k: First)
    monkeypatch.setattr(BT, "sample", no_such_setting if what == "setting" else lambda *a, **k: First)
    monkeypatch.setattr(BT, "copy_pages", lambda *a, **k: None)
    prog = Program(pages=11)
    prog.logprobs = torch.zeros((0, 3))
    prog.cache.open(21)
    prog.cache.open(40)
    before = prog.state()
    one, prompt, n, s = One(), list(range(33)), 31, Sampling()          # 2 pages shared, 2 for each answer's own: 8
    if what == "numbers":
        s = Sampling(given=torch.zeros((30, 3)))
    elif what == "no setting":
        s = None
    elif what == "none asked":
        n = 0
    elif what == "no prompt":
        prompt = []
    elif what == "long":
        n = 97
    elif what == "steps":
        n = 64
    elif what == "pages":
        n = 49                                                          # 81 positions: 2 + 3 * 4 pages
    elif what == "other model":
        one = One(dims=Q.Dims(**{**DIMS.__dict__, "V": 1600}))
    elif what == "other layers":
        one = One(dims=Q.Dims(**{**DIMS.__dict__, "L": 2}))
    elif what == "other layout":
        one = One((2, 9, 4))
    elif what == "fails":
        def failing(*a):
            raise RuntimeError("E_TIMEOUT")
        prog._run = failing
    with pytest.raises((ValueError, RuntimeError)) as e:
        prog.answers(one, prompt, n, s)
    if what == "fails":
        assert "E_TIMEOUT" in str(e.value) and prog.cache.rows() == [] and prog.cache.free_pages == 11 and bool((prog.buf["block_tables"] == 11).all())
        return
    assert isinstance(e.value, ValueError) and prog.state() == before and one.fed == []
    monkeypatch.setattr(drawing, "sample", lambda *a, **k: First)
    monkeypatch.setattr(BT, "sample", lambda *a, **k: First)
    assert prog.answers(One(), list(range(33)), 31, Sampling())[:, 0].tolist() == [3, 4, 5]
    assert [prog.cache.length_of(r) for r in prog.cache.rows()] == [63, 63, 63] and prog.cache.free_pages == 3 and prog.runs == [([[3, 4, 5]], 33, 30)]


def test_answers_go_on_behind_a_first_token_that_there_is_none(on_host, monkeypatch):  # noqa: F811
    """A prompt whose logits allow no token: -1, and the step takes 0 for it, as behind every other token."""
    class First:
        tokens, logprobs = torch.tensor([-1, 7, -1], dtype=torch.int32), torch.zeros(3)
    for mod in (drawing, BT):
        monkeypatch.setattr(mod, "sample", lambda *a, **k: First)
    monkeypatch.setattr(BT, "copy_pages", lambda *a, **k: None)
    prog = Program()
    prog.logprobs = torch.zeros((3, 3))
    got = prog.answers(One(), [5, 6], 4, Sampling())
    assert got[:, 0].tolist() == [-1, 7, -1] and prog.runs == [([[0, 7, 0]], 2, 3)]


@pytest.mark.parametrize("t,pos", [(0, -1), (0, 128), (3, 10 ** 6), (-1, 5), (64, 5), (63, 5)])
def test_steps_over_pages_stay_inside_the_tables(on_host, t, pos):  # noqa: F811
    """A step's position names an entry of each column's table, and the page in it the memory that is written."""
    class Recorded:
        steps = []

        def set_step(self, **kw):
            self.steps.append((kw["tok"], kw["pos"]))

        def run(self, timeout):
            pass
    prog = Program()
    prog.session = Recorded()
    with pytest.raises(ValueError, match="step"):
        prog.step(t, pos, True)
    prog.step(63, 127, False)
    assert Recorded.steps == [(63, 127)]
    Recorded.steps.clear()
