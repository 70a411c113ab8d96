"""Calls of a batch over pages that are refused or fail leave it as it was, and it goes on."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.models import decode as D  # noqa: E402
from etx_megakernel_b200.runtime import Sampling  # noqa: E402
from tests.test_gpu_answers import DEV, SMALL, batch, weights  # noqa: E402,F401


def state(prog):
    return [(r, prog.cache.length_of(r), prog.cache.pages_of(r)) for r in prog.cache.rows()], prog.buf["block_tables"].tolist(), prog.buf["kc"].clone()


def test_refused_calls_leave_the_sequences(weights):  # noqa: F811
    one, prog = D.DecodeProgram(SMALL, weights, device=0, maxlen=256, steps=64), batch(weights, 3, pages=12)
    prompt = np.random.default_rng(1).integers(0, SMALL.V, 19)
    one.generate(prompt, 1)
    prog.adopt(one, 19)
    prog.fork(0, 1)
    before = state(prog)
    wrong = Sampling(temperature=torch.ones(4, device=DEV))
    for call in (lambda: prog.answers(one, prompt, 5, wrong), lambda: prog.answers(one, prompt, 0, Sampling()), lambda: prog.answers(one, prompt, 60, Sampling()),
                 lambda: prog.answers(one, prompt, 300, Sampling()), lambda: prog.answers(one, [], 5, Sampling()), lambda: prog.answers(one, [SMALL.V], 5, Sampling()),
                 lambda: prog.answers(one, prompt, 5, Sampling(given=torch.zeros((5, 3), device=DEV, dtype=torch.float64))), lambda: prog.answers(one, prompt, 5, None),
                 lambda: prog.generate([[1, 2]] * 3, 5, sampling=wrong), lambda: prog.generate([[1, 2]] * 3, 5, sampling=Sampling(given=torch.zeros((5, 3)))),
                 lambda: prog.generate([[1, SMALL.V]] * 3, 5), lambda: prog.generate([[]] * 3, 5), lambda: prog.decode([1, 2, 3], -1, 4),
                 lambda: prog.decode([1, 2, 3], 19, 4, sampling=Sampling(given=torch.zeros((4, 3)))), lambda: prog.decode([1, 2, 3], 19, 4, sampling=wrong)):
        with pytest.raises(ValueError):
            call()
        after = state(prog)
        assert after[:2] == before[:2] and torch.equal(after[2], before[2])
    assert prog.decode([5, 6, 7], 19, 4, sampling=Sampling(given=torch.rand((4, 3), device=DEV))).shape == (3, 4) and prog.cache.length_of(0) == 23
    got = prog.answers(one, prompt, 12, Sampling(seed=3, temperature=0.8))
    assert got.shape == (3, 12) and [prog.cache.length_of(r) for r in prog.cache.rows()] == [30, 30, 30]
    one.close(); prog.close()


def test_a_prompt_that_allows_no_token(weights):  # noqa: F811
    """Weights that make every logit NaN: no token at any step, and the answers come to their end."""
    bad = dict(weights, lm_head=torch.full_like(weights["lm_head"], float("nan")))
    one, prog = D.DecodeProgram(SMALL, bad, device=0, maxlen=256, steps=64), batch(bad, 2, pages=12)
    got = prog.answers(one, [3, 4, 5], 6, Sampling(seed=1))
    assert (got == -1).all() and bool((prog.logprobs == -float("inf")).all())
    one.close(); prog.close()
