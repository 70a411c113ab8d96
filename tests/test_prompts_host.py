"""Prompts and positions that a program cannot hold, on the host: tokens are looked up in the embedding and positions in caches and tables by kernels that trust
them, so they are refused before anything is queued."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.models import batched as BT  # noqa: E402
from etx_megakernel_b200.models import decode as D  # noqa: E402
from etx_megakernel_b200.models import dsv2 as M  # noqa: E402
from etx_megakernel_b200.models import qwen as Q  # noqa: E402
from etx_megakernel_b200.runtime import Sampling  # noqa: E402

DIMS = Q.Dims(name="small", H=512, NH=8, NKV=2, HD=128, INTER=0, L=3, V=1504, qk_norm=True, moe=True, E=16, TOPK=4, MI=128, norm_topk=True)


class NoSession:
    def __getattr__(self, name):
        raise AssertionError("nothing is queued")


def program(kind):
    p = object.__new__(kind)
    p.d, p.maxlen, p.ranks, p.B, p.cache, p.pages, p.dev, p.session = DIMS, 64, 1, 1, None, None, torch.device("cuda:0"), NoSession()
    p.buf = {"token_in": torch.zeros((80, 1) if kind is BT.BatchProgram else 80, dtype=torch.int32)}
    return p


@pytest.mark.parametrize("kind", [D.DecodeProgram, M.MlaProgram, BT.BatchProgram])
@pytest.mark.parametrize("bad", [[-1], [DIMS.V], [3, 5, 2 ** 31 - 1, 4], [3, -(2 ** 31)]])
def test_tokens_outside_the_vocabulary(kind, bad):
    p = program(kind)
    with pytest.raises(ValueError, match="vocabulary of 1504"):
        p.generate([bad] if kind is BT.BatchProgram else bad, 4)
    if kind is not BT.BatchProgram:
        with pytest.raises(ValueError, match="vocabulary of 1504"):
            p.generate_host(np.array(bad), 4)


@pytest.mark.parametrize("kind", [D.DecodeProgram, M.MlaProgram])
@pytest.mark.parametrize("prompt,n,start", [([1, 2], 3, -1), ([1], 5, -16), ([1] * 60, 6, 0), ([1], 4, 61), ([1], 70, 0)])
def test_positions_outside_the_cache(kind, prompt, n, start):
    p = program(kind)
    for f in (p.generate, p.generate_host):
        with pytest.raises(ValueError, match="session was sized for|position"):
            f(prompt, n, start_pos=start)


@pytest.mark.parametrize("kind", [D.DecodeProgram, M.MlaProgram, BT.BatchProgram])
def test_tokens_are_drawn_behind_a_prompt(kind):
    """Without a token of a prompt there are no logits to draw from."""
    p = program(kind)
    for prompt, n in (([], 4), ([3], -1)):
        with pytest.raises(ValueError, match="behind a prompt"):
            p.generate([prompt] if kind is BT.BatchProgram else prompt, n, sampling=Sampling())
