"""Groups of very different sizes: the workspace follows the rows that there are, and the parts of uneven units do not meet."""
import importlib
from array import array
from itertools import accumulate

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from tests.test_gpu_attn_shared import Case  # noqa: E402


@pytest.mark.parametrize("sizes,NH,NKV,HD", [([25] + [1] * 999, 64, 8, 128), ([1] * 500 + [25] + [1] * 499, 64, 8, 256), ([64], 32, 8, 128), ([1] * 1024, 16, 1, 64)])
def test_the_workspace_follows_the_rows(sizes, NH, NKV, HD):
    """Partial results: every row once, and a largest unit (up to 128 rows) more for each worker; as much at most for own positions; numbers beside them."""
    mod = importlib.import_module("etx_megakernel_b200.runtime.attn_shared")
    n = mod._work_bytes(0, array("i", (0, *accumulate(sizes))).tobytes(), sum(sizes), len(sizes), NH, NKV, HD, 100, 10, 10)
    workers = torch.cuda.get_device_properties(0).multi_processor_count
    assert n <= 2 * (sum(sizes) * NH + 128 * workers) * (HD + 2) * 4 + (1 << 20)


@pytest.mark.parametrize("sizes,NH,NKV,HD,plen", [([25] + [1] * 299, 16, 2, 64, 40), ([1] * 100 + [70, 0, 2] + [1] * 50, 12, 2, 128, 300), ([3, 140, 1, 33, 0, 17], 8, 1, 256, 900),
                                                  ([1, 40, 1, 40, 1], 32, 4, 128, 5000)])
def test_uneven_groups(sizes, NH, NKV, HD, plen):
    rng = np.random.default_rng(len(sizes))
    c = Case(NH, NKV, HD, sizes, [int(x) for x in rng.integers(0, plen + 1, len(sizes))], [int(x) for x in rng.integers(0, 60, sum(sizes))], seed=len(sizes))
    out = c.check()
    assert torch.equal(c.run(), out)
