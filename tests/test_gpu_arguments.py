"""Arguments that are no sizes or settings, refused in the operators' own manner before anything is launched."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import EtxbError, attn_shared, sample  # noqa: E402

DEV = "cuda:0"


def test_top_k_is_a_whole_number():
    """A half is not 0, which keeps every token."""
    l, u = torch.randn((3, 500), device=DEV).bfloat16(), torch.full((3,), 0.9, device=DEV)
    for bad in (0.5, 1.5, float("inf"), float("nan"), "many", None):
        with pytest.raises(ValueError, match="top_k"):
            sample(l, u, top_k=bad)
    for k in (7, 7.0, True, 10 ** 12, -3):
        r = sample(l, u, top_k=k)
        assert r.kept.tolist() == [7 if k == 7 else 1 if k is True else 500] * 3


def test_caches_without_heads_are_refused():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, device=DEV, dtype=dtype)  # noqa: E731
    n, t = z(2, dtype=torch.int32), z(2, 1, dtype=torch.int32)
    for kc, vc in ((z(4, 2, 0, 16, 8), z(4, 2, 0, 16)), (z(4, 0, 4, 16, 8), z(4, 0, 32, 16))):
        for q in (z(2, 0), z(2, 64), z(2, 2, 32), z(2, 2, 0)):
            with pytest.raises((ValueError, EtxbError), match="kc|attn_shared"):
                attn_shared(q, kc, vc, t, n, t[:1], n[:1])
