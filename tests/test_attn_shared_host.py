"""What attention over shared prefixes refuses, without a device: the library's checks come before its first CUDA call."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import attn_shared, lib  # noqa: E402


def call(nbytes=None, device=0, first=(0, 2, 3), **f):
    import __graft_entry__ as ge
    ge.build()
    first = np.array(first, np.int32)
    p = 1 << 20
    a = lib.AttnSharedArgs(q=p, out=p, kc=p, vc=p, tables=p, lens=p, prefix_tables=p, prefix_lens=p, group_first=first.ctypes.data, q_stride=1024, out_stride=1024,
                           k_stride=4096, v_stride=4096, table_stride=5, prefix_stride=9, seqs=3, groups=2, NH=8, NKV=2, HD=128, pages=10, table_width=5, prefix_width=9, scale=0.1)
    for k, v in f.items():
        setattr(a, k, v)
    lib.check(lib.load().etxb_attn_shared(device, C.byref(a), C.sizeof(a) if nbytes is None else nbytes, None))


@pytest.mark.parametrize("bad,status", [
    (dict(nbytes=8), "E_ARG"), (dict(device=-1), "E_ARG"), (dict(NH=7), "E_UNSUPPORTED"), (dict(NH=0), "E_UNSUPPORTED"), (dict(NKV=0), "E_UNSUPPORTED"), (dict(NH=34), "E_UNSUPPORTED"),
    (dict(HD=8), "E_UNSUPPORTED"), (dict(HD=120), "E_UNSUPPORTED"), (dict(HD=272), "E_UNSUPPORTED"), (dict(seqs=1025), "E_UNSUPPORTED"), (dict(seqs=-1), "E_UNSUPPORTED"),
    (dict(groups=1025), "E_UNSUPPORTED"), (dict(pages=0), "E_UNSUPPORTED"), (dict(table_width=-1), "E_UNSUPPORTED"), (dict(q=None), "E_ARG"), (dict(lens=None), "E_ARG"), (dict(tables=None), "E_ARG"),
    (dict(group_first=None), "E_ARG"), (dict(q=(1 << 20) + 8), "E_ARG"), (dict(vc=(1 << 20) + 2), "E_ARG"), (dict(lens=(1 << 20) + 2), "E_ARG"), (dict(q_stride=1016), "E_ARG"),
    (dict(q_stride=1028), "E_ARG"), (dict(out_stride=0), "E_ARG"), (dict(k_stride=4088), "E_ARG"), (dict(v_stride=4100), "E_ARG"), (dict(table_stride=4), "E_ARG"), (dict(prefix_stride=8), "E_ARG"),
    (dict(first=(1, 2, 3)), "E_ARG"), (dict(first=(0, 2, 2)), "E_ARG"), (dict(first=(0, 4, 3)), "E_ARG"), (dict(reserved=1), "E_ARG")])
def test_library_refuses(bad, status):
    with pytest.raises(lib.EtxbError) as e:
        call(**bad)
    assert e.value.status == status


def test_no_sequences_is_no_work():
    call(seqs=0, q=None, out=None)


def test_host_tensors_are_refused():
    z = torch.zeros(2, 2, 16, 16, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        attn_shared(z, z, z, z, z, z, z)


def test_packed_arguments_are_the_structure():
    import importlib
    mod = importlib.import_module("etx_megakernel_b200.runtime.attn_shared")
    values = list(range(1, 27)) + [0.5, 28]
    packed = lib.AttnSharedArgs.from_buffer_copy(mod._pack(*values))
    assert C.sizeof(packed) == len(mod._pack(*values)) and [getattr(packed, n) for n, _ in packed._fields_] == values
