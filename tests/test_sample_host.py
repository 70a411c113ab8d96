"""What drawing tokens refuses, checked where there is no device: the library's own checks come before its first CUDA call."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import etx_megakernel_b200  # noqa: E402,F401
from etx_megakernel_b200.runtime import lib, sample  # noqa: E402


def call(device=0, nbytes=None, **f):
    import __graft_entry__ as ge
    ge.build()
    a = lib.SampleArgs(logits=4096, u=4096, tokens=4096, row_stride=100, rows=2, V=100, temperature_all=1.0, top_p_all=1.0)
    for k, v in f.items():
        setattr(a, k, v)
    lib.check(lib.load().etxb_sample(device, C.byref(a), C.sizeof(a) if nbytes is None else nbytes, None))


@pytest.mark.parametrize("bad,status", [(dict(nbytes=8), "E_ARG"), (dict(device=-1), "E_ARG"), (dict(device=64), "E_ARG"), (dict(rows=-1), "E_UNSUPPORTED"),
                                        (dict(V=0), "E_UNSUPPORTED"), (dict(V=524289), "E_UNSUPPORTED"), (dict(dtype=3), "E_UNSUPPORTED"), (dict(dtype=-1), "E_UNSUPPORTED"),
                                        (dict(row_stride=99), "E_ARG"), (dict(logits=None), "E_ARG"), (dict(u=None), "E_ARG"), (dict(tokens=None), "E_ARG"),
                                        (dict(logits=4097), "E_ARG"), (dict(dtype=2, logits=4098), "E_ARG"), (dict(kept=4098), "E_ARG"), (dict(top_p=4097), "E_ARG"),
                                        (dict(reserved=1), "E_ARG")])
def test_library_refuses(bad, status):
    with pytest.raises(lib.EtxbError) as e:
        call(**bad)
    assert e.value.status == status


def test_no_rows_is_no_work():
    call(rows=0, logits=None, u=None, tokens=None)


def test_host_tensors_are_refused():
    l, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA tensor"):
        sample(l, u)
    with pytest.raises(ValueError, match="CUDA tensor"):
        sample([1.0], u)


def test_packed_arguments_are_the_structure():
    import importlib
    mod = importlib.import_module("etx_megakernel_b200.runtime.sampling")
    values = list(range(1, 16)) + [0.5, 0.25, 0.125, 19]
    packed = lib.SampleArgs.from_buffer_copy(mod._pack(*values))
    assert C.sizeof(packed) == len(mod._pack(*values)) and [getattr(packed, n) for n, _ in packed._fields_] == values
