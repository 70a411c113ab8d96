"""What the operators beside the step share: checks of tensors, and the stream of a call."""
from __future__ import annotations

import torch

_Tensor = torch.Tensor
raw_stream = torch._C._cuda_getCurrentRawStream


def cuda_tensor(name: str, t, dtypes, shape=None, inner: bool = True):
    """`t` as a CUDA tensor of one of `dtypes`; `shape` with None for sizes that are free; inner: the last dimension's elements adjoin."""
    if not isinstance(t, _Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor, got {getattr(t, 'device', type(t).__name__)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} is none of {', '.join(str(d) for d in dtypes)}")
    if shape is not None and (t.dim() != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape))):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple('any' if w is None else w for w in shape)}")
    if inner and t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the elements of the last dimension adjoin (stride {t.stride(-1)})")
    return t


def vector(name: str, t, dtype, n: int, index: int):
    """`t` as `n` adjoining values on device `index` (the checks of cuda_tensor and same_device, quick where they pass)."""
    if isinstance(t, _Tensor) and t.is_cuda and t.dtype is dtype and t.shape == (n,) and (n < 2 or t.stride(0) == 1) and t.get_device() == index:
        return t
    cuda_tensor(name, t, (dtype,), (n,))
    raise ValueError(f"{name} is on {t.device}, the call runs on cuda:{index}")


def same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the call runs on {device}")


def other_stream(index: int, stream):
    """`stream` (a raw handle or a torch stream) as a torch stream of device `index`, or None where it is the current one (or None)."""
    if stream is None:
        return None
    handle = int(getattr(stream, "cuda_stream", stream))
    if handle == raw_stream(index):
        return None
    device = torch.device("cuda", index)
    return torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)


def lend(stream, tensors):
    """The tensors' memory, which belongs to other streams, is kept until `stream` has passed what it was given so far when they are released."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


def stream_handle(index: int, stream, tensors) -> int:
    """The raw handle of the call's stream on device `index`: the current one, or `stream` (a raw handle or a torch stream), which the tensors' memory is
    then kept for until it has passed the call.  (For calls that allocate nothing: memory of the current stream's may still be written there by what was
    queued before it was released.)"""
    other = other_stream(index, stream)
    if other is None:
        return raw_stream(index)
    lend(other, tensors)
    return other.cuda_stream
