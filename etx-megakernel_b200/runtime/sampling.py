"""Drawing tokens from logits on the device (etxb_sample): temperature, top-k, top-p and min-p, with given random numbers.

No counterpart in the reference, whose host loop is greedy (examples/vllm_llm/vl_tiles.hip:47-89)."""
from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import lib as L
from ._call import cuda_tensor, lend, other_stream, raw_stream, vector

_DT = {torch.bfloat16: L.DTYPES["bf16"], torch.float16: L.DTYPES["f16"], torch.float32: L.DTYPES["f32"]}
MAX_V = 524288
_T, _BYTES = torch.Tensor, C.sizeof(L.SampleArgs)
_pack = struct.Struct("10Pq4i3fi").pack                            # (the structure's fields in order, quicker than through ctypes)


def _count(name, v) -> int:
    """A whole number, as far as a row has tokens (below 1: 0)."""
    try:
        n = int(v)
        if n == v:
            return max(min(n, MAX_V), 0)
    except (TypeError, ValueError, OverflowError):
        pass
    raise ValueError(f"{name}: a whole number or a tensor, got {v!r}")


class Sampled(NamedTuple):
    tokens: torch.Tensor       # int32 [rows]; -1 where no token of a row is allowed
    logprobs: torch.Tensor     # float32 [rows]: of the token among the kept ones
    kept: torch.Tensor         # int32 [rows]: how many tokens the cuts left


@dataclass(frozen=True)
class Sampling:
    """How a program draws its tokens: the settings of `sample` (numbers, or tensors of one value per sequence) and the seed of the random numbers."""
    temperature: object = 1.0
    top_k: object = 0
    top_p: object = 1.0
    min_p: object = 0.0
    seed: int = 0
    given: torch.Tensor | None = None      # the random numbers themselves, float32 [steps][rows], in place of the seed's

    def numbers(self, steps: int, rows: int, device) -> torch.Tensor:
        """The random numbers of a run: [steps][rows] in [0, 1)."""
        g, device = self.given, torch.device(device)
        if g is not None:
            if not isinstance(g, _T) or tuple(g.shape) != (steps, rows):
                raise ValueError(f"given random numbers {tuple(g.shape) if isinstance(g, _T) else type(g).__name__}, the run takes {(steps, rows)}")
            if g.dtype is not torch.float32 or g.device.type != device.type or device.index not in (None, g.device.index) or (rows > 1 and g.stride(1) != 1):
                raise ValueError(f"given random numbers: {g.dtype} on {g.device} with strides {g.stride()}, the run takes adjoining float32 ones on {device}")
            return g
        return torch.rand((steps, rows), device=device, generator=torch.Generator(device=device).manual_seed(self.seed))


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, tokens=None, next_tokens=None, stream=None) -> Sampled:
    """One token per row of `logits` [rows][V] (bf16, fp16 or fp32; rows may lie further apart), drawn with u [rows] in [0, 1).

    A row's allowed tokens (neither -inf nor NaN) stand in the order "larger logit first, equal ones by index" with the weights
    exp((logit - largest) / temperature).  top_k keeps the first so many (0: all); top_p of those the ones with less than its share of their sum before
    them (1: all); min_p the ones of at least that share of the largest weight (0: all); one is always kept.  The token is the first whose sum up to and
    with itself exceeds u times the sum of the kept ones.  temperature 0: the largest logit.  Equal inputs give equal tokens, whatever else runs.  Weights of 16-bit logits
    are 64-bit numbers; those of fp32 logits are whole steps of 2^-43 of the largest or finer, so that tokens of about a step and less may be counted, or left out, next to a
    border (a top_p within 2^-24 of 1 over a long, even tail).

    temperature, top_k, top_p, min_p: numbers, or tensors [rows] (float32; top_k int32).  tokens / next_tokens: int32 tensors [rows] that take the tokens
    (the second one them once more, 0 where there is none: the next step's input).  stream: a raw handle or torch stream; None is the current one.  What
    the call reads and is given to write has to be ready there; what it returns is memory of that stream, also kept for what the current one still does with it
    when it is released."""
    if not (isinstance(logits, _T) and logits.is_cuda and logits.dtype in _DT and len(logits.shape) == 2 and (logits.shape[1] == 1 or logits.stride(1) == 1)):
        cuda_tensor("logits", logits, _DT, (None, None))          # (says what is wrong)
    rows, V = logits.shape
    if not 1 <= V <= MAX_V:
        raise ValueError(f"logits: {V} tokens outside 1..{MAX_V}")
    stride = logits.stride(0) if rows > 1 else V
    if stride < V:
        raise ValueError(f"logits: rows overlap (stride {stride} below {V})")
    index = logits.get_device()
    vector("u", u, torch.float32, rows, index)
    keep = [logits, u]

    def setting(name, v, dtype):
        """The setting as (address of one value per row, value for all)."""
        if not isinstance(v, _T):
            return 0, _count(name, v) if dtype is torch.int32 else C.c_float(v).value
        keep.append(vector(name, v, dtype, rows, index))
        return v.data_ptr(), 0
    temperatures, temperature = setting("temperature", temperature, torch.float32)
    ks, k = setting("top_k", top_k, torch.int32)
    ps, p = setting("top_p", top_p, torch.float32)
    mins, least = setting("min_p", min_p, torch.float32)
    if next_tokens is not None:
        keep.append(vector("next_tokens", next_tokens, torch.int32, rows, index))
    if tokens is not None:
        keep.append(vector("tokens", tokens, torch.int32, rows, index))
    other = None if stream is None else other_stream(index, stream)
    if other is None:
        logprobs = torch.empty_like(u)
        kept = torch.empty_like(u, dtype=torch.int32)
        if tokens is None:
            tokens = torch.empty_like(kept)
        handle = raw_stream(index)
    else:
        with torch.cuda.stream(other):                            # (the results are of the call's stream: memory of the current one's may still be written there)
            logprobs = torch.empty_like(u)
            kept = torch.empty_like(u, dtype=torch.int32)
            made = torch.empty_like(kept) if tokens is None else None
        lend(other, keep)
        lend(torch.cuda.current_stream(index), (logprobs, kept, made))
        tokens, handle = made if tokens is None else tokens, other.cuda_stream
    a = _pack(logits.data_ptr(), u.data_ptr(), temperatures, ks, ps, mins, tokens.data_ptr(), 0 if next_tokens is None else next_tokens.data_ptr(), logprobs.data_ptr(),
              kept.data_ptr(), stride, rows, V, _DT[logits.dtype], k, temperature, p, least, 0)
    rc = L.load().etxb_sample(index, a, _BYTES, handle)
    if rc:
        L.check(rc)
    return Sampled(tokens, logprobs, kept)
