"""The token loop of a program that draws its tokens: a step, then `sample` on its logits, on one stream, step by step."""
from __future__ import annotations

import torch

from ..runtime import Sampling, sample


def check_sizes(prompt: int, n_gen: int):
    if prompt < 1 or n_gen < 0:
        raise ValueError(f"{n_gen} tokens drawn behind a prompt of {prompt}")


def check(prog, n: int, rows: int, sampling: Sampling):
    """Refuses what `run` would refuse at its first draw of n: settings, a seed, random numbers of another shape, type or place."""
    if not isinstance(sampling, Sampling):
        raise ValueError(f"sampling: a runtime.Sampling, got {type(sampling).__name__}")
    if sampling.given is not None:
        sampling.numbers(n, rows, prog.dev)
    else:
        sampling.numbers(0, rows, prog.dev)                             # (the seed)
    sample(prog.buf["logits"].view(rows, -1), torch.zeros(rows, device=prog.dev), sampling.temperature, sampling.top_k, sampling.top_p, sampling.min_p)


def run(prog, n: int, first: int, pos: int, rows: int, sampling: Sampling, sync_every: int):
    """Steps 0 .. n - 1 at positions pos, pos + 1, ..; from step `first` on the tokens are drawn from the step's logits and are the next step's input.
    Token buffers are [steps][rows].  Leaves the log-probabilities of the drawn tokens, [n - first][rows], in prog.logprobs."""
    b, dev = prog.buf, prog.dev
    stream = getattr(prog, "_draw_stream", None)
    if stream is None:
        stream = prog._draw_stream = torch.cuda.Stream(dev)
    logits, tin, tout = b["logits"].view(rows, -1), b["token_in"].view(-1, rows), b["token_out"].view(-1, rows)
    logprobs = torch.empty((n - first, rows), dtype=torch.float32, device=dev)      # (the caller's: of the caller's stream)
    stream.wait_stream(torch.cuda.current_stream(dev))
    try:
        with torch.cuda.stream(stream):
            u = sampling.numbers(n - first, rows, dev)
            for t in range(n):
                prog.session.set_step(tok=t, pos=pos + t, write_next=0)
                prog.session.launch(stream.cuda_stream)
                if t >= first:
                    r = sample(logits, u[t - first], sampling.temperature, sampling.top_k, sampling.top_p, sampling.min_p, tokens=tout[t], next_tokens=tin[t + 1])
                    logprobs[t - first] = r.logprobs
                if t % sync_every == sync_every - 1 or t == n - 1:
                    prog.session.wait(120.0)
    finally:
        stream.synchronize()                                            # (settings that are refused leave a step behind)
    prog.logprobs = logprobs
