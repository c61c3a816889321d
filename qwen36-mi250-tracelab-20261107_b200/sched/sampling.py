"""Token selection from rows of logits, on the device that holds them.

Greedy at temperature 0 (ties to the lower id); otherwise temperature, top-k, top-p, min-p and a seeded draw. ``masks``
remove the end-of-sequence ids while ``min_tokens`` has not been reached (reference: ``Generator.pick``,
``engine/generator.py:1091-1110``).

All rows of a step are one call (``ops.sample``): their settings go to the device in one copy, only the picked ids come back. The draw is
an inverse-CDF lookup over the filtered distribution in descending order of probability, with ONE uniform number per request and step
taken from the request's own seeded generator on the host: the same seed gives the same tokens on any device and in any batch.
"""

from __future__ import annotations

import torch

from ..ops import torch_ops
from .request import Sampling

MAX_EXCLUDED = 64  # ids per row that the operator leaves out by itself


def pick_tokens(logits: torch.Tensor, samplings: list[Sampling], rngs: list, masks: list) -> list[int]:
    """Next token of each row of ``logits [n, V]``. ``rngs[i]``: the request's CPU generator (unused for greedy
    rows); ``masks[i]``: ids to exclude for this row, or None. A row of which nothing is left gives 0."""
    n, V = logits.shape
    dev = logits.device
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        logits = logits.float()
    most = max((len(m) for m in masks if m), default=0)
    if most > MAX_EXCLUDED:
        rows = [i for i, m in enumerate(masks) for _ in m or ()]
        cols = [t for m in masks for t in m or ()]
        logits = logits.clone()
        logits[torch.tensor(rows, device=dev), torch.tensor(cols, device=dev)] = float("-inf")
        most = 0
    # one block of 32-bit words: temperature, top-p, min-p, uniform number, top-k, excluded ids
    host = torch.empty((5 + most) * n, dtype=torch.float32, pin_memory=dev.type == "cuda")
    real, whole = host[: 4 * n].view(4, n), host[4 * n :].view(torch.int32)
    real.copy_(torch.tensor([[0.0 if s.greedy else max(s.temperature, 1e-6) for s in samplings], [s.top_p for s in samplings],
                             [s.min_p for s in samplings],
                             [0.0 if s.greedy else float(torch.rand(1, generator=g)) for s, g in zip(samplings, rngs)]]))
    whole[:n].copy_(torch.tensor([s.top_k if s.top_k and 0 < s.top_k < V else 0 for s in samplings], dtype=torch.int32))
    if most:
        whole[n:].copy_(torch.tensor([[*(m or ()), *[-1] * (most - len(m or ()))] for m in masks], dtype=torch.int32).view(-1))
    block = host.to(dev)
    t, p, m, u = block[: 4 * n].view(4, n)
    ints = block[4 * n :].view(torch.int32)
    args, exclude = (logits, t, ints[:n], p, m, u), ints[n:].view(n, most) if most else None
    if dev.type == "cuda":
        from ..ops import cuda_ops

        if V <= cuda_ops.SAMPLE_VOCAB:  # (a larger vocabulary by the plain form)
            with torch.cuda.device(dev):  # (the kernels run on the current device)
                return [max(0, i) for i in cuda_ops.sample(*args, exclude=exclude).tolist()]
    picks = torch_ops.sample(*args, exclude=exclude)
    return [max(0, i) for i in picks.tolist()]


def pick_token(logits: torch.Tensor, s: Sampling, rng: torch.Generator | None, mask: set[int] | None = None) -> int:
    """One row (``logits [V]``): see ``pick_tokens``."""
    return pick_tokens(logits[None, :], [s], [rng], [mask])[0]
