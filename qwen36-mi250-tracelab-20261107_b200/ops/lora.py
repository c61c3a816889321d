"""Low-rank adapters of one projection: what a request's own fine-tuning adds to the weights that all requests share.

Adapter ``i`` of a projection ``W [N, K]`` is ``a[i] [R, K]``, ``b[i] [N, R]`` and a number ``scale[i]``; a row ``x`` of a request that uses it gives
``x W^T + scale[i] (x a[i]^T) b[i]^T``. All adapters of a projection are held together with one rank ``R``, smaller ones filled up with zeros,
which add nothing. The numbers are finite (``models/lora.py`` refuses files with others): rows of different adapters share the tiles of a matrix
product, where another request's row meets an adapter's numbers with a factor of 0.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

RANK_STEP = 8  # ranks are multiples of it: rows of b are then whole 16-byte pieces
MAX_RANK = 256
MAX_ADAPTERS = 1024


class LoraWeights(NamedTuple):
    """``a [L, R, K]`` and ``b [L, N, R]`` bf16, ``scale [L]`` fp32."""

    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor


def check_weights(w: LoraWeights, N: int, K: int, what: str) -> tuple[int, int]:
    """Refuse adapters that are not ``w [N, K]``'s, or not as ``LoraWeights`` says; ``(L, R)``."""
    a, b, scale = w
    L, R = a.shape[:2] if a.dim() == 3 else (-1, -1)
    if a.shape != (L, R, K) or b.shape != (L, N, R) or scale.shape != (L,):
        raise ValueError(f"{what}: adapters {tuple(a.shape)}, {tuple(b.shape)} and {tuple(scale.shape)} are not [L, R, {K}], [L, {N}, R] and [L]")
    if not 1 <= L <= MAX_ADAPTERS or not RANK_STEP <= R <= MAX_RANK or R % RANK_STEP:
        raise ValueError(f"{what}: {L} adapters of rank {R}, not 1 to {MAX_ADAPTERS} of a multiple of {RANK_STEP} up to {MAX_RANK}")
    if scale.dtype != torch.float32 or a.dtype != b.dtype:
        raise ValueError(f"{what}: adapters of {a.dtype} and {b.dtype} with {scale.dtype} factors")
    if not (a.is_contiguous() and b.is_contiguous() and scale.is_contiguous()):
        raise ValueError(f"{what}: adapters with strides {a.stride()}, {b.stride()}, {scale.stride()} are not contiguous")
    if a.device != b.device or a.device != scale.device:
        raise ValueError(f"{what}: adapters on {a.device}, {b.device} and {scale.device}")
    return L, R
