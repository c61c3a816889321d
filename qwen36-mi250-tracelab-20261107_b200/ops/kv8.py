"""The 8-bit form of the paged KV cache.

A row of ``D`` numbers (one token's key or value of one KV head) is held as ``D`` float8 e4m3 numbers and ONE power of two:
``x = data * 2 ** (exps - 127)``, where the exponent is the smallest that brings the row's largest number to 448 or below, held to
``[-E_MAX, E_MAX]``. A power of two and not a full scale: scaling is then exact on either side, so quantising has one rounding (to the four
significant bits of e4m3), a row comes back as bf16 without any, and kernels may apply it wherever it is cheapest. A finer scale
would gain nothing: e4m3 is a floating-point format, whose relative step does not depend on where the row's largest number lies.

An exponent byte of 255 marks a row that held a NaN: all of it reads as NaN, and its data bytes are 0, so that no NaN ever lies in
the data, where a masked key's value would still meet a probability of 0. Infinities are held as the largest number.

A token takes ``2 * n_kv * (D + 1)`` bytes, against ``2 * n_kv * 2 * D`` as bf16.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..config import PAGE_SIZE

E_MAX = 60  # rows of up to 448 * 2^60 = 5e20, steps down to 2^-69; ratios of two rows' scales stay within fp32
E_BIAS = 127
E_NAN = 255
HEAD_DIMS = (32, 64, 128, 256)


class Kv8Layer(NamedTuple):
    """One layer: ``data [pages, 2, n_kv, PAGE_SIZE, D]`` float8 e4m3, ``exps [pages, 2, n_kv, PAGE_SIZE]`` uint8."""

    data: torch.Tensor
    exps: torch.Tensor


class Kv8Pool:
    """The pages of all layers, in the place of ``Model.kv``: ``pool[layer]`` is a ``Kv8Layer``, the calls that the engine makes of the
    bf16 pool's tensor (page copies, bytes of a page) work on both parts."""

    def __init__(self, layers: int, pages: int, n_kv: int, head_dim: int, device) -> None:
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"8-bit KV cache: head dim {head_dim} is none of {HEAD_DIMS}")
        shape = (layers, pages, 2, n_kv, PAGE_SIZE)
        self.data = torch.zeros(*shape, head_dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        self.exps = torch.full(shape, E_BIAS, dtype=torch.uint8, device=device)

    def __getitem__(self, layer: int) -> Kv8Layer:
        return Kv8Layer(self.data[layer], self.exps[layer])

    @staticmethod
    def page_bytes_of(layers: int, n_kv: int, head_dim: int) -> int:
        """Bytes of one page over all layers."""
        return layers * 2 * n_kv * PAGE_SIZE * (head_dim + 1)

    @property
    def page_bytes(self) -> int:
        layers, _, _, n_kv, _, head_dim = self.data.shape
        return self.page_bytes_of(layers, n_kv, head_dim)

    def copy_page(self, src: int, dst: int) -> None:
        for t in (self.data.view(torch.uint8), self.exps):
            t[:, dst].copy_(t[:, src])


def check_layer(layer: Kv8Layer, what: str) -> tuple[int, int, int]:
    """``(pages, n_kv, D)`` of a layer whose parts fit each other; ``ValueError`` otherwise."""
    data, exps = layer
    shape, parts = data.shape, exps.shape
    if data.dtype != torch.float8_e4m3fn or exps.dtype != torch.uint8:
        raise ValueError(f"{what}: an 8-bit KV layer holds float8_e4m3fn data and uint8 exponents, not {data.dtype} and {exps.dtype}")
    if len(shape) != 5 or shape[1] != 2 or shape[3] != PAGE_SIZE or parts + shape[4:] != shape:
        raise ValueError(f"{what}: data {tuple(shape)} and exponents {tuple(parts)} are not [pages, 2, n_kv, {PAGE_SIZE}, D] and the same without D")
    if not (data.is_contiguous() and exps.is_contiguous()):
        raise ValueError(f"{what}: the parts of an 8-bit KV layer are contiguous")
    if data.device != exps.device:
        raise ValueError(f"{what}: data on {data.device}, exponents on {exps.device}")
    if shape[4] not in HEAD_DIMS:
        raise ValueError(f"{what}: head dim {shape[4]} is none of {HEAD_DIMS}")
    return shape[0], shape[2], shape[4]


def two_to(e: torch.Tensor) -> torch.Tensor:
    """``2.0 ** e`` in fp32, exactly, for integers in ``[-126, 127]``."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(data, exps)`` of rows ``x [..., D]``."""
    x = x.float()
    nan = x.isnan().any(-1)
    amax = torch.nan_to_num(x.abs(), nan=0.0).amax(-1)
    m, e = torch.frexp(amax.clamp(max=torch.finfo(torch.float32).max))  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-E_MAX, E_MAX)
    e = torch.where(amax > 0, e, torch.full_like(e, -E_MAX))
    y = (x * two_to(-e)[..., None]).clamp(-448.0, 448.0)
    y = torch.where(nan[..., None], torch.zeros_like(y), y)
    return y.to(torch.float8_e4m3fn), torch.where(nan, E_NAN, e + E_BIAS).to(torch.uint8)


def dequantise(data: torch.Tensor, exps: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Rows as numbers of ``dtype`` (exact in fp32 and bf16)."""
    scale = two_to(exps.to(torch.int32).clamp(1, 254) - E_BIAS)
    scale = torch.where(exps == E_NAN, torch.full_like(scale, float("nan")), scale)
    return (data.float() * scale[..., None]).to(dtype)
