"""The operators of the 8-bit KV cache, as measurable cases.

A layer of the cache holds keys and values of 64-token pages as ``data [pages, 2, n_kv, 64, D]`` (float8 e4m3) with one power of
two per row of ``D`` numbers, ``exps [pages, 2, n_kv, 64]`` (uint8, biased by 127): a row's numbers are ``data * 2 ** (exps - 127)``.
Page tables name the pages of each sequence, as for the bf16 cache. Four operators work on it:

* ``write``    rows of keys and values are quantised into their sequences' pages;
* ``read``     the rows of given positions come back as bf16;
* ``decode``   gated attention of ``G`` query rows per sequence (1: a decode step, more: a verify pass) over its pages;
* ``prefill``  causal gated attention of spans of new tokens over what their sequences' pages hold, the spans' own keys included.

``run`` computes them with elementary torch operations in 32 bits, or with the framework's calls where ``own`` is set.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
PAGE = 64
E_MAX = 60  # exponents are held in [-60, 60]: rows of up to 448 * 2^60
HEADS = ((16, 2, 256), (16, 2, 256), (8, 1, 64), (4, 1, 128), (8, 8, 64), (6, 3, 128))  # the served model's twice


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    served = {"n_q": 16, "n_kv": 2, "D": 256}
    return [
        # the benchmark's decode batch: one new token of each of 128 requests
        {"name": "write_step_128", "kind": "write", "seqs": 128, "rows": 128, "context": 1088, "spread": 0.06, "mix": 1, **served},
        # a full prefill pass of eight 1024-token prompts
        {"name": "write_pass_8192", "kind": "write", "seqs": 8, "rows": 8192, "context": 0, "spread": 0.0, "mix": 2, **served},
        # one session's cached prefix of odd length, read to be handed to another replica
        {"name": "read_session", "kind": "read", "seqs": 1, "rows": 6001, "context": 0, "spread": 0.0, "mix": 3, **served},
        # the prefixes of many sessions
        {"name": "read_sessions_16", "kind": "read", "seqs": 16, "rows": 98304, "context": 0, "spread": 0.7, "mix": 4, **served},
        # one interactive request: latency
        {"name": "decode_1", "kind": "decode", "seqs": 1, "G": 1, "context": 900, "spread": 0.0, "mix": 5, **served},
        # the benchmark's batch: 128 requests of 1024 prompt tokens
        {"name": "decode_128", "kind": "decode", "seqs": 128, "G": 1, "context": 1088, "spread": 0.06, "mix": 6, **served},
        # a few coding-agent sessions with long contexts
        {"name": "decode_4_long", "kind": "decode", "seqs": 4, "G": 1, "context": 90000, "spread": 0.5, "mix": 7, **served},
        # a speculative step with three drafts per request on a busy server
        {"name": "verify_40", "kind": "decode", "seqs": 40, "G": 4, "context": 4096, "spread": 0.7, "mix": 8, **served},
        # a session's next turn: a short span on top of a cached context
        {"name": "prefill_turn", "kind": "prefill", "seqs": 1, "rows": 61, "context": 3584, "spread": 0.0, "mix": 9, **served},
        # several short prompts of different lengths packed into one pass, heads of 128 numbers
        {"name": "prefill_ragged", "kind": "prefill", "seqs": 7, "rows": 1531, "context": 0, "spread": 0.8, "mix": 10, "n_q": 6, "n_kv": 3, "D": 128},
        # the benchmark's prefill: a full pass of eight 1024-token prompts
        {"name": "prefill_8x1024", "kind": "prefill", "seqs": 8, "rows": 8192, "context": 0, "spread": 0.0, "mix": 11, **served},
        # a full pass of chunks in the middle of long prompts
        {"name": "prefill_4x2048_long", "kind": "prefill", "seqs": 4, "rows": 8192, "context": 28672, "spread": 0.9, "mix": 12, **served},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    """A case of the same ranges: batch, context, rows and kind at random, never more work than the largest listed one."""
    kind = rng.choice(["write", "read", "decode", "decode", "prefill", "prefill"])
    n_q, n_kv, D = rng.choice(HEADS)
    case = {"kind": kind, "spread": round(rng.uniform(0.0, 0.9), 3), "mix": rng.randrange(1 << 20), "n_q": n_q, "n_kv": n_kv, "D": D}
    if kind == "write":
        rows = _log_int(rng, 1, 8192)
        return {**case, "seqs": min(rows, _log_int(rng, 1, 256)), "rows": rows, "context": _log_int(rng, 1, 4096)}
    if kind == "read":
        rows = _log_int(rng, 1, 65536)
        return {**case, "seqs": min(rows, _log_int(rng, 1, 64)), "rows": rows, "context": 0}
    if kind == "decode":
        seqs = _log_int(rng, 1, 256)
        return {**case, "seqs": seqs, "G": rng.choice([1, 1, 2, 3, 4, 6]), "context": _log_int(rng, 1, min(90000, max(64, 200000 // seqs)))}
    rows = _log_int(rng, 2, 8192)
    seqs = min(rows, _log_int(rng, 1, 16))
    return {**case, "seqs": seqs, "rows": rows, "context": _log_int(rng, 1, min(28672, 90_000_000 // rows, 200000 // seqs))}


def _spread(total: int, parts: int, spread: float, rng) -> list[int]:
    """``parts`` positive numbers that add up to ``total``, uneven by ``spread``."""
    w = [rng.uniform(1.0 - spread, 1.0 + spread) + 1e-3 for _ in range(parts)]
    n = [1 + int((total - parts) * x / sum(w)) for x in w]
    n[-1] += total - sum(n)
    return n


def _shape(case: dict):
    """Per sequence: (position of its first row, its rows). Goes by the case alone."""
    rng = random.Random(case["mix"])
    B, spread = case["seqs"], case["spread"]
    rows = [case["G"]] * B if case["kind"] == "decode" else _spread(case["rows"], B, spread, rng)
    pos0 = [int(case["context"] * rng.uniform(1.0 - spread, 1.0)) if case["context"] else 0 for _ in range(B)]
    return pos0, rows


def _visible(case: dict) -> tuple[int, int]:
    """Keys that the sequences hold, and (row, key) pairs that the masks leave."""
    pos0, rows = _shape(case)
    return sum(p + n for p, n in zip(pos0, rows)), sum(n * p + n * (n + 1) // 2 for p, n in zip(pos0, rows))


def work(case: dict) -> dict:
    n_q, n_kv, D = case["n_q"], case["n_kv"], case["D"]
    T = sum(_shape(case)[1])
    row = n_kv * 2 * (D + 1)  # of a token in the cache
    if case["kind"] in ("write", "read"):
        return {"bytes": T * (row + n_kv * 2 * D * 2 + 12), "flops": T * n_kv * 2 * D * 3}
    keys, pairs = _visible(case)
    return {"bytes": keys * row + T * n_q * D * 2 * 3, "flops": pairs * n_q * D * 4}


# ------------------------------------------------------------------ inputs
def _quantised(shape, g):
    """Rows of normal numbers with a scale of their own and a few strong columns, as a cache holds them."""
    D = shape[-1]
    x = torch.randn(shape, device=DEV, generator=g)
    x *= torch.exp2(torch.randn(shape[:-1], device=DEV, generator=g) * 0.5)[..., None]
    x *= torch.where(torch.rand(D, device=DEV, generator=g) < 0.02, 4.0, 1.0)
    return _quantise(x)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    n_q, n_kv, D = case["n_q"], case["n_kv"], case["D"]
    pos0, rows = _shape(case)
    B, T = len(rows), sum(rows)
    pages = [(p + n + PAGE - 1) // PAGE for p, n in zip(pos0, rows)]
    n_pages = sum(pages) + 1  # page 0 belongs to nobody
    ids = (torch.randperm(n_pages - 1, device=DEV, generator=g) + 1).int().split(pages)
    tables = torch.nn.utils.rnn.pad_sequence(ids, batch_first=True)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    seq = torch.repeat_interleave(torch.arange(B, dtype=torch.int32), torch.tensor(rows)).to(DEV)
    positions = torch.cat([torch.arange(p, p + n) for p, n in zip(pos0, rows)]).to(DEV)
    st = {"case": case, "tables": tables, "positions": positions, "seq": seq, "starts": starts, "pos0": pos0}
    if case["kind"] == "write":
        # keys and values are slices of the rows of a merged projection, as attention has them
        kv = torch.randn(T, 2 * n_kv * D, device=DEV, generator=g) * torch.exp2(torch.randn(T, 1, device=DEV, generator=g))
        kv = kv.bfloat16()
        st["k"], st["v"] = kv[:, : n_kv * D].view(T, n_kv, D), kv[:, n_kv * D :].view(T, n_kv, D)
        st["data"] = torch.zeros(n_pages, 2, n_kv, PAGE, D, device=DEV).to(torch.float8_e4m3fn)
        st["exps"] = torch.full((n_pages, 2, n_kv, PAGE), 127, dtype=torch.uint8, device=DEV)
        return st
    st["data"], st["exps"] = _quantised((n_pages, 2, n_kv, PAGE, D), g)
    if case["kind"] != "read":
        st["q"] = (torch.randn(T, n_q, D, device=DEV, generator=g) * 1.2).bfloat16()
        st["gate"] = torch.randn(T, n_q * D, device=DEV, generator=g).bfloat16()
        # of a pass, shared by its layers: the spans' first rows and positions
        st["spans"] = (torch.tensor(starts, dtype=torch.int32, device=DEV), torch.tensor(pos0, dtype=torch.int32, device=DEV))
    return st


# ------------------------------------------------------------------ the plain form
def _quantise(x: torch.Tensor):
    """Rows of ``x`` as e4m3 and an exponent: the smallest power of two that brings the row's largest number to 448 or below."""
    x = x.float()
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, -E_MAX).clamp(-E_MAX, E_MAX)
    y = (x * _two_to(-e)[..., None]).clamp(-448.0, 448.0)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _two_to(e: torch.Tensor) -> torch.Tensor:
    """2 ** e, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _values(data: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    return data.float() * _two_to(exps.to(torch.int32) - 127)[..., None]


def _padded(st: dict):
    """Per sequence, padded to the longest: the row of every query (and whether it is one), its position."""
    starts, pos0 = torch.tensor(st["starts"], device=DEV), torch.tensor(st["pos0"], device=DEV)
    n = starts[1:] - starts[:-1]
    at = torch.arange(int(max(b - a for a, b in zip(st["starts"], st["starts"][1:]))), device=DEV)
    real = at[None, :] < n[:, None]
    return (starts[:-1, None] + at[None, :]).where(real, 0), real, pos0[:, None] + at[None, :]


def _plain_attention(st: dict) -> torch.Tensor:
    case = st["case"]
    n_q, n_kv, D = case["n_q"], case["n_kv"], case["D"]
    rows, real, pos = _padded(st)
    B, n = rows.shape
    pages = st["tables"].long()
    kv = _values(st["data"][pages], st["exps"][pages])  # [B, pages, 2, n_kv, 64, D]
    k, v = (kv[:, :, i].transpose(1, 2).flatten(2, 3) for i in (0, 1))  # [B, n_kv, keys, D]
    q = st["q"][rows].float().view(B, n, n_kv, n_q // n_kv, D).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, n_kv, heads * n, D]
    s = (q @ k.transpose(-1, -2)).mul_(D ** -0.5).view(B, n_kv, n_q // n_kv, n, -1)
    hidden = torch.arange(s.shape[-1], device=DEV)[None, None, :] > pos[:, :, None]
    s.masked_fill_(hidden[:, None, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (s.flatten(2, 3) @ v).view(B, n_kv, n_q // n_kv, n, D) / s.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, n_q * D)[real]  # rows in their order
    return (o / (1.0 + torch.exp(-st["gate"].float()))).to(torch.bfloat16)


def _where(st: dict):
    """Page and place in it of every row."""
    return st["tables"][st["seq"].long(), st["positions"] // PAGE].long(), st["positions"] % PAGE


def run(st: dict):
    case = st["case"]
    kind = case["kind"]
    if own:
        from b200serve.ops import cuda_ops
        from b200serve.ops.kv8 import Kv8Layer

        layer = Kv8Layer(st["data"], st["exps"])
        if kind == "write":
            cuda_ops.kv8_write(layer, st["k"], st["v"], st["positions"], st["seq"], st["tables"])
            return {"data": st["data"], "exps": st["exps"]}
        if kind == "read":
            k, v = cuda_ops.kv8_read(layer, st["positions"], st["seq"], st["tables"])
            return {"k": k, "v": v}
        if kind == "decode":
            return {"out": cuda_ops.kv8_decode(st["q"], st["gate"], layer, st["tables"], st["positions"], case["G"])}
        return {"out": cuda_ops.kv8_prefill(st["q"], st["gate"], layer, st["tables"], st["starts"], st["pos0"], meta=st["spans"])}
    if kind == "write":
        page, at = _where(st)
        for i, x in enumerate((st["k"], st["v"])):
            data, exps = _quantise(x)
            st["data"].view(torch.uint8)[page, i, :, at] = data.view(torch.uint8)
            st["exps"][page, i, :, at] = exps
        return {"data": st["data"], "exps": st["exps"]}
    if kind == "read":
        page, at = _where(st)
        k, v = (_values(st["data"].view(torch.uint8)[page, i, :, at].view(torch.float8_e4m3fn), st["exps"][page, i, :, at]).bfloat16()
                for i in (0, 1))
        return {"k": k, "v": v}
    return {"out": _plain_attention(st)}


# ------------------------------------------------------------------ in 64 bits
def _power(e: torch.Tensor) -> torch.Tensor:
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    data, exps = st["data"], st["exps"]
    n_q, n_kv, D = case["n_q"], case["n_kv"], case["D"]
    seq, pos, tables = st["seq"].long(), st["positions"], st["tables"].long()
    if case["kind"] == "write":
        out, eout = data.double(), exps.clone()
        for i, x in enumerate((st["k"].double(), st["v"].double())):
            top = x.abs().amax(-1).clamp(min=2.0 ** -200)
            e = torch.floor(torch.log2(top / 448.0))  # off by one at most: a logarithm is rounded
            e = e + (top > 448.0 * _power(e)) + (top > 448.0 * _power(e + 1)) - (top <= 448.0 * _power(e - 1)).double()
            e = e.clamp(-E_MAX, E_MAX)
            y = x * _power(-e)[..., None]
            # e4m3: steps of 2^(exponent - 3), of 2^-9 below 2^-6; ties to even
            step = _power(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
            page, at = tables[seq, pos // PAGE], pos % PAGE
            out[page, i, :, at] = torch.round(y / step) * step
            eout[page, i, :, at] = (e + 127).to(torch.uint8)
        return {"data": out, "exps": eout}
    if case["kind"] == "read":
        got = []
        for i in (0, 1):
            flat = (tables[seq, pos // PAGE][:, None] * 2 + i) * n_kv + torch.arange(n_kv, device=DEV)[None, :]
            flat = flat * PAGE + (pos % PAGE)[:, None]
            x = data.view(torch.uint8).view(-1, D)[flat].view(torch.float8_e4m3fn).double()
            got.append(x * _power(exps.view(-1)[flat].int() - 127)[..., None])
        return {"k": got[0], "v": got[1]}
    group = n_q // n_kv
    out = torch.empty(len(pos), n_q, D, dtype=torch.float64, device=DEV)
    for b, (p0, a, z) in enumerate(zip(st["pos0"], st["starts"], st["starts"][1:])):
        total = p0 + z - a
        pages = tables[b, : (total + PAGE - 1) // PAGE]
        mask = torch.arange(total, device=DEV)[None, :] <= pos[a:z, None]
        for h in range(n_kv):
            x = data[pages, :, h].double() * _power(exps[pages, :, h].int() - 127)[..., None]
            k, v = x[:, 0].reshape(-1, D)[:total], x[:, 1].reshape(-1, D)[:total]
            for j in range(h * group, h * group + group):
                s = torch.where(mask, (st["q"][a:z, j].double() @ k.T) / math.sqrt(D), -math.inf)
                out[a:z, j] = torch.softmax(s, -1) @ v
    return {"out": out.reshape(len(pos), n_q * D) * torch.sigmoid(st["gate"].double())}
