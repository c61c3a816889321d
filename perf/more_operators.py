"""The operators of a batch whose requests each bring something of their own, as measurable cases.

* ``sample``  the next token of every row of logits by the row's own temperature, top-k, top-p and min-p, from one given uniform
  number per row. With ``x`` the row's logits (NaN as minus infinity), ``m`` their maximum and ``w_i = exp((x_i - m) / T)``, tokens
  stand in descending order of ``x``, the lower id first among equals. Kept are the first ``k``; of those the ones before which at most
  ``top_p`` of the k tokens' weight stands; of those the ones with ``w_i >= min_p``. The pick is the first kept token up to which more
  than ``u`` of the kept weight stands. ``T = 0`` picks the first token of the order; a row with nothing left gives -1.
* ``lora``    a projection that all rows share, with the low-rank adapter of each row's own request beside it:
  ``y_t = x_t W^T + s_a (x_t A_a^T) B_a^T`` with ``a`` the row's adapter; a row of adapter -1 has none.

``run`` computes them with elementary torch operations, or with the framework's calls where ``own`` is set. What a draw or a nucleus
border decides lies between numbers as near as 1e-9, so ``sample`` is computed in 64 bits; ``lora`` in 32.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    served = {"V": 248320, "type": "fp32"}  # the served model's vocabulary; its LM head gives fp32 logits
    return [
        # one interactive request: latency
        {"name": "sample_1", "kind": "sample", "n": 1, "ask": "chat", "banned": 0, **served},
        # a small server, every request with a nucleus of its own
        {"name": "sample_16_nucleus", "kind": "sample", "n": 16, "ask": "nucleus", "banned": 0, **served},
        # a decode step of 128 requests that ask for different things, greedy ones among them, two end-of-sequence ids still forbidden
        {"name": "sample_128_mixed", "kind": "sample", "n": 128, "ask": "mixed", "banned": 2, **served},
        # the protocol's defaults (temperature 1, nothing filtered) on a full server
        {"name": "sample_256_open", "kind": "sample", "n": 256, "ask": "open", "banned": 0, **served},
        # 16-bit logits of another vocabulary, many of them equal, an odd size
        {"name": "sample_61_bf16", "kind": "sample", "n": 61, "V": 100003, "type": "bf16", "ask": "mixed", "banned": 1},
        # the tiny checkpoint
        {"name": "sample_5_tiny", "kind": "sample", "n": 5, "V": 1024, "type": "fp32", "ask": "mixed", "banned": 2},
        # one interactive request with an adapter: attention input projection of a decode step
        {"name": "lora_step_1", "kind": "lora", "T": 1, "seqs": 1, "N": 9216, "K": 2048, "L": 8, "R": 16, "bare": 0.0, "out": "bf16"},
        # the same of the benchmark's decode batch, 32 adapters among 128 requests, every eighth request without one
        {"name": "lora_step_128", "kind": "lora", "T": 128, "seqs": 128, "N": 9216, "K": 2048, "L": 32, "R": 16, "bare": 0.125, "out": "bf16"},
        # output projection of a smaller batch, larger adapters
        {"name": "lora_out_40", "kind": "lora", "T": 40, "seqs": 40, "N": 2048, "K": 4096, "L": 12, "R": 64, "bare": 0.0, "out": "bf16"},
        # several prompts of different lengths in one pass: recurrent layer's input projection
        {"name": "lora_ragged_1531", "kind": "lora", "T": 1531, "seqs": 7, "N": 12352, "K": 2048, "L": 7, "R": 32, "bare": 0.2, "out": "bf16"},
        # a full prefill pass of eight prompts
        {"name": "lora_pass_8192", "kind": "lora", "T": 8192, "seqs": 8, "N": 9216, "K": 2048, "L": 8, "R": 16, "bare": 0.0, "out": "bf16"},
        # odd sizes, fp32 rows
        {"name": "lora_odd_77", "kind": "lora", "T": 77, "seqs": 9, "N": 1003, "K": 520, "L": 3, "R": 24, "bare": 0.3, "out": "fp32"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    """A case of the same ranges: rows, vocabulary, settings, or rows, projection, adapters and their ranks at random."""
    if rng.random() < 0.5:
        return {"kind": "sample", "n": _log_int(rng, 1, 256), "V": _log_int(rng, 1000, 248320), "type": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                "ask": rng.choice(["chat", "nucleus", "mixed", "mixed", "open"]), "banned": rng.choice([0, 0, 1, 2, 5])}
    T = _log_int(rng, 1, 8192)
    R = rng.choice([8, 16, 16, 24, 32, 64, 64, 96, 128])
    K = 8 * _log_int(rng, 8, 512)
    most = max(64, min(12352, int(1.4e11 / (T * K))))
    return {"kind": "lora", "T": T, "seqs": min(T, _log_int(rng, 1, 256)), "N": _log_int(rng, 64, most), "K": K, "L": _log_int(rng, 1, min(64, 2048 // R)),
            "R": R, "bare": rng.choice([0.0, 0.0, 0.2, 0.9]), "out": rng.choice(["bf16", "bf16", "bf16", "fp32"])}


def _rows(case: dict) -> list[int]:
    """Adapter of every row: the rows of a sequence follow each other and share one. Goes by the case alone."""
    rng = random.Random("%(T)d %(seqs)d %(L)d %(N)d" % case)
    T, n = case["T"], case["seqs"]
    cuts = sorted(rng.sample(range(1, T), n - 1)) if n < T else list(range(1, T))
    of = [-1 if rng.random() < case["bare"] else rng.randrange(case["L"]) for _ in range(n)]
    ids, at = [], 0
    for a, z in zip(of, cuts + [T]):
        ids += [a] * (z - at)
        at = z
    return ids


def work(case: dict) -> dict:
    if case["kind"] == "sample":
        n, V = case["n"], case["V"]
        return {"bytes": n * (V * torch.finfo(TYPES[case["type"]]).bits // 8 + 28 + 4 * case["banned"]), "flops": n * V * 4}
    T, N, K, R = case["T"], case["N"], case["K"], case["R"]
    ids = [a for a in _rows(case) if a >= 0]
    out = 4 if case["out"] == "fp32" else 2
    return {"bytes": 2 * (T * K + N * K + len(set(ids)) * R * (N + K)) + T * (N * out + 4), "flops": 2 * T * N * K + 2 * len(ids) * R * (N + K)}


# ------------------------------------------------------------------ inputs
def _asks(kind: str, n: int, rng) -> list[tuple]:
    """(temperature, top_k, top_p, min_p) per row."""
    if kind == "chat":
        return [(0.7, 20, 0.8, 0.0)] * n
    if kind == "open":
        return [(1.0, 0, 1.0, 0.0)] * n
    if kind == "nucleus":
        return [(rng.choice([0.6, 0.8, 1.0]), 0, rng.choice([0.8, 0.9, 0.95]), 0.0) for _ in range(n)]
    mix = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (0.6, 0, 0.95, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 1.0, 0.0),
           (1.3, 0, 0.9, 0.02), (1.0, 1000, 0.99, 0.0), (1.5, 0, 1.0, 0.0), (0.3, 0, 0.999, 0.0)]
    return [rng.choice(mix) for _ in range(n)]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "sample":
        n, V = case["n"], case["V"]
        # likelihoods that fall with a power of the token's rank, as a language model's do: some rows are sure, some wide open
        steep = torch.rand(n, 1, device=DEV, generator=g) * 1.6 + 1.1
        x = torch.rand(n, V, device=DEV, generator=g).mul_(V).add_(1.0).log_().mul_(-steep).add_(20.0)
        x += torch.randn(n, V, device=DEV, generator=g) * 0.3
        ask = _asks(case["ask"], n, random.Random(seed))
        t, k, p, m = (list(c) for c in zip(*ask))
        st = {"case": case, "logits": x.to(TYPES[case["type"]]), "u": torch.rand(n, device=DEV, generator=g),
              "temperature": torch.tensor(t, dtype=torch.float32, device=DEV), "top_k": torch.tensor(k, dtype=torch.int32, device=DEV),
              "top_p": torch.tensor(p, dtype=torch.float32, device=DEV), "min_p": torch.tensor(m, dtype=torch.float32, device=DEV), "exclude": None}
        if case["banned"]:
            st["exclude"] = torch.randint(0, V, (n, case["banned"]), device=DEV, generator=g, dtype=torch.int32)
            st["exclude"][:, 0] = st["logits"].argmax(-1).int()  # what a request would have picked
        return st
    T, N, K, L, R = (case[c] for c in "TNKLR")
    bf = lambda *shape, by: (torch.randn(*shape, device=DEV, generator=g) * by).bfloat16()  # noqa: E731
    scale = torch.full((L,), 2.0, device=DEV)
    scale[::3] = 0.5
    # adapters move a projection's outputs by a third or so
    return {"case": case, "x": bf(T, K, by=1.0), "w": bf(N, K, by=K ** -0.5), "a": bf(L, R, K, by=K ** -0.5), "b": bf(L, N, R, by=0.25 * R ** -0.5),
            "scale": scale, "rows": torch.tensor(_rows(case), dtype=torch.int32).to(DEV)}


# ------------------------------------------------------------------ the plain form
def _plain_sample(st: dict) -> torch.Tensor:
    x = st["logits"].double()
    n, V = x.shape
    x = torch.where(x.isnan(), -math.inf, x)
    if st["exclude"] is not None:
        x.scatter_(1, st["exclude"].long(), -math.inf)
    x, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = st["temperature"] <= 0
    t = torch.where(greedy, 1.0, st["temperature"].double())[:, None]
    w = torch.where(x == x[:, :1], 1.0, torch.exp((x - x[:, :1]) / t))
    w = torch.where(x == -math.inf, 0.0, w)
    rank = torch.arange(V, device=DEV)[None, :]
    k = st["top_k"].long()[:, None]
    w.masked_fill_((k > 0) & (rank >= k), 0.0)
    cum = torch.cumsum(w, -1)
    top_p = st["top_p"].double()[:, None]
    keep = (cum - w <= top_p * cum[:, -1:]) | (top_p >= 1.0)
    keep &= (w >= st["min_p"].double()[:, None]) & (w > 0.0)
    last = keep.sum(-1, keepdim=True) - 1  # the kept tokens are the first ones
    total = cum.gather(1, last.clamp(min=0))
    at = (cum <= st["u"].double()[:, None] * total).sum(-1, keepdim=True)
    at = torch.where(greedy[:, None], 0, torch.minimum(at, last.clamp(min=0)))
    return torch.where(x[:, 0] == -math.inf, -1, ids.gather(1, at)[:, 0])


def _plain_lora(st: dict) -> torch.Tensor:
    case = st["case"]
    L, R = case["L"], case["R"]
    x = st["x"].float()
    mine = (st["rows"][:, None] == torch.arange(L, device=DEV)[None, :]) * st["scale"][None, :]
    h = (x @ st["a"].float().view(L * R, -1).T).view(-1, L, R) * mine[:, :, None]
    y = x @ st["w"].float().T + h.view(-1, L * R) @ st["b"].float().transpose(1, 2).reshape(L * R, -1)
    return y.to(TYPES[case["out"]])


def run(st: dict):
    case = st["case"]
    if own:
        from b200serve.ops import cuda_ops
        from b200serve.ops.lora import LoraWeights

        if case["kind"] == "sample":
            return {"ids": cuda_ops.sample(st["logits"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], st["u"], exclude=st["exclude"])}
        adapters = LoraWeights(st["a"], st["b"], st["scale"])
        return {"y": cuda_ops.lora_linear(st["x"], st["w"], adapters, st["rows"], out_dtype=TYPES[case["out"]])}
    return {"ids": _plain_sample(st)} if case["kind"] == "sample" else {"y": _plain_lora(st)}


# ------------------------------------------------------------------ in 64 bits
def _exact_pick(x: torch.Tensor, t: float, k: int, p: float, m: float, u: float) -> int:
    """One row, by its tokens alone: the order from one sort of (value, id) pairs."""
    real = torch.nonzero(x > -math.inf).view(-1)
    if not len(real):
        return -1
    v, at = x[real].sort(descending=True)
    new = torch.cat([torch.zeros(1, dtype=torch.bool, device=DEV), v[1:] != v[:-1]])
    ids = real[at]
    ids = ids[torch.argsort(new.cumsum(0) * len(x) + ids)]  # equal values by their ids
    if t <= 0:
        return int(ids[0])
    v = x[ids][: k if k > 0 else None]
    w = torch.exp((v - v[0]) / t)
    before = w.cumsum(0) - w
    if p < 1:
        w = w[before <= p * w.sum()]
    w = w[w >= m]
    up = w.cumsum(0)
    return int(ids[min(int((up <= u * up[-1]).sum()), len(w) - 1)])


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "sample":
        x = st["logits"].double()
        if st["exclude"] is not None:
            for c in st["exclude"].long().T:
                x[torch.arange(len(x), device=DEV), c] = -math.inf
        asks = zip(*(st[c].double().tolist() for c in ("temperature", "top_k", "top_p", "min_p", "u")))
        return {"ids": torch.tensor([_exact_pick(r, t, int(k), p, m, u) for r, (t, k, p, m, u) in zip(x, asks)], device=DEV)}
    x = st["x"].double()
    y = x @ st["w"].double().T
    for i in range(case["L"]):
        at = torch.nonzero(st["rows"] == i).view(-1)
        y[at] += (x[at] @ st["a"][i].double().T) @ st["b"][i].double().T * st["scale"][i].double()
    return {"y": y}
