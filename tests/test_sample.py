"""The rules of sampling, token by token in plain Python, and what refuses before any GPU is asked."""

import math
import random

import pytest
import torch

from b200serve.ops import torch_ops


def _rules(row, t, k, p, m, u, exclude=()):
    """The rules as they are written down, with exact sums of 64-bit weights."""
    x = [-math.inf if (v != v or i in exclude) else v for i, v in enumerate(row)]
    ids = sorted((i for i in range(len(x)) if x[i] != -math.inf), key=lambda i: (-x[i], i))
    if not ids:
        return -1
    if not t > 0:
        return ids[0]
    top = x[ids[0]]
    w = [1.0 if x[i] == top else math.exp((x[i] - top) / t) for i in ids]
    if 0 < k < len(w):
        w = w[:k]
    kept = [j for j in range(len(w)) if (p >= 1 or math.fsum(w[:j]) <= p * math.fsum(w)) and w[j] >= m and w[j] > 0]
    w = [w[j] for j in kept] or w[:1]
    for j in range(len(w)):
        if math.fsum(w[: j + 1]) > u * math.fsum(w):
            return ids[j]
    return ids[len(w) - 1]


@pytest.mark.parametrize("V", [1, 2, 7, 60])
def test_the_operator_is_the_rules(V):
    rng = random.Random(V)
    n = 200
    rows = [[rng.choice([rng.gauss(0, 2), float(rng.randrange(3)), -math.inf, math.nan]) if rng.random() < 0.9 else 0.5 for _ in range(V)] for _ in range(n)]
    ask = [(rng.choice([0.0, 0.3, 1.0, 2.5]), rng.choice([0, 0, 1, 3, 50, V, V + 1]), rng.choice([1.0, 0.9, 0.4, 0.0]), rng.choice([0.0, 0.0, 0.1, 1.0]),
            rng.random()) for _ in range(n)]
    ban = [[rng.randrange(-2, V + 2) for _ in range(3)] for _ in range(n)]
    t, k, p, m, u = (list(c) for c in zip(*ask))
    x = torch.tensor(rows, dtype=torch.float32)
    f = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
    args = (f(t), torch.tensor(k, dtype=torch.int32), f(p), f(m), f(u))
    got = torch_ops.sample(x, *args, exclude=torch.tensor(ban, dtype=torch.int32))
    as32 = [[float(v) for v in c.tolist()] for c in (args[0], args[2], args[3], args[4])]  # the settings as fp32 holds them
    want = [_rules(x[i].tolist(), as32[0][i], k[i], as32[1][i], as32[2][i], as32[3][i], ban[i]) for i in range(n)]
    assert got.tolist() == want
    assert torch_ops.sample(x, *args).tolist() == [_rules(x[i].tolist(), as32[0][i], k[i], as32[1][i], as32[2][i], as32[3][i]) for i in range(n)]


def test_the_kernels_refuse_logits_of_the_host():
    from b200serve.ops import cuda_ops

    f = torch.zeros(2)
    with pytest.raises(ValueError, match="torch_ops"):
        cuda_ops.sample(torch.zeros(2, 5), f, f.int(), f, f, f)


def test_pick_tokens_takes_every_setting():
    from b200serve.sched.request import Sampling
    from b200serve.sched.sampling import pick_tokens

    torch.manual_seed(0)
    logits = torch.randn(1, 400) * 2
    w = torch.softmax(logits[0].double() / 0.9, -1)
    allowed = set((w >= 0.3 * w.max()).nonzero().view(-1).tolist())
    g = torch.Generator().manual_seed(1)
    got = {pick_tokens(logits, [Sampling(temperature=0.9, min_p=0.3, seed=0)], [g], [None])[0] for _ in range(200)}
    assert got <= allowed and len(got) == len(allowed) > 1
    # more ids to leave out than the operator takes by itself
    order = logits[0].argsort(descending=True).tolist()
    assert pick_tokens(logits, [Sampling()], [None], [set(order[:80])]) == [order[80]]
    assert pick_tokens(logits[:, :3], [Sampling()], [None], [{0, 1, 2}]) == [0]


def test_settings_that_are_no_numbers_filter_nothing():
    """A NaN as top-p or min-p, which no comparison holds for, leaves every token in."""
    g = torch.Generator().manual_seed(3)
    x, n = torch.randn(64, 50, generator=g), 64
    u = torch.rand(n, generator=g)
    one, zero, nan, k = torch.ones(n), torch.zeros(n), torch.full((n,), math.nan), torch.zeros(n, dtype=torch.int32)
    want = torch_ops.sample(x, one, k, one, zero, u)
    assert len(set(want.tolist())) > 20
    for p, m in ((nan, zero), (one, nan), (nan, nan)):
        assert torch.equal(torch_ops.sample(x, one, k, p, m, u), want)
    assert torch.equal(torch_ops.sample(x, one, k + 7, nan, nan, u), torch_ops.sample(x, one, k + 7, one, zero, u))


def _pick64(row, t, k, p, m, u, exclude=()):
    """The rules for a row of thousands, by the tokens that it has and sums in 64 bits."""
    x = row.double().clone()
    x[x.isnan()] = -math.inf
    x[[i for i in exclude if 0 <= i < len(x)]] = -math.inf
    ids = (x > -math.inf).nonzero().view(-1)
    if not len(ids):
        return -1
    v, at = x[ids].sort(descending=True, stable=True)
    ids = ids[at]
    if not t > 0:
        return int(ids[0])
    w = torch.where(v == v[0], 1.0, torch.exp((v - v[0]) / t).nan_to_num(0.0))[: k if k > 0 else None]
    cum = w.cumsum(0)
    if p < 1:
        w = w[cum - w <= p * cum[-1]]
    w = w[(w >= m) & (w > 0)]
    w = w if len(w) else torch.ones(1, dtype=torch.float64)
    cum = w.cumsum(0)
    return int(ids[min(int((cum <= u * cum[-1]).sum()), len(w) - 1)])


def _random_asks(rng, n, V):
    ask = [(rng.choice([0.0, 0.3, 1.0, 1.0, 2.5, 50.0, math.inf]), rng.choice([0, 0, 0, 1, 20, 63, 64, 65, 1000, 2047, 2048, V - 1, V, V + 1]),
            rng.choice([1.0, 0.999, 0.9, 0.5, 1e-6, 0.0]), rng.choice([0.0, 0.0, 1e-4, 0.05, 1.0]), rng.random()) for _ in range(n)]
    f = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
    t, k, p, m, u = (list(c) for c in zip(*ask))
    return f(t), torch.tensor(k, dtype=torch.int32), f(p), f(m), f(u)


@pytest.mark.parametrize("V", [63, 2049, 4096, 4097, 6001])
def test_large_rows_are_the_rules(V):
    """Rows longer than what is put in order at first: steep and flat ones, ties, whole blocks of minus infinity, excluded ids."""
    rng, g = random.Random(V), torch.Generator().manual_seed(V)
    n = 120
    x = 12 - (torch.rand(n, 1, generator=g) * 3) * torch.log(torch.rand(n, V, generator=g) * V + 1)
    x[::4] = x[::4].round()
    x[1::8] = 0.0
    x[2::16, 40:] = -math.inf
    x[3::16, rng.randrange(V)] = math.inf
    x[5::16, : V // 2] = math.nan
    args = _random_asks(rng, n, V)
    ban = torch.cat([x.nan_to_num(-1e9).argmax(-1, keepdim=True), torch.randint(-2, V + 2, (n, 3), generator=g)], 1).int()
    as32 = list(zip(*(a.tolist() for a in args)))
    for dtype in (torch.float32, torch.bfloat16, torch.float16, torch.float64):
        y = x.to(dtype)
        for exclude in (None, ban):
            got = torch_ops.sample(y, *args, exclude=exclude).tolist()
            want = [_pick64(y[i], *as32[i], () if exclude is None else ban[i].tolist()) for i in range(n)]
            assert got == want, dtype
        assert torch.equal(y.nan_to_num(7.5), x.to(dtype).nan_to_num(7.5))  # (the logits stay as they are)
        alone = [int(torch_ops.sample(y[i : i + 1], *(a[i : i + 1] for a in args))[0]) for i in range(0, n, 7)]
        assert alone == torch_ops.sample(y, *args)[::7].tolist()


@pytest.mark.parametrize("ask", [(0.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (0.8, 50, 1.0, 0.05), (1.0, 1000, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05)])
def test_rows_that_need_no_order_of_the_vocabulary_do_without(ask, monkeypatch):
    """The plain form puts as much of a row in order as decides it: a sort of every row's whole vocabulary took ten times as long."""
    n, V = 4, 100000
    g = torch.Generator().manual_seed(1)
    x = 15 - 2 * torch.log(torch.rand(n, V, generator=g) * V + 1)
    f = lambda v: torch.full((n,), v)  # noqa: E731
    sorted_at_all, sort = [0], torch.sort

    def counted(t, *args, **kw):
        sorted_at_all[0] += t.numel()
        return sort(t, *args, **kw)

    args = (f(ask[0]), f(ask[1]).int(), f(ask[2]), f(ask[3]), torch.rand(n, generator=g) * 0.8)
    ban = x.argmax(-1, keepdim=True).int()
    for exclude in (None, ban):
        monkeypatch.setattr(torch, "sort", counted)
        got = torch_ops.sample(x, *args, exclude=exclude).tolist()
        monkeypatch.setattr(torch, "sort", sort)
        as32 = list(zip(*(a.tolist() for a in args)))
        for i in range(n):
            assert got[i] == _pick64(x[i], *as32[i], () if exclude is None else ban[i].tolist())
    assert sorted_at_all[0] <= 2 * 2 * n * 2200


def test_no_rows():
    from b200serve.sched.sampling import pick_tokens

    for V in (1, 50, 5000):
        e = torch.empty(0)
        got = torch_ops.sample(torch.empty(0, V), e, e.int(), e, e, e, exclude=torch.empty(0, 2, dtype=torch.int32))
        assert got.shape == (0,) and got.dtype == torch.int64
        assert pick_tokens(torch.empty(0, V), [], [], []) == []


@pytest.mark.parametrize("graphs", [False, True])
def test_warmup_draws_tokens_of_every_step_size(graphs, monkeypatch):
    """No request pays for the first use of what draws tokens: the LM head's logits and the draw, at every size that a step may have."""
    from b200serve.config import EngineConfig, ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.sched import engine as module

    drawn, pick = [], module.pick_tokens
    monkeypatch.setattr(module, "pick_tokens", lambda logits, *a: (drawn.append(logits.shape[0]), pick(logits, *a))[1])
    w = random_weights(ModelConfig.tiny(), seed=0, dtype=torch.float32, std=0.05, lm_head_std=0.5)
    eng = module.Engine(w, EngineConfig(max_model_len=256, prefill_chunk_tokens=64, max_seqs=6, mtp=False, decode_buckets=(1, 4, 8), graphs_on_cpu=graphs,
                                        cuda_graphs=graphs))
    eng.warmup()
    assert set(drawn) == {1, 4, 6}
    assert not any(eng.stats.values()) and len(eng.cache) == 0 and not eng.has_work() and not eng.running
    assert eng.slots.free == eng.slots.num_slots - 1
    del drawn[:]
    eng.cfg.max_seqs, eng.cfg.decode_buckets = 1000, (1, 512)  # (as many rows as its forms tell apart, not all that there may be)
    eng.warmup()
    assert set(drawn) == {1, 256}
