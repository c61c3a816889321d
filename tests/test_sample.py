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
