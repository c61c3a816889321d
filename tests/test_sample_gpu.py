"""The sampling kernels against the rules in 64 bits."""

import math

import pytest
import torch

from b200serve.ops import torch_ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
# (temperature, top_k, top_p, min_p): each rule alone, together, and at its ends
ASKS = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (0.6, 0, 0.95, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 1.0, 0.1), (1.3, 0, 0.9, 0.02),
        (1.0, 1000, 0.99, 0.0), (1.5, 0, 1.0, 1e-5), (2.0, 30000, 0.999, 1e-6), (1.0, 1, 1.0, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 0.0, 0.0),
        (100.0, 0, 0.5, 0.0), (0.01, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0), (math.inf, 0, 1.0, 0.0), (0.5, 1 << 30, 0.7, 0.0), (3.0, 7000, 1.0, 0.0)]


@pytest.fixture(scope="module")
def C():
    from b200serve.ops import cuda_ops

    cuda_ops.lib()
    return cuda_ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(n, V, seed, dtype=torch.float32):
    """Likelihoods that fall with a power of the rank, from sure rows to wide open ones."""
    g = _gen(seed)
    steep = torch.rand(n, 1, device=DEV, generator=g) * 2 + 0.5
    x = 15 - steep * torch.log(torch.rand(n, V, device=DEV, generator=g) * V + 1)
    return (x + torch.randn(n, V, device=DEV, generator=g) * 0.3).to(dtype)


def _settings(asks, n, seed=0):
    g = _gen(seed + 1)
    asks = [asks[i % len(asks)] for i in range(n)]
    t, k, p, m = zip(*asks)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
    return f(t), torch.tensor(k, dtype=torch.int32, device=DEV), f(p), f(m), torch.rand(n, device=DEV, generator=g)


def _same(C, logits, settings, exclude=None):
    got = C.sample(logits, *settings, exclude=exclude)
    want = torch_ops.sample(logits, *settings, exclude=exclude)
    bad = (got != want).nonzero().view(-1).tolist()
    assert not bad, [(i, int(got[i]), int(want[i]), *(float(t[i]) for t in settings)) for i in bad[:5]]
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 2047, 2048, 2049, 5003, 16384, 16385, 50021, 248320])
def test_every_rule_at_every_size(C, V, dtype):
    n = len(ASKS) * (3 if V < 100000 else 1)
    _same(C, _logits(n, V, V, dtype), _settings(ASKS, n, V))


@pytest.mark.parametrize("n", [1, 2, 7, 64, 300])
def test_rows(C, n):
    _same(C, _logits(n, 9001, n), _settings(ASKS, n, n))


def test_a_row_of_equal_logits(C):
    """Ties alone: the order is that of the ids, and whole groups are cut by count and by weight."""
    for V in (5, 2048, 3000, 70000):
        n = len(ASKS)
        x = torch.full((n, V), 2.5, device=DEV)
        _same(C, x, _settings(ASKS, n, V))
        x[:, ::2] = 2.25
        _same(C, x, _settings(ASKS, n, V))
        _same(C, (torch.randint(0, 4, (n, V), device=DEV, generator=_gen(V)) * 0.5), _settings(ASKS, n, V + 1))


@pytest.mark.parametrize("V", [1 << 18, (1 << 18) + 1, 1 << 22])
def test_equal_logits_that_fill_every_part_of_the_search(C, V):
    """2^14 and 2^18 tokens of the largest weight in each of 16 parts: their sums take all the bits that there are."""
    asks = [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.5, 0.0), (1.0, V - 1, 0.9, 0.0), (1.0, 0, 1.0, 0.5)]
    _same(C, torch.full((len(asks), V), -7.0, device=DEV), _settings(asks, len(asks), V))
    x = torch.full((len(asks), V), 1.0, device=DEV)
    x[:, V // 16 : V // 8] = 2.0
    _same(C, x, _settings(asks, len(asks), V + 1))


@pytest.mark.parametrize("V", [100003, 248320, 262145, 300001])
def test_draws_among_tokens_of_little_weight(C, V):
    """The last of the weight lies in thousands of equal tokens of 1e-11 of the largest one's: sums need their bits there as well."""
    n = 40
    asks = [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (1.0, V - 1, 1.0, 0.0), (0.9, 0, 1.0, 1e-13)]
    t, k, p, m, u = _settings(asks, n, V)
    u = 1 - torch.arange(1, n + 1, device=DEV) * 2.0**-24
    x = (torch.randn(n, V, device=DEV, generator=_gen(V)) * 2).round()
    x[:, 17] = 30.0
    for dtype in (torch.float32, torch.float16):
        _same(C, x.to(dtype), (t, k, p, m, u))
    _same(C, x + torch.rand(n, V, device=DEV, generator=_gen(V + 1)), (t, k, p, m, u))


def test_few_distinct_values_in_a_large_vocabulary(C):
    n, V = 2 * len(ASKS), 120001
    g = _gen(3)
    x = (torch.randn(n, V, device=DEV, generator=g) * 1.5).bfloat16()
    x[:, torch.randint(0, V, (40,), device=DEV, generator=g)] = 6.0
    _same(C, x, _settings(ASKS, n))


def test_signed_zeros_are_equal(C):
    n, V = len(ASKS), 4099
    x = torch.full((n, V), -20.0, device=DEV)
    x[:, 100:4000:3] = 0.0
    x[:, 101:4000:3] = -0.0
    _same(C, x, _settings(ASKS, n))


def test_masked_logits(C):
    """Most of the vocabulary masked by minus infinity, by the type's lowest value or by NaN; rows with one token, rows with none."""
    for V in (1500, 30011):
        for hole in (-math.inf, torch.finfo(torch.float32).min, math.nan, -1e30):
            n = len(ASKS)
            x = _logits(n, V, 5)
            keep = torch.rand(n, V, device=DEV, generator=_gen(6)) < 0.004
            keep[:, 17] = True
            keep[1] = False
            keep[2] = False
            keep[2, V - 1] = True
            x = torch.where(keep, x, hole)
            got = _same(C, x, _settings(ASKS, n))
            if hole != hole or hole == -math.inf:
                assert got[1] == -1 and got[2] == V - 1


def test_infinite_and_far_logits(C):
    n, V = len(ASKS), 20003
    x = _logits(n, V, 7)
    x[:, 77] = math.inf
    _same(C, x, _settings(ASKS, n))
    x[:, 5] = math.inf
    x[:, 12345] = math.inf
    _same(C, x, _settings(ASKS, n))
    x = _logits(n, V, 8) * 1e36
    _same(C, x, _settings(ASKS, n))
    x = _logits(n, V, 8) * 1e-36
    _same(C, x, _settings(ASKS, n))
    x = _logits(n, V, 9)
    x[:, 9000] = 3e38  # one far token among ordinary ones
    x[:, 9001] = -3e38
    _same(C, x, _settings(ASKS, n))


def test_sorted_and_clustered_vocabularies(C):
    """Logits whose places tell their size: in order, in reverse, in one block, in a period."""
    n, V = len(ASKS), 64000
    x = _logits(n, V, 10).sort(-1).values
    _same(C, x, _settings(ASKS, n))
    _same(C, x.flip(-1), _settings(ASKS, n, 1))
    y = _logits(n, V, 11) - 12
    y[:, 30000:33000] += 12
    _same(C, y, _settings(ASKS, n, 2))
    z = _logits(n, V, 12) - 10
    z[:, ::256] += 10
    _same(C, z, _settings(ASKS, n, 3))
    z = _logits(n, V, 12) - 10
    z[:, 255::256] += 10
    _same(C, z, _settings(ASKS, n, 3))


def test_exclude(C):
    n, V = len(ASKS), 12007
    x = _logits(n, V, 13)
    order = x.argsort(-1, descending=True)
    for m in (1, 3, 64):
        ex = order[:, :m].int().contiguous()
        got = _same(C, x, _settings(ASKS, n), ex)
        assert not (got[:, None] == ex).any()
    ex = torch.tensor([-1, V, 5, 5, 1 << 30, -(1 << 31), 0, V - 1], dtype=torch.int32, device=DEV).repeat(n, 1)
    _same(C, x, _settings(ASKS, n), ex)
    _same(C, x, _settings(ASKS, n), ex[:, :0].contiguous())
    small = _logits(4, 3, 14)
    got = _same(C, small, _settings([(1.0, 0, 1.0, 0.0)], 4), torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV).repeat(4, 1))
    assert (got == -1).all()


def test_uniform_numbers_at_their_ends(C):
    for V in (700, 40009):
        for u in (0.0, 1 - 2.0 ** -24, 2.0 ** -149):
            n = len(ASKS)
            t, k, p, m, _ = _settings(ASKS, n)
            _same(C, _logits(n, V, 15), (t, k, p, m, torch.full((n,), u, device=DEV)))


def test_strides_and_out(C):
    big = _logits(24, 33000, 16)
    for x in (big[::2, 7:30010], big[:, 1:20002], big[3:9, :10001].clone()[:, 1:], big.bfloat16()[1::3, 3:]):
        n = x.shape[0]
        s = _settings(ASKS, n)
        _same(C, x, s)
        out = torch.full((n + 2,), -7, dtype=torch.int64, device=DEV)
        got = C.sample(x, *s, out=out[1:-1])
        assert got.data_ptr() == out[1:].data_ptr() and out[0] == -7 and out[-1] == -7
        assert torch.equal(got, torch_ops.sample(x, *s))
    t = torch.randn(50, 9, device=DEV).t()  # tokens further apart than rows
    _same(C, t, _settings(ASKS, 9))


def test_a_pick_does_not_depend_on_the_batch(C):
    n, V = 40, 60001
    x, s = _logits(n, V, 17), _settings(ASKS, n)
    together = C.sample(x, *s)
    for a, b in ((0, 1), (7, 8), (3, 20), (39, 40)):
        assert torch.equal(C.sample(x[a:b], *(t[a:b] for t in s)), together[a:b])
    for _ in range(5):
        assert torch.equal(C.sample(x, *s), together)


def test_draws_follow_the_weights(C):
    """Each token's share of 40,000 evenly spaced draws is its weight's to one draw at either of its borders."""
    n = 40000
    w = torch.tensor([0.5, 0.25, 0.125, 0.125], dtype=torch.float64)
    x = torch.log(w).float().to(DEV)[None, :].expand(n, 4)
    f = lambda v: torch.full((n,), v, device=DEV)  # noqa: E731
    got = C.sample(x, f(1.0), torch.zeros(n, dtype=torch.int32, device=DEV), f(1.0), f(0.0), (torch.arange(n, device=DEV) + 0.5) / n)
    assert ((got.bincount(minlength=4).cpu() - w * n).abs() <= 2).all()


def test_captured_and_replayed_on_two_streams(C):
    n, V = 20, 30011
    x, s = _logits(n, V, 18), _settings(ASKS, n)
    C.sample(x, *s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(C.sample(x, *s))
        graphs.append(g)
    for seed in (19, 20):
        x.copy_(_logits(n, V, seed))
        for t, new in zip(s, _settings(ASKS, n, seed)):
            t.copy_(new)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        want = torch_ops.sample(x, *s)
        assert all(torch.equal(o, want) for o in outs)


def test_no_rows(C):
    s = [t[:0] for t in _settings(ASKS, 1)]
    assert C.sample(torch.zeros(0, 100, device=DEV), *s).shape == (0,)


def test_refusals(C):
    x, s = _logits(3, 50, 21), _settings(ASKS, 3)
    with pytest.raises(ValueError, match="torch_ops"):
        C.sample(x.cpu(), *s)
    for bad in (x.double(), x[0], x[None], x[:, :0]):
        with pytest.raises(ValueError, match="logits"):
            C.sample(bad, *s)
    for i, name in enumerate(("temperature", "top_k", "top_p", "min_p", "u")):
        for t in (s[i][:2], s[i].cpu(), s[i].double(), s[i].repeat(2)[::2]):
            with pytest.raises(ValueError, match=name):
                C.sample(x, *s[:i], t, *s[i + 1:])
    for e in (torch.zeros(3, 2, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV),
              torch.zeros(3, 65, dtype=torch.int32, device=DEV), torch.zeros(3, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="exclude"):
            C.sample(x, *s, exclude=e)
    for o in (torch.zeros(3, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(6, dtype=torch.int64, device=DEV)[::2]):
        with pytest.raises(ValueError, match="out"):
            C.sample(x, *s, out=o)


@pytest.mark.parametrize("V", [900, 60000])
def test_settings_that_are_no_numbers(C, V):
    asks = [(1.0, 0, math.nan, 0.0), (1.0, 0, 1.0, math.nan), (0.7, 30, math.nan, math.nan), (math.nan, 0, 1.0, 0.0), (1.5, 0, 0.9, math.nan), (1.0, 0, math.nan, 0.1)]
    got = _same(C, _logits(60, V, V), _settings(asks, 60, V))
    filters_off = [(t, k, 1.0 if math.isnan(p) else p, 0.0 if math.isnan(m) else m) for t, k, p, m in asks]
    assert torch.equal(got, C.sample(_logits(60, V, V), *_settings(filters_off, 60, V)))


def test_pick_tokens_goes_to_the_device_of_the_logits(C, monkeypatch):
    """Logits of another device than the current one: the kernels run on theirs."""
    from b200serve.sched import sampling
    from b200serve.sched.request import Sampling

    entered = []

    class Device(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            super().__enter__()

    monkeypatch.setattr(torch.cuda, "device", Device)
    x = _logits(3, 5000, 1)
    assert sampling.pick_tokens(x, [Sampling()] * 3, [None] * 3, [None] * 3) == x.argmax(-1).tolist()
    assert entered == [x.device.index]


def test_pick_tokens_of_a_vocabulary_beyond_the_kernels(C):
    from b200serve.sched.request import Sampling
    from b200serve.sched.sampling import pick_tokens

    V = C.SAMPLE_VOCAB + 3
    x = _logits(3, V, 1)
    asks = [Sampling(), Sampling(temperature=0.7, top_k=20, top_p=0.9, seed=1), Sampling(temperature=1.0, seed=2)]

    def picks(x):
        return pick_tokens(x, asks, [None, *(torch.Generator().manual_seed(s) for s in (1, 2))], [{int(x[0].argmax())}, None, None])

    assert picks(x) == picks(x.cpu())
    with pytest.raises(ValueError, match="sample"):
        _same(C, x, _settings(ASKS, 3))
