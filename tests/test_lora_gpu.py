"""Projections with each row's own low-rank adapter, against the formula in 64 bits."""

import pytest
import torch

from b200serve.ops.lora import LoraWeights

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def C():
    from b200serve.ops import cuda_ops

    cuda_ops.lib()
    return cuda_ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bf(*shape, by=1.0, seed=0):
    return (torch.randn(*shape, device=DEV, generator=_gen(seed)) * by).bfloat16()


def _adapters(L, R, N, K, seed=0, by=0.25):
    scale = torch.rand(L, device=DEV, generator=_gen(seed + 2)) * 3 - 1
    return LoraWeights(_bf(L, R, K, by=K ** -0.5, seed=seed), _bf(L, N, R, by=by * R ** -0.5, seed=seed + 1), scale)


def _rows(T, L, seed=0, bare=0.2, run=1):
    """Adapters of the rows, ``run`` rows of one after the other, some of none."""
    g = torch.Generator().manual_seed(seed)
    n = -(-T // run)
    ids = torch.randint(0, L, (n,), generator=g)
    ids[torch.rand(n, generator=g) < bare] = -1
    return ids.repeat_interleave(run)[:T].int().to(DEV)


def _check(got, x, w, ad, rows, what=""):
    """Within what the roundings leave. A sum of K products is added up sixteen at a time: K / 16 additions to a running sum, which is at most the sum of
    the products' magnitudes, each cut to 24 bits: off by 2^-23 of that at most, so K / 16 * 2^-23 of the magnitudes in all (so is h's). h is
    rounded to bf16 (half a step: 2^-9 of each h, 2^-8 taken), or to three bf16 parts for fp32 outputs (2^-24 of it, 2^-23 taken); the result to bf16 by 2^-9 of itself
    (2^-8 taken), or to fp32 (2^-24, 2^-23 taken)."""
    acc = (x.shape[1] / 16 + 1) * 2.0 ** -23
    x64, w64 = x.double(), w.double()
    y, mag, off = x64 @ w64.t(), x64.abs() @ w64.abs().t(), torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    f32 = got.dtype == torch.float32
    for i in range(ad.a.shape[0]):
        at = (rows == i).nonzero().view(-1)
        if len(at):
            s, b = ad.scale[i].double(), ad.b[i].double()
            h, hm = x64[at] @ ad.a[i].double().t() * s, x64[at].abs() @ ad.a[i].double().abs().t() * s.abs()
            y[at] += h @ b.t()
            mag[at] += h.abs() @ b.abs().t()
            off[at] += (h.abs() * (2.0 ** -23 if f32 else 2.0 ** -8) + hm * acc) @ b.abs().t()
    tol = mag * (acc + ad.a.shape[1] / 16 * 2.0 ** -23) + off + y.abs() * (2.0 ** -23 if f32 else 2.0 ** -8) + 1e-30
    assert got.isfinite().all(), what
    worst = ((got.double() - y).abs() / tol).max().item()
    assert worst <= 1, f"{what}: off by {worst:.3g} times the tolerance"


SHAPES = [(9216, 2048), (2048, 4096), (12352, 2048), (1003, 520), (64, 64), (257, 2048), (100, 72), (4096, 320)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,K", SHAPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 100, 128, 129, 257, 700])
def test_shapes(C, T, N, K, dt):
    R, L = {0: 16, 1: 8, 2: 64, 3: 32}[(T + N) % 4], 1 + (T + K) % 9
    x, w, ad = _bf(T, K, seed=T), _bf(N, K, by=K ** -0.5, seed=N), _adapters(L, R, N, K, seed=T)
    for run in (1, 40):
        rows = _rows(T, L, T, run=run)
        _check(C.lora_linear(x, w, ad, rows, out_dtype=dt), x, w, ad, rows, f"{T} rows, runs of {run}")
    C.check_errors(x.device)


@pytest.mark.parametrize("R", [*range(8, 129, 8), 136, 192, 200, 256])
def test_ranks(C, R):
    N, K, L = 520, 256, 5
    w, ad = _bf(N, K, by=K ** -0.5, seed=1), _adapters(L, R, N, K, seed=R)
    for T in (3, 50, 300, 1000):
        x, rows = _bf(T, K, seed=T), _rows(T, L, T, run=1 + T // 100)
        for dt in (torch.bfloat16, torch.float32):
            _check(C.lora_linear(x, w, ad, rows, out_dtype=dt), x, w, ad, rows, f"rank {R}, {T} rows")


@pytest.mark.parametrize("L", [1, 33, 200, 1024])
def test_many_adapters(C, L):
    N, K, R = 384, 192, 16
    w, ad = _bf(N, K, by=K ** -0.5, seed=1), _adapters(L, R, N, K, seed=L)
    for T in (5, 128, 513, 2500):
        x, rows = _bf(T, K, seed=T), _rows(T, L, T)
        rows[0] = L - 1
        _check(C.lora_linear(x, w, ad, rows), x, w, ad, rows, f"{L} adapters, {T} rows")


@pytest.mark.parametrize("T", [1, 16, 40, 128, 200, 1531, 8192])
def test_packed_weights_and_the_bits_of_linear(C, T):
    for N, K in ((9216, 2048), (12352, 2048), (2048, 4096)):
        w, ad = _bf(N, K, by=K ** -0.5, seed=N), _adapters(6, 16, N, K, seed=T)
        packed = C.pack_weight(w.clone())
        x, rows = _bf(T, K, seed=T), _rows(T, 6, T, run=1 + T // 8)
        got = C.lora_linear(x, packed, ad, rows)
        assert got.shape == (T, packed.shape[0])
        assert torch.equal(got[:, :N], C.lora_linear(x, w, ad, rows))
        if T <= 1531:
            _check(got[:, :N], x, w, ad, rows, f"{T} x {N}")
        bare = rows < 0
        assert torch.equal(got[bare], C.linear(x, packed)[bare])
        none = torch.full_like(rows, -1)
        assert torch.equal(C.lora_linear(x, packed, ad, none), C.linear(x, packed))


def test_a_row_does_not_depend_on_the_batch(C):
    """One row alone, in a decode batch, in a prefill pass, among other adapters and in other places: the same bits."""
    for N, K, R in ((9216, 2048, 16), (2048, 4096, 64), (1003, 520, 24), (2048, 2048, 128)):
        w, ad = _bf(N, K, by=K ** -0.5, seed=N), _adapters(20, R, N, K, seed=3)
        for dt in (torch.bfloat16, torch.float32):
            x, rows = _bf(1500, K, seed=5), _rows(1500, 20, 6, run=3)
            whole = C.lora_linear(x, w, ad, rows, out_dtype=dt)
            for a, b in ((0, 1), (7, 8), (100, 117), (33, 161), (1000, 1300), (1, 1500)):
                assert torch.equal(C.lora_linear(x[a:b], w, ad, rows[a:b].clone(), out_dtype=dt), whole[a:b]), (N, a, b)
            for _ in range(3):
                assert torch.equal(C.lora_linear(x, w, ad, rows, out_dtype=dt), whole)


def test_rows_that_are_further_apart(C):
    N, K = 640, 512
    w, ad = _bf(N, K, by=K ** -0.5, seed=1), _adapters(4, 32, N, K)
    for T in (1, 30, 400):
        big = _bf(T, 2 * K + 64, seed=T)
        for x in (big[:, 8 : 8 + K], big[:, K:][:, :K]):
            rows = _rows(T, 4, T)
            got = C.lora_linear(x, w, ad, rows)
            _check(got, x, w, ad, rows)
            assert torch.equal(got, C.lora_linear(x.contiguous(), w, ad, rows))
    rows2 = _rows(800, 4, 9)[1:401]  # an odd word of its tensor
    x = _bf(400, K, seed=2)
    _check(C.lora_linear(x, w, ad, rows2), x, w, ad, rows2)


def test_numbers_of_one_row_stay_in_it(C):
    """A NaN, an infinity or an overflow in a row reaches no other row; an adapter's number out of range leaves its row bare and is reported."""
    N, K, L = 512, 256, 6
    w, ad = _bf(N, K, by=K ** -0.5, seed=1), _adapters(L, 16, N, K)
    for T in (20, 200, 1000):
        x, rows = _bf(T, K, seed=T), _rows(T, L, T, bare=0.0)
        want = C.lora_linear(x, w, ad, rows)
        y = x.clone()
        y[3, 5], y[11, 0], y[T - 1] = float("nan"), float("inf"), 3e38
        got = C.lora_linear(y, w, ad, rows)
        clean = torch.ones(T, dtype=torch.bool, device=DEV)
        clean[[3, 11, T - 1]] = False
        assert torch.equal(got[clean], want[clean])
        assert not got[3].isfinite().any()
        bad = rows.clone()
        bad[7] = L
        bad[9] = 1 << 30
        got = C.lora_linear(x, w, ad, bad)
        with pytest.raises(C.KernelError, match="out of range"):
            C.check_errors(x.device)
        clean = torch.ones(T, dtype=torch.bool, device=DEV)
        clean[[7, 9]] = False
        assert torch.equal(got[clean], want[clean])
        assert torch.equal(got[~clean], C.linear(x, w)[~clean])


def test_captured_and_replayed(C):
    N, K, L = 2048, 512, 9
    w, ad = _bf(N, K, by=K ** -0.5, seed=1), _adapters(L, 16, N, K)
    for T in (1, 48, 300):
        x, rows = _bf(T, K, seed=T), _rows(T, L, T)
        C.lora_linear(x, w, ad, rows)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = C.lora_linear(x, w, ad, rows)
                z = C.lora_linear(y[:, :K].contiguous(), w, ad, rows)
            graphs.append((g, y, z))
        for seed in (1, 2):
            x.copy_(_bf(T, K, seed=seed))
            rows.copy_(_rows(T, L, seed, bare=0.5))
            torch.cuda.synchronize()
            for g, _, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = C.lora_linear(x, w, ad, rows)
            again = C.lora_linear(want[:, :K].contiguous(), w, ad, rows)
            assert all(torch.equal(y, want) and torch.equal(z, again) for _, y, z in graphs)


def test_another_stream(C):
    N, K = 1024, 1024
    w, ad = _bf(N, K, by=K ** -0.5, seed=1), _adapters(4, 16, N, K)
    xs = [_bf(t, K, seed=t) for t in (3, 90, 500)]
    rows = [_rows(x.shape[0], 4, 1) for x in xs]
    want = [C.lora_linear(x, w, ad, r) for x, r in zip(xs, rows)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None] * len(xs)
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = C.lora_linear(xs[i], w, ad, rows[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows(C):
    ad = _adapters(2, 16, 128, 64)
    got = C.lora_linear(_bf(0, 64), _bf(128, 64), ad, torch.zeros(0, dtype=torch.int32, device=DEV))
    assert got.shape == (0, 128) and got.dtype == torch.bfloat16


def test_refusals(C):
    x, w, ad, rows = _bf(4, 64), _bf(128, 64), _adapters(3, 16, 128, 64), _rows(4, 3)
    a, b, s = ad
    wrong = [(x.float(), w, ad, rows), (x[:, :56], w, ad, rows), (x, w.float(), ad, rows), (x, w, ad, rows.long()), (x, w, ad, rows[:3]), (x, w, ad, rows.cpu()),
             (x, w, LoraWeights(a[:2], b, s), rows), (x, w, LoraWeights(a, b[:, :120], s), rows), (x, w, LoraWeights(a.float(), b.float(), s), rows),
             (x, w, LoraWeights(a[:, :12], b[..., :12], s), rows), (x, w, LoraWeights(a, b, s.double()), rows), (x, w, LoraWeights(a, b, s.cpu()), rows),
             (x, w, LoraWeights(a.repeat(1, 17, 1), b.repeat(1, 1, 17), s), rows), (x, w, LoraWeights(a, b.transpose(1, 2).contiguous().transpose(1, 2), s), rows),
             (x.cpu(), w, ad, rows), (_bf(4, 65)[:, 1:], w, ad, rows), (_bf(4, 128)[:, ::2], w, ad, rows), (x, w, ad, _rows(8, 3)[::2])]
    for args in wrong:
        with pytest.raises(ValueError, match="lora_linear"):
            C.lora_linear(*args)
    with pytest.raises(ValueError, match="outputs"):
        C.lora_linear(x, w, ad, rows, out_dtype=torch.float16)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [257, 513, 1531])
def test_a_call_cut_into_parts(C, monkeypatch, T, dt):
    """A call whose workspace would be too large goes out by parts of its rows, with the bits of the whole; captured as well."""
    L, R, cuts = 24, 40, []
    part = C._lora_part
    monkeypatch.setattr(C, "_lora_part", lambda *args: (cuts.append(args[5]), part(*args))[1])
    for N, K in ((1003, 520), (2048, 1024), (12352, 512)):
        w, ad = _bf(N, K, by=K ** -0.5, seed=N), _adapters(L, R, N, K, seed=T)
        x = _bf(T, K + 24, seed=T)[:, 8 : 8 + K]
        rows = _rows(T, L, T, run=2)
        for weights in (w, C.pack_weight(w.clone())) if K % 64 == 0 else (w,):
            monkeypatch.setattr(C, "LORA_WORK", 256 << 20)
            del cuts[:]
            whole = C.lora_linear(x, weights, ad, rows, out_dtype=dt)
            assert cuts == [T]
            monkeypatch.setattr(C, "LORA_WORK", 200 << 10)
            cut = C.lora_linear(x, weights, ad, rows, out_dtype=dt)
            ends = [n for n in cuts[1:] if n <= 256]  # (parts of up to 256 rows are not cut)
            assert len(ends) == -(-T // 256) and sum(ends) == T
            assert torch.equal(cut, whole)
            _check(cut[:, :N], x, w, ad, rows, f"{T} rows in parts")
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = C.lora_linear(x, weights, ad, rows, out_dtype=dt)
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, whole)
    C.check_errors(x.device)
