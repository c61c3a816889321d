"""The 8-bit KV cache's kernels against the formulas in 64 bits."""

import math

import pytest
import torch

from b200serve.ops.kv8 import E_BIAS, E_NAN, Kv8Layer, dequantise, quantise

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def C():
    from b200serve.ops import cuda_ops

    cuda_ops.lib()
    return cuda_ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _layer(pages, n_kv, D, seed=0, spread=1.0):
    """Rows with powers of two from far apart, as keys and values of different tokens may have."""
    g = _gen(seed)
    x = torch.randn(pages, 2, n_kv, 64, D, device=DEV, generator=g)
    x *= torch.exp2(torch.randn(pages, 2, n_kv, 64, 1, device=DEV, generator=g) * spread)
    return Kv8Layer(*quantise(x))


def _tables(lens, width, pages, seed=0):
    """Page tables of sequences of ``lens`` keys, no page twice; entries behind a sequence's own are far out of range."""
    g = torch.Generator().manual_seed(seed)
    ids = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    t = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range((n + 63) // 64):
            t[i, j] = ids.pop()
    return t.to(DEV)


def _attention(q, gate, layer, tables, positions):
    """The formula in 64 bits, and what an output may be off by.

    Outputs are rounded to bf16 (2^-9 of the output, 2^-8 taken). A weight is rounded to half precision (2^-11 of its part). A score is off by
    what the query's form loses, at most 2^-18 of its largest number per dim, and by fp32 sums over D products (2^-20 of their magnitudes):
    weights and their sum are off by twice that relative part of sum p |v|."""
    T, n_q, D = q.shape
    n_kv = layer.data.shape[2]
    out = torch.zeros(T, n_q, D, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    sig = torch.sigmoid(gate.double()).view(T, n_q, D)
    for t in range(T):
        n = int(positions[t]) + 1
        if n <= 0:
            continue
        pages = tables[t, : (n + 63) // 64].long()
        kv = dequantise(layer.data.view(torch.uint8)[pages].view(torch.float8_e4m3fn), layer.exps[pages], torch.float32).double()
        k, v = (kv[:, i].transpose(0, 1).reshape(n_kv, -1, D)[:, :n] for i in (0, 1))
        qt = q[t].double().view(n_kv, n_q // n_kv, D)
        p = torch.softmax(qt @ k.transpose(1, 2) / math.sqrt(D), -1)
        o, mag = (p @ v).view(n_q, D), (p @ v.abs()).view(n_q, D)
        off = (qt.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None] * 2.0 ** -18
               + qt.abs() @ k.abs().transpose(1, 2) * 2.0 ** -20).amax(-1) / math.sqrt(D)
        out[t] = o * sig[t]
        tol[t] = 2.0 ** -8 * out[t].abs() + mag * sig[t] * (2.0 ** -10 + 2 * off.view(n_q, 1))
    return out.view(T, -1), tol.view(T, -1)


def _check(got, want, what=""):
    out, tol = want
    assert got.isfinite().all(), what
    over = ((got.double() - out).abs() - tol - 1e-30) / tol.clamp(min=1e-30)
    assert over.max() <= 0, f"{what}: off by {over.max().item() + 1:.3g} times the tolerance"


def _rows(T, n_q, D, seed, scale=1.2):
    g = _gen(seed)
    return ((torch.randn(T, n_q, D, device=DEV, generator=g) * scale).bfloat16(),
            torch.randn(T, n_q * D, device=DEV, generator=g).bfloat16())


HEADS = [(16, 2, 256), (8, 1, 64), (4, 1, 128), (8, 8, 64), (6, 3, 128), (3, 1, 256), (16, 1, 64), (10, 2, 64)]


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("n_kv,D", [(2, 256), (1, 32), (3, 64), (2, 128)])
@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("form", ["packed", "slices", "odd", "heads_first", "strided"])
def test_write_is_the_quantiser(C, n_kv, D, T, form):
    g = _gen(T + D)
    width = 2 * n_kv * D + (3 if form == "odd" else 0)
    if form == "packed":
        k, v = (torch.randn(T, n_kv, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    elif form == "heads_first":
        k, v = (torch.randn(n_kv, T, D, device=DEV, generator=g).bfloat16().transpose(0, 1) for _ in range(2))
    elif form == "strided":
        k, v = (torch.randn(T, n_kv, D, 2, device=DEV, generator=g).bfloat16()[..., 1] for _ in range(2))
    else:  # slices of a projection's rows, at an odd element where `odd`
        a = torch.randn(T, width, device=DEV, generator=g).bfloat16()
        o = width - 2 * n_kv * D
        k, v = a[:, o : o + n_kv * D].view(T, n_kv, D) if o == 0 else a[:, o : o + n_kv * D].unflatten(1, (n_kv, D)), \
            a[:, o + n_kv * D :].unflatten(1, (n_kv, D))
    layer = _layer(40, n_kv, D, seed=1)
    lens = [T // 3 + 60, T - T // 3 + 130]
    tables = _tables(lens, 9, 40)
    seq = (torch.arange(T, device=DEV) >= T // 3).int()
    pos = torch.where(seq == 0, torch.arange(T, device=DEV) + 60, torch.arange(T, device=DEV) - T // 3 + 130).long()
    want = Kv8Layer(layer.data.clone(), layer.exps.clone())
    page, at = tables[seq.long(), pos // 64].long(), pos % 64
    for i, x in enumerate((k, v)):
        data, exps = quantise(x)
        want.data.view(torch.uint8)[page, i, :, at] = data.view(torch.uint8)
        want.exps[page, i, :, at] = exps
    C.kv8_write(layer, k, v, pos, seq, tables)
    C.check_errors(k.device)
    assert torch.equal(layer.data.view(torch.uint8), want.data.view(torch.uint8)) and torch.equal(layer.exps, want.exps)
    rk, rv = C.kv8_read(layer, pos, seq, tables)
    for got, x in ((rk, k), (rv, v)):
        assert torch.equal(got, dequantise(*quantise(x), torch.bfloat16))


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_write_of_far_numbers_nan_and_infinity(C, D):
    g = _gen(D)
    T = 64
    x = torch.randn(T, 1, D, device=DEV, generator=g) * torch.exp2(torch.linspace(-130, 127, T, device=DEV))[:, None, None]
    x[3], x[4, 0, 5], x[5, 0, D - 1], x[6, 0, 0] = 0.0, float("nan"), float("inf"), -float("inf")
    x[7, 0, 1], x[7, 0, 2] = float("nan"), float("inf")
    k, v = x.bfloat16(), x.flip(0).bfloat16()
    layer = _layer(3, 1, D)
    pos, seq, tables = torch.arange(T, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV), torch.tensor([[2]], dtype=torch.int32, device=DEV)
    C.kv8_write(layer, k, v, pos, seq, tables)
    C.check_errors(x.device)
    for i, y in enumerate((k, v)):
        data, exps = quantise(y)
        assert torch.equal(layer.data.view(torch.uint8)[2, i], data.view(torch.uint8).transpose(0, 1))
        assert torch.equal(layer.exps[2, i], exps.transpose(0, 1))
    assert layer.exps[2, 0, 0, 4] == E_NAN and layer.exps[2, 0, 0, 7] == E_NAN
    rk, _ = C.kv8_read(layer, pos, seq, tables)
    assert rk[4].isnan().all() and rk[5, 0, D - 1] == 448 * 2.0 ** 60


def test_pages_behind_two_to_the_31_bytes(C):
    """A cache of more than 2^32 bytes of data: its last pages are written, read and attended to."""
    n_q, n_kv, D = 16, 2, 256
    pages = (1 << 32) // (2 * n_kv * 64 * D) + 40
    layer = Kv8Layer(torch.zeros(pages, 2, n_kv, 64, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
                     torch.full((pages, 2, n_kv, 64), E_BIAS, dtype=torch.uint8, device=DEV))
    n = 700
    tables = torch.tensor([[pages - 1 - i for i in range((n + 63) // 64)]], dtype=torch.int32, device=DEV)
    g = _gen(1)
    k, v = (torch.randn(n, n_kv, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    pos, seq = torch.arange(n, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    C.kv8_write(layer, k, v, pos, seq, tables)
    rk, rv = C.kv8_read(layer, pos, seq, tables)
    assert torch.equal(rk, dequantise(*quantise(k), torch.bfloat16)) and torch.equal(rv, dequantise(*quantise(v), torch.bfloat16))
    q, gate = _rows(1, n_q, D, 2)
    _check(C.kv8_decode(q, gate, layer, tables, pos[-1:], 1), _attention(q, gate, layer, tables, pos[-1:]))
    q, gate = _rows(40, n_q, D, 2)
    _check(C.kv8_prefill(q, gate, layer, tables, [0, 40], [n - 40]), _attention(q, gate, layer, tables.expand(40, -1), pos[-40:]))
    C.check_errors(q.device)


# ------------------------------------------------------------------ decode
@pytest.mark.parametrize("n_q,n_kv,D", HEADS)
@pytest.mark.parametrize("lens,G", [([1], 1), ([1, 16, 17, 63, 64, 65], 1), ([511, 512, 513, 100], 1), ([2000, 5], 1),
                                    ([3, 514, 65], 2), ([4, 513, 1026], 4), ([700, 8], 7)])
def test_decode(C, n_q, n_kv, D, lens, G):
    width = max(lens) // 64 + 3
    pages = sum((n + 63) // 64 for n in lens) + 2
    layer = _layer(pages, n_kv, D, seed=D + G)
    tables = _tables(lens, width, pages)
    positions = torch.tensor([n - G + i for n in lens for i in range(G)], device=DEV)
    q, gate = _rows(len(lens) * G, n_q, D, 3)
    got = C.kv8_decode(q, gate, layer, tables, positions, G)
    C.check_errors(q.device)
    _check(got, _attention(q, gate, layer, tables.repeat_interleave(G, 0), positions))


@pytest.mark.parametrize("n_q,n_kv,D", [(16, 2, 256), (8, 1, 64), (6, 3, 128), (16, 1, 128)])
def test_decode_rows_have_the_same_bits_in_any_batch_and_pass(C, n_q, n_kv, D):
    lens = [1, 513, 1030, 64, 700, 2, 1537, 512, 90]
    pages = sum((n + 63) // 64 for n in lens) + 2
    layer = _layer(pages, n_kv, D, seed=5)
    tables = _tables(lens, 40, pages)
    G = 4
    positions = torch.tensor([n - 1 - (G - 1) + i for n in lens for i in range(G)], device=DEV)  # negative for the shortest: rows without keys
    q, gate = _rows(len(lens) * G, n_q, D, 6)
    verify = C.kv8_decode(q, gate, layer, tables, positions, G)
    rows = tables.repeat_interleave(G, 0)
    plain = C.kv8_decode(q, gate, layer, rows, positions, 1)
    assert torch.equal(verify, plain)
    pairs = C.kv8_decode(q, gate, layer, tables.repeat_interleave(2, 0), positions, 2)
    assert torch.equal(pairs, plain)
    for r in range(len(lens) * G):
        w = max(1, int(positions[r]) // 64 + 1)
        one = C.kv8_decode(q[r : r + 1], gate[r : r + 1], layer, rows[r : r + 1, :w].contiguous(), positions[r : r + 1], 1)
        assert torch.equal(one, plain[r : r + 1]), r
        if positions[r] < 0:
            assert (one == 0).all()
    C.check_errors(q.device)


def test_decode_of_more_sequences_than_one_launch_takes(C):
    n_q, n_kv, D, B = 8, 8, 64, 1500
    lens = [1 + (i * 37) % 90 for i in range(B)]
    pages = 2 * B + 2
    layer = _layer(pages, n_kv, D)
    tables = _tables(lens, 2, pages)
    positions = torch.tensor(lens, device=DEV) - 1
    q, gate = _rows(B, n_q, D, 1)
    _check(C.kv8_decode(q, gate, layer, tables, positions, 1), _attention(q, gate, layer, tables, positions))
    C.check_errors(q.device)


def test_decode_of_a_long_context(C):
    n_q, n_kv, D = 16, 2, 256
    lens = [131072, 70001]
    pages = sum((n + 63) // 64 for n in lens) + 2
    layer = _layer(pages, n_kv, D)
    tables = _tables(lens, 2100, pages)
    positions = torch.tensor(lens, device=DEV) - 1
    q, gate = _rows(2, n_q, D, 1, scale=0.7)
    _check(C.kv8_decode(q, gate, layer, tables, positions, 1), _attention(q, gate, layer, tables, positions))
    C.check_errors(q.device)


def _run(C, kind, q, gate, layer, tables, pos0, n):
    """The last ``n`` rows of one sequence by either operator."""
    if kind == "decode":
        return C.kv8_decode(q, gate, layer, tables, torch.arange(pos0, pos0 + n, device=DEV), n)
    return C.kv8_prefill(q, gate, layer, tables, [0, n], [pos0])


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_masked_keys_may_hold_anything(C, kind, D):
    """Behind the last row's key: rows marked as NaN, the largest numbers, the largest exponents."""
    n_q, n_kv, n, total = 8, 1, 5, 600
    layer = _layer(12, n_kv, D)
    tables = _tables([640], 10, 12)
    want_layer = Kv8Layer(layer.data.clone(), layer.exps.clone())
    flat_d, flat_e = layer.data.view(torch.uint8), layer.exps
    for j in range(total, 640):
        page = int(tables[0, j // 64])
        flat_d[page, :, :, j % 64], flat_e[page, :, :, j % 64] = 0x7E, (E_NAN, E_BIAS + 60, 0)[j % 3]
    q, gate = _rows(n, n_q, D, 4)
    pos = torch.arange(total - n, total, device=DEV)
    got = _run(C, kind, q, gate, layer, tables, total - n, n)
    C.check_errors(q.device)
    _check(got, _attention(q, gate, want_layer, tables.expand(n, -1), pos))


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("first", [False, True])
def test_a_nan_row_reaches_those_who_see_it_and_nobody_else(C, kind, which, first):
    n_q, n_kv, D, n, total = 16, 2, 256, 8, 70
    layer = _layer(4, n_kv, D)
    tables = _tables([total], 2, 4)
    at = 0 if first else total - 4  # four rows before it, or none
    page = int(tables[0, at // 64])
    layer.data.view(torch.uint8)[page, which, 1, at % 64] = 0
    layer.exps[page, which, 1, at % 64] = E_NAN
    q, gate = _rows(n, n_q, D, 4)
    got = _run(C, kind, q, gate, layer, tables, total - n, n).view(n, n_q, D)
    C.check_errors(q.device)
    sees = torch.arange(total - n, total, device=DEV) >= at
    assert got[sees][:, 8:].isnan().all()
    assert got[~sees].isfinite().all() and got[:, :8].isfinite().all()


@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_queries_of_zeros_far_numbers_nan_and_infinity(C, kind):
    n_q, n_kv, D, total = 16, 2, 256, 300
    layer = _layer(8, n_kv, D)
    tables = _tables([total], 5, 8)
    q, gate = _rows(6, n_q, D, 4)
    q[0] = 0
    q[1] *= 2.0 ** -100
    q[2, :, 0] = 2.0 ** 9   # one strong dim
    q[4, 3, 7], q[5, 9, 200] = float("nan"), float("inf")
    got = _run(C, kind, q, gate, layer, tables, total - 6, 6).view(6, n_q, D)
    C.check_errors(q.device)
    bad = torch.zeros(6, n_q, dtype=torch.bool, device=DEV)
    bad[4, 3] = bad[5, 9] = True
    assert got[bad].isnan().all()
    q2 = q.clone()
    q2[bad] = 0
    out, tol = _attention(q2, gate, layer, tables.expand(6, -1), torch.arange(total - 6, total, device=DEV))
    keep = ~bad
    _check(got[keep], (out.view(6, n_q, D)[keep], tol.view(6, n_q, D)[keep]))


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("D", [64, 256])
def test_many_small_weights_beside_a_large_one(C, kind, D):
    """A key that takes most of the weight (an attention sink) and thousands that share the rest, on values of powers of two far
    apart: what the thousands add is there. Of their weights, 2^-18 of the sink's and less, nothing may be lost."""
    n_q, n_kv, total = 8, 1, 8192
    q = torch.zeros(4, n_q, D, device=DEV)
    q[:, :, 0] = 1.0
    k = torch.zeros(total, n_kv, D, device=DEV)
    k[0, :, 0] = 14.0 * D ** 0.5  # e^14 is 1.2e6 of the others
    v = torch.zeros(total, n_kv, D, device=DEV)
    v[0], v[1:], v[1::3] = 2.0 ** -20, 1.0, 2.0 ** 6
    layer = Kv8Layer(torch.zeros(140, 2, n_kv, 64, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
                     torch.full((140, 2, n_kv, 64), E_BIAS, dtype=torch.uint8, device=DEV))
    tables = _tables([total], 128, 140)
    pos = torch.arange(total, device=DEV)
    C.kv8_write(layer, k.bfloat16(), v.bfloat16(), pos, torch.zeros(total, dtype=torch.int32, device=DEV), tables)
    gate = torch.zeros(4, n_q * D, device=DEV).bfloat16()
    got = _run(C, kind, q.bfloat16(), gate, layer, tables, total - 4, 4)
    C.check_errors(q.device)
    _check(got, _attention(q.bfloat16(), gate, layer, tables.expand(4, -1), pos[-4:]))


# ------------------------------------------------------------------ prefill
@pytest.mark.parametrize("n_q,n_kv,D", HEADS)
@pytest.mark.parametrize("lens,pos0", [([1], [0]), ([1, 16, 17, 64, 65], [0, 0, 3, 60, 64]), ([130, 40], [0, 700]), ([33], [1500]),
                                       ([3, 0, 5], [64, 9, 63]), ([200], [129])])
def test_prefill(C, n_q, n_kv, D, lens, pos0):
    total = [a + b for a, b in zip(lens, pos0)]
    pages = sum((n + 63) // 64 for n in total) + 2
    layer = _layer(pages, n_kv, D, seed=D)
    tables = _tables(total, max(total) // 64 + 2, pages)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    q, gate = _rows(starts[-1], n_q, D, 9)
    got = C.kv8_prefill(q, gate, layer, tables, starts, pos0)
    C.check_errors(q.device)
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).to(DEV)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(lens, pos0)]).to(DEV)
    _check(got, _attention(q, gate, layer, tables[seq], pos))
    meta = tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (starts, pos0))
    assert torch.equal(C.kv8_prefill(q, gate, layer, tables, starts, pos0, meta=meta), got)


def test_prefill_rows_have_the_same_bits_beside_other_spans(C):
    n_q, n_kv, D = 16, 2, 256
    lens, pos0 = [70, 5, 300, 1, 64], [0, 1200, 64, 2500, 700]
    total = [a + b for a, b in zip(lens, pos0)]
    pages = sum((n + 63) // 64 for n in total) + 2
    layer = _layer(pages, n_kv, D)
    tables = _tables(total, 41, pages)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    q, gate = _rows(starts[-1], n_q, D, 9)
    together = C.kv8_prefill(q, gate, layer, tables, starts, pos0)
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        alone = C.kv8_prefill(q[a:b], gate[a:b], layer, tables[i : i + 1], [0, b - a], [pos0[i]])
        assert torch.equal(alone, together[a:b]), i
    C.check_errors(q.device)


def test_prefill_of_a_full_pass(C):
    """As many tiles as the GPU holds at a time and more, and maxima that grow page by page: outputs are rescaled while products are under way."""
    n_q, n_kv, D, spans, n = 16, 2, 256, 8, 1024
    layer = _layer(spans * n // 64, n_kv, D)
    tables = torch.arange(spans * n // 64, device=DEV, dtype=torch.int32).view(spans, -1)
    q, gate = _rows(spans * n, n_q, D, 9, scale=6.0)
    starts = [i * n for i in range(spans + 1)]
    got = C.kv8_prefill(q, gate, layer, tables, starts, [0] * spans)
    for _ in range(4):
        assert torch.equal(C.kv8_prefill(q, gate, layer, tables, starts, [0] * spans), got)
    for i in range(spans):  # every other one of the rows in the last eight tiles
        rows = torch.arange(i * n + n - 128, i * n + n, 2, device=DEV)
        _check(got[rows], _attention(q[rows], gate[rows], layer, tables[i].expand(len(rows), -1), rows - i * n), i)
    C.check_errors(q.device)


@pytest.mark.parametrize("n", [300, 1500])  # a run of keys, several
def test_gates_of_all_sizes(C, n):
    """Far below and above where a sigmoid is 0 and 1 in bf16, infinite and NaN: a number's gate is its own alone."""
    n_q, n_kv, D = 16, 2, 128
    layer = _layer(n // 64 + 3, n_kv, D)
    tables = _tables([n], n // 64 + 1, n // 64 + 3)
    q, gate = _rows(80, n_q, D, 4)
    odd = torch.tensor([float("nan"), float("inf"), float("-inf"), -1000.0, -100.0, -60.0, -44.0, 60.0, 1000.0], device=DEV).bfloat16()
    at = torch.arange(0, gate.numel(), 3, device=DEV)
    gate.view(-1)[at] = odd[torch.arange(len(at), device=DEV) % len(odd)]
    pos = torch.arange(n - 80, n, device=DEV)
    sig = torch.sigmoid(gate.double())
    clean = gate.clone()
    clean.view(-1)[at] = 0
    out, tol = _attention(q, clean, layer, tables.expand(80, -1), pos)
    of_one = 1 / torch.sigmoid(clean.double())
    want, tol = out * of_one * sig, tol * of_one * sig + 1e-30  # an output below a bf16 number's least is one there
    for got in (C.kv8_prefill(q, gate, layer, tables, [0, 80], [n - 80]), C.kv8_decode(q, gate, layer, tables, pos, 80)):
        assert torch.equal(got.isnan(), gate.isnan())
        ok = ~gate.isnan()
        assert ((got.double() - want).abs() <= tol)[ok].all()


# ------------------------------------------------------------------ how they are called
@pytest.mark.parametrize("kind", ["decode", "prefill"])
def test_another_stream_views_and_index_types(C, kind):
    n_q, n_kv, D, n, total = 16, 2, 256, 4, 900
    layer = _layer(20, n_kv, D)
    wide = torch.full((1, 64), 1 << 30, dtype=torch.int64, device=DEV)
    wide[:, ::2][:, :15] = _tables([total], 15, 20).long()
    tables = wide[:, ::2]  # int64, every second entry
    base = torch.randn(n, 2, n_q * D + 1, device=DEV, generator=_gen(2)).bfloat16()
    q, gate = base[:, 0, 1:].unflatten(1, (n_q, D)), base[:, 1, 1:]
    want = _attention(q, gate, layer, tables[:, :15].expand(n, -1), torch.arange(total - n, total, device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(C, kind, q, gate, layer, tables, total - n, n)
        if kind == "decode":
            got32 = C.kv8_decode(q, gate, layer, tables, torch.arange(total - n, total, device=DEV, dtype=torch.int32), n)
            assert torch.equal(got, got32)
    side.synchronize()
    C.check_errors(q.device)
    _check(got, want)


def test_calls_are_capturable_and_read_their_inputs_at_each_replay(C):
    n_q, n_kv, D, B = 16, 2, 256, 3
    layer = _layer(80, n_kv, D)
    tables = _tables([1300] * B, 24, 80)
    positions = torch.tensor([10, 600, 1200], device=DEV)
    seq = torch.arange(B, dtype=torch.int32, device=DEV)
    q, gate = _rows(B, n_q, D, 1)
    k, v = (torch.randn(B, n_kv, D, device=DEV, generator=_gen(5)).bfloat16() for _ in range(2))
    C.kv8_write(layer, k, v, positions, seq, tables)
    C.kv8_decode(q, gate, layer, tables, positions, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C.kv8_write(layer, k, v, positions, seq, tables)
        out = C.kv8_decode(q, gate, layer, tables, positions, 1)
    for step in range(3):
        q.copy_(_rows(B, n_q, D, 10 + step)[0])
        k.copy_(torch.randn(B, n_kv, D, device=DEV, generator=_gen(20 + step)))
        positions += 37
        graph.replay()
        C.check_errors(q.device)
        rk, _ = C.kv8_read(layer, positions, seq, tables)
        assert torch.equal(rk, dequantise(*quantise(k), torch.bfloat16))
        _check(out, _attention(q, gate, layer, tables, positions), f"replay {step}")


def test_a_page_out_of_range_is_reported_and_nothing_is_touched(C):
    n_q, n_kv, D = 16, 2, 256
    layer = _layer(6, n_kv, D)
    before = layer.data.clone().view(torch.uint8), layer.exps.clone()
    k = v = torch.ones(1, n_kv, D, device=DEV).bfloat16()
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    for table, pos in ((6, 0), (-1, 0), (1, 64), (1, -1)):
        tables = torch.tensor([[table]], dtype=torch.int32, device=DEV)
        C.kv8_write(layer, k, v, torch.tensor([pos], device=DEV), zero, tables)
        with pytest.raises(C.KernelError):
            C.check_errors(k.device)
        rk, rv = C.kv8_read(layer, torch.tensor([pos], device=DEV), zero, tables)
        with pytest.raises(C.KernelError):
            C.check_errors(k.device)
        assert (rk == 0).all() and (rv == 0).all()
    assert torch.equal(layer.data.view(torch.uint8), before[0]) and torch.equal(layer.exps, before[1])
    q, gate = _rows(1, n_q, D, 1)
    for call in (lambda t: C.kv8_decode(q, gate, layer, t, torch.tensor([70], device=DEV), 1),
                 lambda t: C.kv8_prefill(q, gate, layer, t, [0, 1], [70])):
        call(torch.tensor([[2, 77]], dtype=torch.int32, device=DEV))
        with pytest.raises(C.KernelError):
            C.check_errors(k.device)


def test_arguments_that_do_not_fit_are_refused(C):
    n_q, n_kv, D = 16, 2, 256
    layer = _layer(6, n_kv, D)
    q, gate = _rows(4, n_q, D, 1)
    tables = _tables([64] * 4, 1, 6)
    pos, seq = torch.arange(4, device=DEV), torch.arange(4, dtype=torch.int32, device=DEV)
    k = torch.zeros(4, n_kv, D, device=DEV).bfloat16()
    bad_layer = Kv8Layer(layer.data, layer.exps.int())
    calls = [
        lambda: C.kv8_write(bad_layer, k, k, pos, seq, tables),
        lambda: C.kv8_write(layer, k.float(), k, pos, seq, tables),
        lambda: C.kv8_write(layer, k[:, :1], k, pos, seq, tables),
        lambda: C.kv8_write(layer, k, k, pos[:3], seq, tables),
        lambda: C.kv8_write(layer, k, k, pos, seq, tables[0]),
        lambda: C.kv8_write(layer, k.cpu(), k, pos, seq, tables),
        lambda: C.kv8_read(bad_layer, pos, seq, tables),
        lambda: C.kv8_read(layer, pos, seq[:2], tables),
        lambda: C.kv8_read(layer, pos, seq, tables.cpu()),
        lambda: C.kv8_decode(q, gate, bad_layer, tables, pos, 1),
        lambda: C.kv8_decode(q.float(), gate, layer, tables, pos, 1),
        lambda: C.kv8_decode(q[..., :128], gate, layer, tables, pos, 1),
        lambda: C.kv8_decode(q[:, :15], gate, layer, tables, pos, 1),
        lambda: C.kv8_decode(q, gate[:, 1:], layer, tables, pos, 1),
        lambda: C.kv8_decode(q, gate, layer, tables, pos, 3),
        lambda: C.kv8_decode(q, gate, layer, tables[:3], pos, 1),
        lambda: C.kv8_decode(q, gate, layer, tables, pos[:2], 1),
        lambda: C.kv8_decode(q.cpu(), gate, layer, tables, pos, 1),
        lambda: C.kv8_prefill(q, gate, bad_layer, tables, [0, 4], [0]),
        lambda: C.kv8_prefill(q.half(), gate, layer, tables, [0, 4], [0]),
        lambda: C.kv8_prefill(q, gate, layer, tables, [0, 3], [0]),
        lambda: C.kv8_prefill(q, gate, layer, tables, [0, 2, 4], [0]),
        lambda: C.kv8_prefill(q, gate, layer, tables[:1], [0, 2, 4], [0, 0]),
        lambda: C.kv8_prefill(q, gate, layer, tables, [0, 3, 2, 4], [0, 0, 0]),
    ]
    small = _layer(6, n_kv, 32)
    calls.append(lambda: C.kv8_decode(q[..., :32].contiguous(), gate[:, : n_q * 32], small, tables, pos, 1))
    calls.append(lambda: C.kv8_prefill(q[..., :32].contiguous(), gate[:, : n_q * 32], small, tables, [0, 4], [0]))
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="kv8_"):
            call()
            pytest.fail(f"call {i} was taken")
    none = torch.zeros(0, n_kv, D, device=DEV).bfloat16()
    C.kv8_write(layer, none, none, pos[:0], seq[:0], tables)
    assert C.kv8_read(layer, pos[:0], seq[:0], tables)[0].shape == (0, n_kv, D)
    assert C.kv8_decode(q[:0], gate[:0], layer, tables, pos[:0], 1).shape == (0, n_q * D)
    assert C.kv8_prefill(q[:0], gate[:0], layer, tables, [0, 0], [0]).shape == (0, n_q * D)
    C.check_errors(q.device)


# ------------------------------------------------------------------ in the model and the engine
@pytest.mark.parametrize("n_q,n_kv,D,G", [(16, 2, 256, 1), (16, 2, 256, 4), (4, 1, 64, 2), (16, 2, 256, 0), (6, 3, 128, 0), (4, 1, 32, 1), (4, 1, 32, 0)])
def test_attention_writes_what_the_quantiser_makes_of_the_bf16_rows(C, n_q, n_kv, D, G):
    """The block over the 8-bit pool against the block over the bf16 pool: the same rows, quantised; and its output against the formula."""
    from b200serve.ops import torch_ops as O

    B, rot = 3, D // 4
    per = [G] * B if G else [70, 1, 130]
    pos0 = [5, 64, 300]
    starts = [0]
    for n in per:
        starts.append(starts[-1] + n)
    T = starts[-1]
    g = _gen(D + G)
    layer = _layer(30, n_kv, D, seed=2)
    kv = torch.zeros(30, 2, n_kv, 64, D, dtype=torch.bfloat16, device=DEV)
    tables = _tables([a + b for a, b in zip(per, pos0)], 8, 30)
    tables[tables > 29] = 0  # the fallback for other head dims gathers whole tables
    qkv = torch.randn(T, n_q * 2 * D + 2 * n_kv * D, device=DEV, generator=g).bfloat16()
    positions = torch.cat([torch.arange(p, p + n) for p, n in zip(pos0, per)]).to(DEV)
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(per)]).int().to(DEV)
    qn, kn = ((torch.randn(D, device=DEV, generator=g) * 0.1).bfloat16() for _ in range(2))
    args = (qn, kn, n_q, n_kv, D, rot, 1e7, 1e-6, G, starts, pos0)
    before = Kv8Layer(layer.data.clone(), layer.exps.clone())
    got = C.attention(qkv, positions, seq, tables, layer, *args)
    C.check_errors(qkv.device)
    if D != 32:
        C.attention(qkv, positions, seq, tables, kv, *args)
        page, at = tables[seq.long(), positions // 64].long(), positions % 64
        for i in (0, 1):
            data, exps = quantise(kv[page, i, :, at])
            before.data.view(torch.uint8)[page, i, :, at] = data.view(torch.uint8)
            before.exps[page, i, :, at] = exps
        assert torch.equal(layer.data.view(torch.uint8), before.data.view(torch.uint8)) and torch.equal(layer.exps, before.exps)
    q, gate, _, _ = O.attn_prep(qkv.float(), positions, qn.float(), kn.float(), n_q, n_kv, D, rot, 1e7, 1e-6)
    want, tol = _attention(q, gate, layer, tables[seq.long()], positions)
    # beyond what the operators may be off by: q, rounded to bf16 where the reference's is not (its norm in fp32 and its rotation: 3 roundings of
    # 2^-9 each in a score of up to a few times sqrt D), moves weights by 2^-7 of their parts
    kv32 = dequantise(layer.data, layer.exps, torch.float32)
    assert ((got.double() - want).abs() <= tol + 0.05 * kv32.abs().max()).all()
    assert torch.nn.functional.cosine_similarity(got.double(), want, dim=-1).min() > 0.999


def test_captured_prefill_takes_device_tables_alone(C):
    n_q, n_kv, D = 16, 2, 256
    layer = _layer(30, n_kv, D)
    lens, pos0 = [40, 0, 70], [100, 0, 200]
    tables = _tables([a + b for a, b in zip(lens, pos0)], 8, 30)
    starts = [0, 40, 40, 110]
    q, gate = _rows(110, n_q, D, 1)
    meta = tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (starts, pos0))
    graph = torch.cuda.CUDAGraph()
    C.kv8_prefill(q, gate, layer, tables, None, None, meta=meta)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = C.kv8_prefill(q, gate, layer, tables, None, None, meta=meta)
    graph.replay()
    C.check_errors(q.device)
    seq = torch.tensor([0] * 40 + [2] * 70, device=DEV)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(lens, pos0)]).to(DEV)
    _check(out, _attention(q, gate, layer, tables[seq], pos))
    meta[1].copy_(torch.tensor([20, 0, 150], dtype=torch.int32))  # other positions in the same tables
    graph.replay()
    C.check_errors(q.device)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(lens, [20, 0, 150])]).to(DEV)
    _check(out, _attention(q, gate, layer, tables[seq], pos))
    with pytest.raises(ValueError, match="kv8_prefill"):
        C.kv8_prefill(q, gate, layer, tables, None, None)


def test_engine_with_the_8_bit_pool(C):
    """Greedy tokens are the same alone, in a batch, with and without graphs, and with draft chains verified."""
    from b200serve.config import EngineConfig, ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.ops.kv8 import Kv8Pool
    from b200serve.sched.engine import Engine
    from b200serve.sched.request import Sampling

    cfg = ModelConfig.tiny(head_dim=64, num_attention_heads=4, num_key_value_heads=1)
    w = random_weights(cfg, seed=0, device=DEV, dtype=torch.bfloat16, std=0.05, lm_head_std=0.5)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(3, 1024, (int(n),), generator=g).tolist() for n in (17, 190, 64, 600, 130)]
    s = Sampling(max_tokens=24, ignore_eos=True)

    def run(prompts, **kw):
        ecfg = EngineConfig(max_model_len=1024, prefill_chunk_tokens=64, max_seqs=8, kv_pages=256, decode_buckets=(1, 4, 8), kv_dtype="e4m3", **kw)
        eng = Engine(w, ecfg)
        return eng, [x.output for x in eng.generate(prompts, s)]

    eng, batched = run(prompts, mtp=False)
    assert isinstance(eng.model.kv, Kv8Pool) and eng._graphs is not None and not eng._graphs.errors
    for p, want in zip(prompts[:3], batched):
        assert run([p], mtp=False)[1] == [want]
    assert run(prompts, mtp=False, cuda_graphs=False)[1] == batched
    spec, out = run(prompts, mtp=True, spec_k=2)
    assert out == batched and spec.stats["mtp_verify_steps"] > 0
    graphs, out = run(prompts[:1], mtp=False, prefill_graphs=True)
    assert out == batched[:1]
    C.check_errors(torch.device(DEV))
