"""The 8-bit KV cache's format and its PyTorch operators, against definitions in 64 bits, on the CPU."""

import math

import pytest
import torch

from b200serve.ops import torch_ops as O
from b200serve.ops.kv8 import E_BIAS, E_MAX, E_NAN, HEAD_DIMS, Kv8Layer, Kv8Pool, check_layer, dequantise, quantise


def _e4m3_values():
    bits = torch.arange(256, dtype=torch.uint8)
    x = bits.view(torch.float8_e4m3fn).double()
    return x[x.isfinite()].unique()


def _nearest(y: float, values) -> float:
    """The nearest e4m3 number, ties to the one with an even last bit."""
    d = (values - y).abs()
    best = values[d == d.min()]
    if len(best) == 1:
        return best.item()
    even = [v.item() for v in best if int(v.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)) % 2 == 0]
    return even[0]


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -30, 2.0 ** 40, 3e-22, 1e21])
def test_a_row_is_held_to_the_nearest_numbers_of_the_smallest_power(scale):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(6, 32, generator=g, dtype=torch.float64) * scale).bfloat16()
    data, exps = quantise(x)
    values = _e4m3_values()
    for row, d, e in zip(x.double(), data.double(), exps.tolist()):
        top = row.abs().max().item()
        want = min(range(-E_MAX, E_MAX + 1), key=lambda c: (top > 448 * 2.0 ** c, c))
        if top > 448 * 2.0 ** E_MAX:
            want = E_MAX
        assert e == want + E_BIAS
        for a, b in zip(row.tolist(), d.tolist()):
            y = max(-448.0, min(448.0, math.ldexp(a, -want)))
            assert b == _nearest(y, values)


def test_rows_at_the_edges_of_a_power():
    x = torch.zeros(6, 32)
    for i, top in enumerate([448.0, 449.0, 896.0, 1.75, 0.0, 2.0 ** -100]):
        x[i, 3] = -top
    data, exps = quantise(x)
    assert (exps.int() - E_BIAS).tolist() == [0, 1, 1, -8, -E_MAX, -E_MAX]
    assert data[0, 3].float() == -448 and data[1, 3].float() == -224 and data[3, 3].float() == -448
    assert (data[4].float() == 0).all() and (data[5].float() == 0).all()


def test_nan_marks_the_row_and_infinity_is_the_largest_number():
    x = torch.ones(3, 64)
    x[0, 7], x[1, 9], x[1, 10] = float("nan"), float("inf"), -float("inf")
    data, exps = quantise(x)
    assert exps.tolist() == [E_NAN, E_MAX + E_BIAS, 127 - 8]
    assert (data[0].float() == 0).all()
    back = dequantise(data, exps, torch.float32)
    assert back[0].isnan().all() and back[1, 9] == 448 * 2.0 ** E_MAX and back[1, 10] == -448 * 2.0 ** E_MAX
    assert (back[2] == 1).all()


def test_a_row_comes_back_exactly_and_stays():
    """What was held once is held again without a change: e4m3 numbers times a power of two are bf16 numbers."""
    g = torch.Generator().manual_seed(2)
    data, exps = quantise(torch.randn(50, 128, generator=g).bfloat16() * 3.7)
    x = dequantise(data, exps, torch.bfloat16)
    assert torch.equal(x.float(), dequantise(data, exps, torch.float32))
    again = quantise(x)
    assert torch.equal(again[0].view(torch.uint8), data.view(torch.uint8)) and torch.equal(again[1], exps)


def _layer(pages=9, n_kv=2, D=32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return Kv8Layer(*quantise(torch.randn(pages, 2, n_kv, 64, D, generator=g)))


def test_write_and_read_by_page_table():
    layer = _layer()
    before = layer.data.clone().view(torch.uint8), layer.exps.clone()
    tables = torch.tensor([[3, 5], [7, 1]], dtype=torch.int32)
    seq, pos = torch.tensor([0, 0, 1, 1]), torch.tensor([63, 64, 0, 127])
    g = torch.Generator().manual_seed(5)
    k, v = torch.randn(4, 2, 32, generator=g), torch.randn(4, 2, 32, generator=g) * 9
    O.kv8_write(layer, k, v, pos, seq, tables)
    rk, rv = O.kv8_read(layer, pos, seq, tables)
    for got, want in ((rk, k), (rv, v)):
        assert torch.equal(got.float(), dequantise(*quantise(want), torch.float32))
    changed = (layer.exps != before[1]) | (layer.data.view(torch.uint8) != before[0]).any(-1)
    places = {(int(p), int(o)) for p, _, _, o in changed.nonzero()}
    assert places == {(3, 63), (5, 0), (7, 0), (1, 63)}


@pytest.mark.parametrize("n_q,n_kv,D,G", [(4, 1, 32, 1), (6, 3, 64, 3)])
def test_attention_is_the_formula(n_q, n_kv, D, G):
    layer = _layer(n_kv=n_kv, D=D)
    tables = torch.tensor([[3, 5], [7, 1]], dtype=torch.int32)
    last = [70, 3]
    positions = torch.tensor([p + i - (G - 1) for p in last for i in range(G)])
    g = torch.Generator().manual_seed(7)
    q, gate = torch.randn(2 * G, n_q, D, generator=g), torch.randn(2 * G, n_q * D, generator=g)
    got = O.kv8_decode(q, gate, layer, tables, positions, G).view(2 * G, n_q, D)
    kv = dequantise(layer.data, layer.exps, torch.float32).double()
    for r in range(2 * G):
        pages = tables[r // G].long()
        for h in range(n_q):
            k, v = (kv[pages, i, h // (n_q // n_kv)].reshape(-1, D)[: positions[r] + 1] for i in (0, 1))
            p = torch.softmax(k @ q[r, h].double() / math.sqrt(D), 0)
            want = (p @ v) * torch.sigmoid(gate.double().view(2 * G, n_q, D)[r, h])
            assert (got[r, h].double() - want).abs().max() < 1e-5


def test_prefill_is_decode_row_by_row_and_a_row_without_keys_is_zero():
    layer = _layer()
    tables = torch.tensor([[3, 5], [7, 1]], dtype=torch.int32)
    g = torch.Generator().manual_seed(8)
    starts, pos0 = [0, 5, 5 + 70], [60, 0]
    q, gate = torch.randn(75, 4, 32, generator=g), torch.randn(75, 128, generator=g)
    got = O.kv8_prefill(q, gate, layer, tables, starts, pos0)
    for r, (s, pos) in ((0, (0, 60)), (4, (0, 64)), (5, (1, 0)), (74, (1, 69))):
        one = O.kv8_decode(q[r : r + 1], gate[r : r + 1], layer, tables[s : s + 1], torch.tensor([pos]), 1)
        assert (got[r : r + 1] - one).abs().max() < 1e-5  # sums of fp32 in another order
    none = O.kv8_decode(q[:2], gate[:2], layer, tables, torch.tensor([-1, 5]), 1)
    assert (none[0] == 0).all() and (none[1] != 0).any()


def test_layers_that_do_not_fit_are_refused():
    data, exps = _layer()
    for bad in (Kv8Layer(data.view(torch.uint8), exps), Kv8Layer(data, exps.int()), Kv8Layer(data[:3], exps), Kv8Layer(data[..., :24], exps),
                Kv8Layer(data[::2], exps[::2]), Kv8Layer(data[:, :1], exps[:, :1]),
                Kv8Layer(data.transpose(2, 3).contiguous(), exps.transpose(2, 3).contiguous())):
        with pytest.raises(ValueError, match="kv8"):
            check_layer(bad, "kv8")
    assert check_layer(Kv8Layer(data, exps), "kv8") == (9, 2, 32)
    with pytest.raises(ValueError):
        Kv8Pool(1, 4, 2, 48, "cpu")


@pytest.mark.parametrize("D", HEAD_DIMS)
def test_pool_pages(D):
    pool = Kv8Pool(3, 5, 2, D, "cpu")
    assert pool.page_bytes == sum(t[:, 0].numel() for t in (pool.data, pool.exps))
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 2, D, generator=g)
    O.kv8_write(pool[1], x, 2 * x, torch.tensor([5]), torch.tensor([0]), torch.tensor([[4]]))
    pool.copy_page(4, 2)
    k, v = O.kv8_read(pool[1], torch.tensor([5]), torch.tensor([0]), torch.tensor([[2]]))
    assert torch.equal(v.float(), 2 * k.float()) and (k != 0).any()
    assert (O.kv8_read(pool[0], torch.tensor([5]), torch.tensor([0]), torch.tensor([[2]]))[0] == 0).all()


def _engine(kv_dtype, **kw):
    from b200serve.config import EngineConfig, ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.sched.engine import Engine

    cfg = ModelConfig.tiny()
    w = random_weights(cfg, seed=0, device="cpu", dtype=torch.float32)
    return Engine(w, EngineConfig(device="cpu", kv_dtype=kv_dtype, max_seqs=4, kv_pages=64, max_model_len=512, **kw))


def test_an_engine_with_the_8_bit_pool_serves_the_same_alone_and_in_a_batch():
    from b200serve.sched.request import Sampling

    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(5, 1000, (n,), generator=g).tolist() for n in (20, 130, 65)]
    s = Sampling(max_tokens=8, ignore_eos=True)
    with pytest.raises(ValueError, match="kv_dtype"):
        _engine("int3")
    together = _engine("e4m3")
    outs = [x.output for x in together.generate(prompts, s)]
    for p, want in zip(prompts, outs):
        assert _engine("e4m3").generate([p], s)[0].output == want
    pool = together.model.kv
    assert isinstance(pool, Kv8Pool) and together.model.page_bytes == pool.page_bytes
    plain = _engine("auto").model
    assert plain.page_bytes == 4 * pool.page_bytes * 32 // 33  # fp32 on the CPU


def test_a_prefix_moves_between_pools_of_either_type():
    from b200serve.config import ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.models.qwen36 import Model

    cfg = ModelConfig.tiny()
    w = random_weights(cfg, seed=0, device="cpu", dtype=torch.float32)
    eight, other, plain = (Model(w, 8, 2, kv_dtype=t) for t in (torch.float8_e4m3fn, torch.float8_e4m3fn, None))
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(100, cfg.num_key_value_heads, cfg.head_dim, generator=g) for _ in range(2))
    eight.write_kv(0, torch.tensor([3, 5], dtype=torch.int32), k, v)
    a = eight.read_kv(0, torch.tensor([3, 5], dtype=torch.int32), 100)
    other.write_kv(0, torch.tensor([1, 7], dtype=torch.int32), *a)
    plain.write_kv(0, torch.tensor([2, 4], dtype=torch.int32), *a)
    b = other.read_kv(0, torch.tensor([1, 7], dtype=torch.int32), 100)
    c = plain.read_kv(0, torch.tensor([2, 4], dtype=torch.int32), 100)
    for x, y, z, src in zip(a, b, c, (k, v)):
        assert torch.equal(x, y) and torch.equal(x.float(), z.float())
        assert torch.equal(x.float(), dequantise(*quantise(src), torch.float32))


@pytest.mark.parametrize("kind", ["decode", "prefill"])
@pytest.mark.parametrize("which", [0, 1])
def test_a_nan_row_reaches_the_rows_that_see_it_alone(kind, which):
    """A key or value that is marked as NaN is masked for the rows before it: their weights of 0 must not meet it."""
    layer = _layer(n_kv=2, D=32)
    tables = torch.tensor([[3, 5]], dtype=torch.int32)
    layer.data.view(torch.uint8)[5, which, 1, 4], layer.exps[5, which, 1, 4] = 0, E_NAN  # position 68, KV head 1
    g = torch.Generator().manual_seed(3)
    q, gate = torch.randn(8, 4, 32, generator=g), torch.randn(8, 128, generator=g)
    if kind == "decode":
        got = O.kv8_decode(q, gate, layer, tables, torch.arange(64, 72), 8)
    else:
        got = O.kv8_prefill(q, gate, layer, tables, [0, 8], [64])
    got = got.view(8, 4, 32)
    assert got[4:, 2:].isnan().all()
    assert got[:4].isfinite().all() and got[:, :2].isfinite().all()


def test_the_kernels_calls_refuse_tensors_that_are_not_on_a_gpu():
    from b200serve.ops import cuda_ops as C

    layer = _layer(n_kv=2, D=64)
    tables, pos, seq = torch.tensor([[3, 5]], dtype=torch.int32), torch.arange(4), torch.zeros(4, dtype=torch.int32)
    k, q, gate = torch.zeros(4, 2, 64).bfloat16(), torch.zeros(4, 4, 64).bfloat16(), torch.zeros(4, 256).bfloat16()
    words = dict(C._err)
    norm = torch.zeros(64).bfloat16()
    for call in (lambda: C.kv8_write(layer, k, k, pos, seq, tables), lambda: C.kv8_read(layer, pos, seq, tables),
                 lambda: C.kv8_decode(q, gate, layer, tables, pos, 4), lambda: C.kv8_prefill(q, gate, layer, tables, [0, 4], [0]),
                 lambda: C.attention(torch.zeros(4, 768).bfloat16(), pos, seq, tables, layer, norm, norm, 4, 2, 64, 16, 1e7, 1e-6, 4)):
        with pytest.raises(ValueError, match="(kv8_|attention).* cpu"):
            call()
    assert C._err == words


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (6, 2), (5, 1)])
def test_the_layers_of_a_pass_share_the_spans_device_tensors(n_q, n_kv):
    """Whatever the heads: a group that has no table of query tiles has its spans' rows and positions on the device all the same."""
    import types

    from b200serve.config import ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.models.qwen36 import Model, PackedBatch

    cfg = ModelConfig.tiny(num_attention_heads=n_q, num_key_value_heads=n_kv)
    w = random_weights(cfg, seed=0, device="cpu", dtype=torch.float32)
    ops = types.SimpleNamespace(**{k: getattr(O, k) for k in dir(O) if not k.startswith("__")}, SPAN_TABLES=True)
    model = Model(w, 8, 4, ops=ops, kv_dtype=torch.float8_e4m3fn)
    batch = PackedBatch.prefill([[1] * 5, [2] * 70], [1, 2], [3, 0], torch.tensor([[1, 2], [3, 4]], dtype=torch.int32), "cpu")
    args = model._attention_spans(batch)
    assert (args["seg_starts"], args["seg_pos0"]) == ([0, 5, 75], [3, 0])
    assert [t.tolist() for t in args["meta"]] == [[0, 5, 75], [3, 0]] and all(t.dtype == torch.int32 for t in args["meta"])
    again = model._attention_spans(batch)["meta"]
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(args["meta"], again))


def test_two_ranks_over_the_8_bit_pool():
    from test_tp import _launch

    r = _launch("kv8_ranks", 2, 29661, env={"CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 0 and "OK kv8_ranks" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]


def hand_over(ops, device, dtype, kv_dtypes, head_dim):
    """A prefix's keys, values and recurrent states go from one model to another, into other pages and another slot; the next
    tokens' hidden states over either, and what was handed over."""
    from b200serve.config import ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.models.qwen36 import Model, PackedBatch

    cfg = ModelConfig.tiny(num_hidden_layers=8, head_dim=head_dim, mtp_num_hidden_layers=0)
    w = random_weights(cfg, seed=0, device=device, dtype=dtype, std=0.05)
    a, b = (Model(w, 8, 4, ops=ops, kv_dtype=t) for t in kv_dtypes)
    n = 100
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(3, 1024, (n + 3,), generator=g).tolist()
    ta, tb = torch.tensor([3, 5], dtype=torch.int32), torch.tensor([6, 2], dtype=torch.int32)
    a.forward(PackedBatch.prefill([tokens[:n]], [1], [0], ta[None], device))
    rows = []
    for layer in range(cfg.num_kv_layers):
        rows.append(a.read_kv(layer, ta.to(device), n))
        b.write_kv(layer, tb.to(device), *rows[-1])
    b.conv_state[:, 2].copy_(a.conv_state[:, 1])
    b.rec_state[:, 2].copy_(a.rec_state[:, 1])
    outs = [[], []]
    for i in range(n, n + 3):
        for out, model, slot, table in zip(outs, (a, b), (1, 2), (ta, tb)):
            out.append(model.forward(PackedBatch.uniform([tokens[i]], [i], [slot], table[None], 1, device)).clone())
    return outs, rows


@pytest.mark.parametrize("to", [torch.float8_e4m3fn, None])
def test_a_generation_goes_on_over_a_prefix_that_was_handed_over(to):
    (here, there), rows = hand_over(O, "cpu", torch.float32, (torch.float8_e4m3fn, to), 32)
    assert all(k.abs().max() > 0 and k.shape == (100, 1, 32) for k, _ in rows)
    for x, y in zip(here, there):  # into a pool of full width: what is new there is not rounded to 8 bits
        assert torch.equal(x, y) if to is not None else torch.nn.functional.cosine_similarity(x, y).min() > 0.99
