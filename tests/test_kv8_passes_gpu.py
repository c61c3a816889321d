"""Passes over the 8-bit KV cache as the engine makes them: unlike spans packed together, captured passes, spans from device memory."""

import gc

import pytest
import torch
from test_kv8_gpu import _attention, _check, _layer, _rows, _tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def C():
    from b200serve.ops import cuda_ops

    cuda_ops.lib()
    return cuda_ops


@pytest.fixture(autouse=True)
def collected():
    """No engine of a test before is collected, and its graphs freed, while one of this test captures."""
    gc.collect()


class _Pass:
    """Spans of ``lens`` new rows on ``pos0`` cached tokens each, with the call over all of them and over one alone."""

    def __init__(self, C, lens, pos0, heads=(16, 2, 256), width=None, seed=9):
        n_q, n_kv, D = heads
        total = [a + b for a, b in zip(lens, pos0)]
        pages = sum((n + 63) // 64 for n in total) + 2
        self.C, self.lens, self.pos0 = C, lens, pos0
        self.layer = _layer(pages, n_kv, D)
        self.tables = _tables(total, width or max(total) // 64 + 1, pages)
        self.starts = [0]
        for n in lens:
            self.starts.append(self.starts[-1] + n)
        self.q, self.gate = _rows(self.starts[-1], n_q, D, seed)
        self.meta = tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (self.starts, pos0))

    def packed(self, meta=True):
        return self.C.kv8_prefill(self.q, self.gate, self.layer, self.tables, self.starts, self.pos0, meta=self.meta if meta else None)

    def from_device(self, starts=None, pos0=None, tables=None):
        """The call of a captured pass: no lists."""
        meta = tuple(m if x is None else torch.tensor(x, dtype=torch.int32, device=DEV) for m, x in zip(self.meta, (starts, pos0)))
        return self.C.kv8_prefill(self.q, self.gate, self.layer, self.tables if tables is None else tables, None, None, meta=meta)

    def alone(self, i):
        a, b = self.starts[i], self.starts[i + 1]
        return self.C.kv8_prefill(self.q[a:b], self.gate[a:b], self.layer, self.tables[i : i + 1], [0, b - a], [self.pos0[i]])

    def check(self, got, spans=None):
        for i in range(len(self.lens)) if spans is None else spans:
            a, b = self.starts[i], self.starts[i + 1]
            pos = torch.arange(self.pos0[i], self.pos0[i] + b - a, device=DEV)
            _check(got[a:b], _attention(self.q[a:b], self.gate[a:b], self.layer, self.tables[i].expand(b - a, -1), pos), f"span {i}")


def test_device_spans_that_do_not_fit_are_refused(C):
    p = _Pass(C, [40, 70], [100, 200])
    starts, pos0 = p.meta
    for meta in ((torch.stack([starts, starts], 1)[:, 0], pos0), (starts, torch.stack([pos0, pos0], 1)[:, 0]), (starts.long(), pos0),
                 (starts, pos0.view(1, -1)), (starts.cpu(), pos0), (starts[:2], pos0)):
        for lists in ((p.starts, p.pos0), (None, None)):
            with pytest.raises(ValueError, match="kv8_prefill: meta"):
                C.kv8_prefill(p.q, p.gate, p.layer, p.tables, *lists, meta=meta)
    with pytest.raises(ValueError, match="kv8_prefill"):
        p.from_device(tables=p.tables[:1])
    C.check_errors(p.q.device)


@pytest.mark.parametrize("starts,pos0", [([0, 40, 111], None), ([0, 40, 39], None), ([0, 40, 1 << 30], None), (None, [100, -1]),
                                         (None, [100, 251]), (None, [100, 2**31 - 1])])
def test_a_device_span_outside_its_rows_or_pages_is_left_out_and_reported(C, starts, pos0):
    p = _Pass(C, [40, 70], [100, 200], width=5)
    got = p.from_device(starts, pos0)
    with pytest.raises(C.KernelError, match="index"):
        C.check_errors(p.q.device)
    p.check(got, [0])
    p.check(p.from_device())
    C.check_errors(p.q.device)


def test_device_spans_with_more_runs_than_the_lists_say_are_reported(C):
    p = _Pass(C, [40, 70], [5000, 600])
    small = C.kv8_prefill  # the lists name short contexts, the tensors a long one
    meta = (p.meta[0], p.meta[1])
    small(p.q, p.gate, p.layer, p.tables, p.starts, [500, 600], meta=meta)
    with pytest.raises(C.KernelError, match="index"):
        C.check_errors(p.q.device)


@pytest.mark.parametrize("G", [1, 4])
def test_decode_behind_the_page_table_is_reported(C, G):
    p = _Pass(C, [G], [128 - G], width=2)
    last = torch.arange(128 - G, 128, device=DEV)
    C.kv8_decode(p.q, p.gate, p.layer, p.tables, last, G)
    C.check_errors(p.q.device)
    for beyond in (1, 64, 1 << 40):
        C.kv8_decode(p.q, p.gate, p.layer, p.tables, last + beyond, G)
        with pytest.raises(C.KernelError, match="index"):
            C.check_errors(p.q.device)


@pytest.mark.parametrize("G", [0, 1])
def test_the_block_writes_nothing_behind_the_page_table(C, G):
    """A position that no entry of the row's own table names, a sequence that the tables lack: reported, and no page changes."""
    n_q, n_kv, D, rows = 16, 2, 256, 3
    layer = _layer(8, n_kv, D)
    tables = _tables([128, 128, 100], 2, 8)
    before = layer.data.view(torch.uint8).clone(), layer.exps.clone()
    qkv = torch.randn(rows, 2 * (n_q + n_kv) * D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    norm = torch.zeros(D, device=DEV).bfloat16()
    seq = torch.arange(rows, dtype=torch.int32, device=DEV)
    good = torch.tensor([5, 6, 7], device=DEV)

    def call(positions, seq, layer=layer, qkv=qkv, n_q=n_q, n_kv=n_kv, D=D):
        return C.attention(qkv, positions, seq, tables, layer, norm, norm, n_q, n_kv, D, D // 4, 1e7, 1e-6, G, [0, 1, 2, 3], [5, 6, 7])

    for positions, of in ((torch.tensor([128, 200, 1 << 33], device=DEV), seq), (good, seq + 3), (good, seq - 3), (torch.tensor([-1, -64, -70], device=DEV), seq)):
        call(positions, of)
        with pytest.raises(C.KernelError, match="index"):
            C.check_errors(qkv.device)
        assert torch.equal(layer.data.view(torch.uint8), before[0]) and torch.equal(layer.exps, before[1])
    for wrong in ({"n_kv": 4}, {"D": 128}, {"n_q": 15}, {"qkv": qkv[:, :-1]}, {"qkv": qkv.float()}, {"positions": good[:2]}, {"seq": seq[:2]},
                  {"layer": _layer(8, 1, D)}):
        with pytest.raises(ValueError, match="attention"):
            call(**{"positions": good, "seq": seq, **wrong})
    call(good.int(), seq.long())  # other index types are taken as for the operators
    C.check_errors(qkv.device)


# ------------------------------------------------------------------ unlike spans in one pass
def test_partials_go_by_the_cut_rows_alone(C):
    """Sixteen rows on a long context are cut into 57 runs; the 6,144 rows beside them are not, and take no partials."""
    p = _Pass(C, [16, 2048, 2048, 2048], [32768, 0, 0, 0])
    alone = [p.alone(i) for i in range(4)]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = p.packed()
    torch.cuda.synchronize()
    taken = torch.cuda.max_memory_allocated() - before - got.numel() * got.element_size()
    C.check_errors(got.device)
    assert taken <= 17 << 20  # 128 CTAs of 128 rows of 258 numbers
    for i in range(4):
        assert torch.equal(got[p.starts[i] : p.starts[i + 1]], alone[i]), i
    p.check(got, [0])


MANY = ([(i * 37) % 50 + (i % 5 == 0) * 150 for i in range(75)], [(i * 977) % 4000 for i in range(75)])  # 75 spans, one of them empty


@pytest.mark.parametrize("heads", [(16, 2, 256), (6, 3, 128), (8, 1, 64)])
def test_more_spans_than_a_warp_looks_at_once(C, heads):
    p = _Pass(C, *MANY, heads=heads)
    got = p.packed()
    assert torch.equal(p.packed(meta=False), got)
    for i in range(0, 75, 7):
        assert torch.equal(got[p.starts[i] : p.starts[i + 1]], p.alone(i)), i
    C.check_errors(got.device)
    p.check(got, [0, 1, 31, 32, 33, 63, 64, 74])


def test_a_pass_of_more_partials_than_a_launch_takes(C, monkeypatch):
    p = _Pass(C, *MANY)
    want, n0 = p.packed(), C.launch_count()
    p.packed()
    one = C.launch_count() - n0
    monkeypatch.setattr(C, "KV8_PREFILL_PARTS", 40 << 20)
    n0 = C.launch_count()
    got = p.packed()
    assert C.launch_count() - n0 > 2 * one
    assert torch.equal(got, want)
    C.check_errors(got.device)


def test_lists_that_are_not_the_tensors_numbers_are_reported(C):
    """Fewer tiles, less room for partials, fewer tiles that are cut than the tensors' spans make."""
    p = _Pass(C, [40, 70], [700, 600], width=13)
    for starts, pos0 in (([0, 110, 110], [0, 0]), ([0, 5, 110], [700, 0]), ([0, 110, 110], [700, 0])):
        p.C.kv8_prefill(p.q, p.gate, p.layer, p.tables, starts, pos0, meta=p.meta)
        with pytest.raises(C.KernelError, match="index"):
            C.check_errors(p.q.device)


# ------------------------------------------------------------------ captured passes
@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 8, 64), (6, 3, 128)])
@pytest.mark.parametrize("lens,pos0", [([61], [3584]), ([600], [0]), ([64], [704]), ([1, 17, 300], [5000, 900, 40]), ([2000, 30], [100, 4000]), ([5], [100])])
@pytest.mark.parametrize("width", [None, 600])
def test_spans_from_device_memory_are_cut_as_from_the_lists(C, heads, lens, pos0, width):
    p = _Pass(C, lens, pos0, heads, width=width)
    want = p.packed()
    assert torch.equal(p.from_device(), want)
    for i in range(len(lens)):
        assert torch.equal(p.alone(i), want[p.starts[i] : p.starts[i + 1]]), i
    C.check_errors(want.device)
    p.check(want, [i for i, n in enumerate(lens) if n <= 64])


def test_many_spans_from_device_memory(C, monkeypatch):
    p = _Pass(C, *MANY)
    want = p.packed()
    assert torch.equal(p.from_device(), want)
    monkeypatch.setattr(C, "KV8_PREFILL_PARTS", 40 << 20)
    assert torch.equal(p.from_device(), want)
    C.check_errors(want.device)


def test_a_captured_pass_has_the_eager_bits_at_each_replay(C):
    """One graph, whose spans and positions change between replays: cut, not cut, cut otherwise."""
    p = _Pass(C, [90, 20, 18], [3000, 0, 0], width=80)
    p.tables[1:] = p.tables[:1]  # the fillers' keys are whatever lies there
    graph = torch.cuda.CUDAGraph()
    p.from_device()
    torch.cuda.synchronize()
    meta = tuple(m.clone() for m in p.meta)
    with torch.cuda.graph(graph):
        out = C.kv8_prefill(p.q, p.gate, p.layer, p.tables, None, None, meta=meta)
    for starts, pos0 in (([0, 90, 110, 128], [3000, 0, 0]), ([0, 1, 64, 128], [2999, 0, 0]), ([0, 90, 110, 128], [17, 0, 0]), ([0, 128, 128, 128], [2900, 0, 0])):
        meta[0].copy_(torch.tensor(starts, dtype=torch.int32))
        meta[1].copy_(torch.tensor(pos0, dtype=torch.int32))
        graph.replay()
        want = C.kv8_prefill(p.q, p.gate, p.layer, p.tables, starts, pos0)
        assert torch.equal(out, want), (starts, pos0)
    C.check_errors(out.device)


def test_engine_with_captured_prefill_of_cut_spans(C):
    """Prompts whose later chunks are cut, and a session's next turn: alone with captured passes, alone without, and packed."""
    from b200serve.config import EngineConfig, ModelConfig
    from b200serve.models.checkpoint import random_weights
    from b200serve.sched.engine import Engine
    from b200serve.sched.request import Sampling

    cfg = ModelConfig.tiny(head_dim=64, num_attention_heads=4, num_key_value_heads=1)
    w = random_weights(cfg, seed=0, device=DEV, dtype=torch.bfloat16, std=0.05, lm_head_std=0.5)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(3, 1024, (n,), generator=g).tolist() for n in (600, 333, 850)]
    s = Sampling(max_tokens=24, ignore_eos=True)

    def engine(**kw):
        return Engine(w, EngineConfig(max_model_len=1024, prefill_chunk_tokens=64, max_seqs=8, kv_pages=256, decode_buckets=(1, 4), kv_dtype="e4m3", mtp=False, **kw))

    packed = engine()
    want = [x.output for x in packed.generate(prompts, s)]
    graphs, plain = engine(prefill_graphs=True), engine()
    for p, out in zip(prompts, want):
        assert graphs.generate([p], s)[0].output == plain.generate([p], s)[0].output == out
        turn = p + out + [9, 8, 7, 6, 5]
        assert graphs.generate([turn], s)[0].output == plain.generate([turn], s)[0].output
    assert graphs.stats["prefill_graph_passes"] >= sum(len(p) // 64 for p in prompts) and not graphs._pgraphs.errors
    C.check_errors(torch.device(DEV))


# ------------------------------------------------------------------ the model's pool
def _tiny(C, head_dim=64, n_q=4, n_kv=1):
    from b200serve.config import ModelConfig
    from b200serve.models.checkpoint import random_weights

    cfg = ModelConfig.tiny(head_dim=head_dim, num_attention_heads=n_q, num_key_value_heads=n_kv)
    return cfg, random_weights(cfg, seed=0, device=DEV, dtype=torch.bfloat16, std=0.05, lm_head_std=0.5)


def test_rows_of_other_types_go_into_the_8_bit_pool(C):
    from b200serve.models.qwen36 import Model
    from b200serve.ops.kv8 import dequantise, quantise

    cfg, w = _tiny(C)
    model = Model(w, 8, 2, ops=C, kv_dtype=torch.float8_e4m3fn)
    table = torch.tensor([3, 5], dtype=torch.int32, device=DEV)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        k, v = (torch.randn(100, 1, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)).to(dtype) for i in (0, 1))
        model.write_kv(0, table, k, v)
        for got, src in zip(model.read_kv(0, table, 100), (k, v)):
            assert torch.equal(got, dequantise(*quantise(src.bfloat16()), torch.bfloat16))
    C.check_errors(k.device)


@pytest.mark.parametrize("head_dim,n_q,n_kv,native", [(32, 4, 1, False), (64, 6, 2, True), (64, 4, 4, True)])
def test_engine_captures_what_can_be_captured(C, head_dim, n_q, n_kv, native):
    """Heads without an attention kernel over the 8-bit pool run without graphs, and none is tried."""
    from b200serve.config import EngineConfig
    from b200serve.sched.engine import Engine
    from b200serve.sched.request import Sampling

    cfg, w = _tiny(C, head_dim, n_q, n_kv)
    assert C.kv8_kernels(n_q, n_kv, head_dim) == native
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(3, 1024, (n,), generator=g).tolist() for n in (17, 190)]
    s = Sampling(max_tokens=8, ignore_eos=True)

    def run(prompts, **kw):
        gc.collect()
        eng = Engine(w, EngineConfig(max_model_len=512, prefill_chunk_tokens=64, max_seqs=4, kv_pages=64, decode_buckets=(1, 4), kv_dtype="e4m3", **kw))
        eng.warmup()
        return eng, [x.output for x in eng.generate(prompts, s)]

    eng, outs = run(prompts, mtp=False)
    assert (eng._graphs is not None) == native and not (native and eng._graphs.errors)
    assert run(prompts[1:], mtp=False)[1] == outs[1:] and all(len(o) == 8 for o in outs)
    assert run(prompts, mtp=True, spec_k=2)[1] == outs
    C.check_errors(torch.device(DEV))


def test_a_generation_goes_on_over_a_prefix_that_was_handed_over(C):
    from test_kv8 import hand_over

    (here, there), rows = hand_over(C, DEV, torch.bfloat16, (torch.float8_e4m3fn,) * 2, 64)
    C.check_errors(torch.device(DEV))
    assert all(torch.equal(x, y) and x.isfinite().all() for x, y in zip(here, there))
    assert all(k.abs().max() > 0 and k.shape == (100, 1, 64) for k, _ in rows)


# ------------------------------------------------------------------ more than a launch, and the block
@pytest.mark.parametrize("heads", [(16, 2, 256), (8, 1, 64), (6, 3, 128)])
@pytest.mark.parametrize("G", [1, 3])
def test_decode_of_more_sequences_than_a_launch_takes_with_partials(C, heads, G):
    """Two launches, each with the join of its own rows; lengths around the ends of runs, and rows without keys."""
    B = 300
    lens = [(0, 1, 511, 512, 513, 700, 1024, 1025, 64, 1300)[i % 10] for i in range(B)]
    n_q, n_kv, D = heads
    pages = sum((n + 63) // 64 for n in lens) + 2
    layer = _layer(pages, n_kv, D)
    tables = _tables(lens, 22, pages)
    positions = torch.tensor([n - G + i for n in lens for i in range(G)], device=DEV)
    q, gate = _rows(B * G, n_q, D, 1)
    got = C.kv8_decode(q, gate, layer, tables, positions, G)
    C.check_errors(q.device)
    for a, b in ((0, 20), (250, 262), (290, 300)):
        rows = slice(a * G, b * G)
        _check(got[rows], _attention(q[rows], gate[rows], layer, tables[a:b].repeat_interleave(G, 0), positions[rows]), (a, b))
        one = C.kv8_decode(q[rows], gate[rows], layer, tables[a:b], positions[rows], G)
        assert torch.equal(one, got[rows])


@pytest.mark.parametrize("n_q,n_kv,D,G", [(16, 2, 256, 1), (16, 2, 256, 4), (16, 2, 256, 0), (6, 3, 128, 0), (4, 1, 64, 2)])
def test_the_block_is_the_fused_write_and_the_operator(C, n_q, n_kv, D, G):
    """The block's output has the bits of the operator on the queries and gates that the fused write leaves, and keeps the operator's
    bound; the queries are the formula's, rounded to bf16 at each of the kernel's steps."""
    from b200serve.ops import torch_ops as O
    from b200serve.ops.kv8 import Kv8Layer

    rot, theta, eps = D // 4, 1e7, 1e-6
    per, pos0 = ([G] * 3 if G else [70, 1, 130]), [5, 64, 600]
    starts = [0]
    for n in per:
        starts.append(starts[-1] + n)
    T = starts[-1]
    g = torch.Generator(device=DEV).manual_seed(D + G)
    layer = _layer(30, n_kv, D, seed=2)
    tables = _tables([a + b for a, b in zip(per, pos0)], 12, 30)
    qkv = torch.randn(T, n_q * 2 * D + 2 * n_kv * D, device=DEV, generator=g).bfloat16()
    positions = torch.cat([torch.arange(p, p + n) for p, n in zip(pos0, per)]).to(DEV)
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(per)]).int().to(DEV)
    qn, kn = ((torch.randn(D, device=DEV, generator=g) * 0.1).bfloat16() for _ in range(2))
    q = torch.empty(T, n_q, D, dtype=torch.bfloat16, device=DEV)
    gate = torch.empty(T, n_q * D, dtype=torch.bfloat16, device=DEV)
    other = Kv8Layer(layer.data.clone(), layer.exps.clone())
    rc = C.lib().b200_attn_prep_kv8(
        qkv.data_ptr(), qkv.stride(0), positions.data_ptr(), tables.data_ptr(), 12, 12, 3, seq.data_ptr(), qn.data_ptr(), kn.data_ptr(), q.data_ptr(),
        gate.data_ptr(), other.data.data_ptr(), other.exps.data_ptr(), T, n_q, n_kv, D, rot, theta, eps, 30,
        C.err_word(qkv.device).data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    got = C.attention(qkv, positions, seq, tables, layer, qn, kn, n_q, n_kv, D, rot, theta, eps, G, starts, pos0)
    C.check_errors(qkv.device)
    assert torch.equal(layer.data.view(torch.uint8), other.data.view(torch.uint8)) and torch.equal(layer.exps, other.exps)
    want = C.kv8_decode(q, gate, layer, tables, positions, G) if G else C.kv8_prefill(q, gate, layer, tables, starts, pos0)
    assert torch.equal(got, want)
    _check(got, _attention(q, gate, layer, tables[seq.long()], positions))
    rq, rgate, _, _ = O.attn_prep(qkv.float(), positions, qn.float(), kn.float(), n_q, n_kv, D, rot, theta, eps)
    assert torch.equal(gate.float(), rgate)
    # three roundings to bf16 (the norm, cosine and sine, their products) of numbers no larger than the head's largest rotated ones, and the last one
    assert ((q.float() - rq).abs() <= 5 * 2.0 ** -8 * rq.abs().amax(-1, keepdim=True)).all()
