"""Adapters and sampling together on the CUDA path: a batch whose requests each bring their own."""

import pytest
import torch

from adapter_util import write_adapter
from b200serve.config import EngineConfig, ModelConfig
from b200serve.models.checkpoint import random_weights
from b200serve.sched.engine import Engine
from b200serve.sched.request import Sampling

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def spec(tmp_path_factory):
    root, cfg = tmp_path_factory.mktemp("adapters"), ModelConfig.tiny()
    for i, (r, only) in enumerate(((4, None), (16, ("q_proj", "v_proj", "o_proj", "in_proj_qkv")), (7, ("out_proj", "o_proj", "in_proj_z")))):
        write_adapter(root / f"a{i}", cfg, i, r=r, only=only, dtype=torch.bfloat16)
    return ",".join(f"a{i}={root / f'a{i}'}" for i in range(3))


def _engine(adapters="", **kw):
    w = random_weights(ModelConfig.tiny(), seed=0, device="cuda", dtype=torch.bfloat16, std=0.05, lm_head_std=0.5)
    return Engine(w, EngineConfig(**{**dict(max_model_len=1024, prefill_chunk_tokens=64, max_seqs=8, mtp=False, kv_pages=256, decode_buckets=(1, 4, 8)),
                                     "adapters": adapters, **kw}))


def _prompts(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(3, 1024, (int(torch.randint(16, 200, (1,), generator=g)),), generator=g).tolist() for _ in range(n)]


NAMES = ["a0", None, "a1", "a2", "a0", None, "a2", "a1"]


def _asks():
    s = lambda **kw: Sampling(max_tokens=14, ignore_eos=True, **kw)  # noqa: E731
    return [s(), s(temperature=0.8, top_k=20, top_p=0.9, seed=1), s(temperature=1.0, min_p=0.1, seed=2), s(), s(temperature=1.2, top_p=0.95, seed=3),
            s(), s(temperature=0.7, seed=4), s(temperature=1.0, top_k=3, seed=5)]


@pytest.mark.parametrize("pack", [False, True])
def test_a_mixed_batch_is_its_requests_alone(spec, pack):
    from b200serve.ops import cuda_ops

    prompts = _prompts(8)
    eng = _engine(spec, pack_weights=pack)
    together = [g.output for g in eng.generate(prompts, _asks(), adapters=NAMES)]
    assert eng._graphs is not None and not eng._graphs.errors
    solo = _engine(spec, pack_weights=pack)
    for i in range(8):
        solo.cache.clear()
        assert solo.generate([prompts[i]], [_asks()[i]], adapters=[NAMES[i]])[0].output == together[i], i
    eager = _engine(spec, pack_weights=pack, cuda_graphs=False)
    assert [g.output for g in eager.generate(prompts, _asks(), adapters=NAMES)] == together
    # an engine without adapters gives the bare requests' tokens
    bare = [i for i, n in enumerate(NAMES) if n is None]
    plain = _engine(pack_weights=pack)
    assert [g.output for g in plain.generate([prompts[i] for i in bare], [_asks()[i] for i in bare])] == [together[i] for i in bare]
    assert together[0] != plain.generate([prompts[0]], [_asks()[0]])[0].output
    cuda_ops.check_errors(torch.device("cuda"))


def test_speculation_and_captured_prefill_with_adapters(spec):
    prompts, s = _prompts(4, 2), Sampling(max_tokens=14, ignore_eos=True)
    names = NAMES[:4]
    want = [g.output for g in _engine(spec).generate(prompts, s, adapters=names)]
    fast = _engine(spec, mtp=True, spec_k=2)
    assert fast.spec is not None
    assert [g.output for g in fast.generate(prompts, s, adapters=names)] == want
    captured = _engine(spec, prefill_graphs=True, prefill_graph_rows=(128,))
    got = []
    for p, n in zip(prompts, names):
        got.append(captured.generate([p], s, adapters=[n])[0].output)
    assert got == want


def test_adapters_against_the_cpu_path(spec):
    """The same adapters in bf16 through the kernels and through the PyTorch operators: the first hidden rows of a pass differ by roundings alone."""
    from b200serve.models.lora import attach_adapters, parse_adapters
    from b200serve.models.qwen36 import Model, PackedBatch
    from b200serve.ops import cuda_ops, torch_ops

    toks, hidden = [_prompts(1, i)[0][:16] for i in range(4)], []
    for ops in (cuda_ops, torch_ops):
        w = random_weights(ModelConfig.tiny(), seed=0, device="cuda", dtype=torch.bfloat16, std=0.05, lm_head_std=0.5)
        w.layers = w.layers[:1]
        w.config.num_hidden_layers, w.config.layer_types = 1, w.config.layer_types[:1]
        full = ModelConfig.tiny()
        w.config, one = full, w.config
        w.layers = w.layers
        attach_adapters(w, parse_adapters(spec))
        w.config = one
        m = Model(w, 8, 8, ops=ops)
        m.slot_adapter[1:5] = torch.tensor([0, -1, 1, 2], dtype=torch.int32, device="cuda")
        table = torch.arange(1, 5, dtype=torch.int32)[:, None]
        hidden.append(m.forward(PackedBatch.prefill(toks, [1, 2, 3, 4], [0] * 4, table, "cuda")).float())
    a, b = hidden
    # one layer: a dozen bf16 roundings (2^-9 each) between the adapters and the normed output, whose numbers are about 1
    assert (a - b).norm() / b.norm() < 12 * 2.0 ** -9


@pytest.mark.parametrize("pack", [False, True])
def test_engines_over_one_set_of_weights(spec, pack):
    """Two engines with other adapters under one name, and one without, over the same weights: captured and eager passes of each go by its own."""
    own = [f"x={part.split('=')[1]}" for part in spec.split(",")[:2]] + [""]
    kw = dict(max_model_len=1024, prefill_chunk_tokens=64, max_seqs=8, mtp=False, kv_pages=256, decode_buckets=(1, 4, 8), pack_weights=pack)
    prompts, s = _prompts(4, 7), Sampling(max_tokens=10, ignore_eos=True)

    def ask(eng, name):
        eng.cache.clear()
        return [g.output for g in eng.generate(prompts, s, adapters=[name, None, name, name])]

    want = [ask(_engine(a, pack_weights=pack), "x" if a else None) for a in own]
    assert want[0] != want[1] != want[2]
    w = random_weights(ModelConfig.tiny(), seed=0, device="cuda", dtype=torch.bfloat16, std=0.05, lm_head_std=0.5)
    engines = []
    for a in own:
        engines.append(Engine(w, EngineConfig(**kw, adapters=a)))
        for _ in range(2):
            assert [ask(e, "x" if b else None) for e, b in zip(engines, own)] == want[: len(engines)]
