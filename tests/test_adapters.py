"""Low-rank adapters: loading, serving several beside the shared weights, and what is refused."""

import json

import pytest
import torch

from adapter_util import merged, write_adapter
from b200serve.config import EngineConfig, ModelConfig
from b200serve.models.checkpoint import random_weights
from b200serve.models.lora import attach_adapters, parse_adapters, read_adapter
from b200serve.ops import torch_ops
from b200serve.ops.lora import LoraWeights
from b200serve.sched.engine import Engine
from b200serve.sched.request import Sampling


def _weights():
    return random_weights(ModelConfig.tiny(), seed=0, dtype=torch.float32, std=0.05, lm_head_std=0.5)


def _engine(weights, adapters="", **kw):
    return Engine(weights, EngineConfig(max_model_len=1024, prefill_chunk_tokens=64, max_seqs=8, mtp=False, adapters=adapters, **kw))


def _prompts(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(3, 1024, (int(torch.randint(16, 150, (1,), generator=g)),), generator=g).tolist() for _ in range(n)]


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    root, cfg = tmp_path_factory.mktemp("adapters"), ModelConfig.tiny()
    parts = {"all": write_adapter(root / "all", cfg, 1), "narrow": write_adapter(root / "narrow", cfg, 2, r=3, alpha=3.0, only=("q_proj", "out_proj", "in_proj_z")),
             "root": write_adapter(root / "root", cfg, 3, r=16, alpha=4.0, only=("v_proj", "o_proj", "in_proj_qkv"), use_rslora=True)}
    return {n: str(root / n) for n in parts}, parts, {"all": 2.0, "narrow": 1.0, "root": 1.0}


def test_the_operator_is_the_formula():
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(9, 24, generator=g), torch.randn(17, 24, generator=g)
    ad = LoraWeights(torch.randn(3, 8, 24, generator=g), torch.randn(3, 17, 8, generator=g), torch.tensor([1.0, -2.0, 0.5]))
    rows = torch.tensor([0, 1, 2, -1, 0, -5, 2, 1, 3], dtype=torch.int32)
    got = torch_ops.lora_linear(x, w, ad, rows)
    for t, i in enumerate(rows.tolist()):
        want = w.double() @ x[t].double()
        if 0 <= i < 3:
            want = want + ad.scale[i].double() * ad.b[i].double() @ (ad.a[i].double() @ x[t].double())
        # fp32 sums of 24 and 8 products: 40 roundings of 2^-24 of their magnitudes at most
        assert (got[t].double() - want).abs().max() <= 40 * 2.0 ** -24 * (w.abs().sum(1).max() * x.abs().max() * (1 + 20))


def test_adapters_together_are_their_merged_weights_alone(dirs):
    """A batch of requests with different adapters and none: each gets the tokens of an engine whose weights have its adapter merged in."""
    paths, parts, scale = dirs
    eng = _engine(_weights(), ",".join(f"{n}={p}" for n, p in paths.items()))
    assert eng.adapters == {"all": 0, "narrow": 1, "root": 2}
    prompts, s = _prompts(8), Sampling(max_tokens=12, ignore_eos=True)
    names = ["all", None, "narrow", "root", "all", None, "root", "narrow"]
    together = eng.generate(prompts, s, adapters=names)
    plain = _engine(_weights())
    for name in (None, "all", "narrow", "root"):
        alone = plain if name is None else _engine(merged(_weights(), parts[name], scale[name]))
        mine = [i for i, n in enumerate(names) if n == name]
        assert [together[i].output for i in mine] == [g.output for g in alone.generate([prompts[i] for i in mine], s)]
    assert together[0].output != plain.generate([prompts[0]], s)[0].output  # (the adapter shows)


def test_cached_prefixes_belong_to_their_adapter(dirs):
    paths, _, _ = dirs
    spec = ",".join(f"{n}={p}" for n, p in paths.items())
    eng, s = _engine(_weights(), spec), Sampling(max_tokens=6, ignore_eos=True)
    prompt = _prompts(1, 5)[0] + _prompts(1, 6)[0]
    first = eng.generate([prompt], s, adapters=["all"])[0]
    follow = prompt + first.output + [7, 8]
    for name in (None, "narrow"):
        other = eng.generate([follow], s, adapters=[name])[0]
        assert other.cached_tokens == 0
        assert other.output == _engine(_weights(), spec).generate([follow], s, adapters=[name])[0].output
    again = eng.generate([follow], s, adapters=["all"])[0]
    assert again.cached_tokens >= len(prompt)
    cold = _engine(_weights(), spec).generate([follow], s, adapters=["all"])[0]
    assert cold.cached_tokens == 0 and cold.output == again.output
    assert eng.generate([follow + again.output], s)[0].output == _engine(_weights()).generate([follow + again.output], s)[0].output


def test_a_slot_forgets_its_adapter(dirs):
    """More requests than state slots: a slot's next sequence runs with its own adapter, or none."""
    paths, _, _ = dirs
    eng = _engine(_weights(), f"all={paths['all']}", prefix_cache_entries=0)
    prompts, s = _prompts(12, 9), Sampling(max_tokens=5, ignore_eos=True)
    names = [None if i % 3 else "all" for i in range(12)]
    got = [g.output for g in eng.generate(prompts, s, adapters=names)]
    plain = _engine(_weights())
    for i in (1, 2, 10, 11):
        assert got[i] == plain.generate([prompts[i]], s)[0].output


def test_captured_pass_scheduling_with_adapters(dirs):
    """The decode-graph scheduling (buckets, run-ahead), run without a CUDA device."""
    paths, _, _ = dirs
    spec = ",".join(f"{n}={p}" for n, p in paths.items())
    prompts, s, names = _prompts(6, 3), Sampling(max_tokens=10, ignore_eos=True), ["all", None, "root", "narrow", None, "all"]
    graphs = _engine(_weights(), spec, graphs_on_cpu=True, decode_buckets=(1, 4, 8))
    got = [g.output for g in graphs.generate(prompts, s, adapters=names)]
    assert graphs._graphs is not None and graphs._graphs.buckets and graphs.stats["ahead_steps"] > 0
    assert got == [g.output for g in _engine(_weights(), spec, cuda_graphs=False).generate(prompts, s, adapters=names)]


def test_speculation_with_adapters(dirs):
    paths, _, _ = dirs
    prompts, s, names = _prompts(4, 4), Sampling(max_tokens=10, ignore_eos=True), ["all", None, "all", None]
    spec = Engine(_weights(), EngineConfig(max_model_len=1024, prefill_chunk_tokens=64, max_seqs=8, mtp=True, spec_k=2, adapters=f"all={paths['all']}"))
    assert spec.spec is not None
    assert [g.output for g in spec.generate(prompts, s, adapters=names)] == [
        g.output for g in _engine(_weights(), f"all={paths['all']}").generate(prompts, s, adapters=names)]


def test_refused_adapters(tmp_path, dirs):
    cfg = ModelConfig.tiny()
    ok = write_adapter(tmp_path / "ok", cfg, 0)
    assert len(read_adapter(tmp_path / "ok", cfg).parts) == len(ok) > 0
    with pytest.raises(ValueError, match="No such file"):
        read_adapter(tmp_path / "nowhere", cfg)
    for conf in ({"use_dora": True}, {"bias": "all"}, {"modules_to_save": ["lm_head"]}, {"rank_pattern": {"q_proj": 2}}, {"peft_type": "IA3"}, {"r": 5}):
        write_adapter(tmp_path / "bad", cfg, 0, **{k: v for k, v in conf.items() if k != "r"})
        if "r" in conf:
            c = json.loads((tmp_path / "bad/adapter_config.json").read_text())
            (tmp_path / "bad/adapter_config.json").write_text(json.dumps({**c, **conf}))
        with pytest.raises(ValueError, match="adapter"):
            read_adapter(tmp_path / "bad", cfg)
    from safetensors.torch import load_file, save_file

    good = load_file(str(tmp_path / "ok/adapter_model.safetensors"))
    some = next(k for k in good if "lora_A" in k)
    nan = good[some].clone()
    nan[0, 0] = float("nan")
    huge = good[some].float()
    huge[0, 0] = 3.4e38  # finite, and infinite as bf16
    write_adapter(tmp_path / "odd", cfg, 0)
    for state in ({}, {k: v for k, v in good.items() if k != some}, {**good, "base_model.model.lm_head.lora_A.weight": torch.zeros(4, 128)},
                  {**good, some: nan}, {**good, some: huge}, {**good, some: good[some][:, 1:].contiguous()}, {some.replace("layers.0", "layers.9"): good[some]}):
        save_file(state, str(tmp_path / "odd/adapter_model.safetensors"))
        with pytest.raises(ValueError, match="adapter"):
            read_adapter(tmp_path / "odd", cfg)
    write_adapter(tmp_path / "big", cfg, 0, r=100)
    with pytest.raises(ValueError, match="rank"):
        attach_adapters(_weights(), {"big": tmp_path / "big"})
    for alpha in (1e300, float("inf"), float("nan")):  # out of fp32's range
        write_adapter(tmp_path / "loud", cfg, 0)
        c = json.loads((tmp_path / "loud/adapter_config.json").read_text())
        (tmp_path / "loud/adapter_config.json").write_text(json.dumps({**c, "lora_alpha": alpha}))
        with pytest.raises(ValueError, match="alpha"):
            read_adapter(tmp_path / "loud", cfg)
    for spec in ("a", "=x", "a=", "a=x,a=y"):
        with pytest.raises(ValueError, match="adapter"):
            parse_adapters(spec)
    assert parse_adapters(" a=x , b=/y=z,") == {"a": "x", "b": "/y=z"}


def test_refused_requests_and_engines(dirs):
    paths, _, _ = dirs
    eng = _engine(_weights(), f"all={paths['all']}")
    g = eng.generate([[5, 6, 7]], Sampling(max_tokens=3), adapters=["none"])[0]
    assert g.finish_reason == "error" and g.output == []
    assert eng.generate([[5, 6, 7]], Sampling(max_tokens=3, ignore_eos=True), adapters=["all"])[0].finish_reason == "length"
    plain = _engine(_weights()).generate([[5, 6, 7]], Sampling(max_tokens=3), adapters=["all"])[0]
    assert plain.finish_reason == "error"
    with pytest.raises(ValueError, match="one GPU"):
        Engine(_weights(), EngineConfig(max_model_len=256, max_seqs=2, mtp=False, adapters=f"all={paths['all']}"), tp=object())
    ad = LoraWeights(torch.zeros(2, 8, 16), torch.zeros(2, 5, 8), torch.ones(2))
    x, w, rows = torch.zeros(3, 16), torch.zeros(5, 16), torch.zeros(3, dtype=torch.int32)
    for bad in (LoraWeights(ad.a[:1], ad.b, ad.scale), LoraWeights(ad.a[:, :7], ad.b[..., :7], ad.scale), LoraWeights(ad.a, ad.b, ad.scale.double()),
                LoraWeights(ad.a, ad.b[:, :4], ad.scale), LoraWeights(ad.a, ad.b.bfloat16(), ad.scale), LoraWeights(ad.a[0], ad.b, ad.scale)):
        with pytest.raises(ValueError, match="lora_linear"):
            torch_ops.lora_linear(x, w, bad, rows)
    from b200serve.ops import cuda_ops

    with pytest.raises(ValueError, match="torch_ops"):
        cuda_ops.lora_linear(x, w, ad, rows)


def test_ranks_of_a_replica_refuse_the_same_requests():
    """A request for an adapter reaches the other ranks with the adapter's name: were it refused by the first rank alone, they would wait for it."""
    import torch.distributed as dist

    from b200serve.parallel.lockstep import Coordinator
    from b200serve.sched.request import Generation

    sent = []

    class Wire:
        ReduceOp = dist.ReduceOp

        def all_reduce(self, t, op=None, group=None):
            pass

        def broadcast_object_list(self, msg, src, group):
            if msg[0] is not None:
                sent.append(msg[0])
            msg[0] = sent[-1]

    engines = [_engine(_weights()) for _ in range(2)]
    for rank, eng in enumerate(engines):
        eng.coordinator = Coordinator(None, rank)
        eng.coordinator.dist = Wire()
    gens = [engines[0].submit(Generation([5, 6, 7], Sampling(max_tokens=3, ignore_eos=True), adapter=a)) for a in ("all", None)]
    for eng in engines:
        eng.coordinator.sync(eng)
        eng.step(synced=True)
    assert gens[0].finish_reason == "error" and [len(e.prefilling) + len(e.running) for e in engines] == [1, 1]


def test_the_server_serves_adapters_as_models(dirs):
    import threading

    import requests

    from b200serve.api.server import Server, Service

    paths, _, _ = dirs
    eng = _engine(_weights(), f"all={paths['all']}")
    with pytest.raises(ValueError, match="adapter"):
        Service(eng, None, "all")
    from b200serve.api.tokenizer import TextCodec
    from b200serve.models.tiny import build_tokenizer
    import tempfile

    with tempfile.TemporaryDirectory() as d:
        build_tokenizer(512).save_pretrained(d)
        service = Service(eng, TextCodec(d), "tiny")
    server = Server(("127.0.0.1", 0), service)
    threading.Thread(target=server.serve_forever, daemon=True).start()
    url = f"http://127.0.0.1:{server.server_address[1]}"
    try:
        models = requests.get(url + "/v1/models", timeout=20).json()["data"]
        assert [m["id"] for m in models] == ["tiny", "all"] and models[1]["parent"] == "tiny"
        body = {"prompt": [9, 8, 7, 6], "max_tokens": 6, "temperature": 0, "ignore_eos": True, "return_token_ids": True}

        def ask(model, **more):
            return requests.post(url + "/v1/completions", json={**body, "model": model, **more}, timeout=60)

        base, tuned = ask("tiny").json(), ask("all").json()
        s = Sampling(max_tokens=6, ignore_eos=True)
        assert tuned["model"] == "all" and base["model"] == "tiny"
        assert base["choices"][0]["token_ids"] == _engine(_weights()).generate([[9, 8, 7, 6]], s)[0].output
        assert tuned["choices"][0]["token_ids"] == _engine(_weights(), f"all={paths['all']}").generate([[9, 8, 7, 6]], s, adapters=["all"])[0].output
        assert ask("other").status_code == 404
        assert ask("all", temperature=0.8, min_p=0.2, seed=3).status_code == 200
        for bad in (-0.1, 1.5, "x", True):
            assert ask("tiny", min_p=bad).status_code == 400
    finally:
        server.shutdown()
        service.worker.stop()


@pytest.mark.parametrize("graphs", [False, True])
def test_engines_over_one_set_of_weights_keep_apart(dirs, graphs):
    """Adapters belong to the engine that was given them: others over the same weights, made before or after, run with their own or with none."""
    paths, _, _ = dirs
    kw = dict(graphs_on_cpu=True, decode_buckets=(1, 4)) if graphs else dict(cuda_graphs=False)
    prompts, s = _prompts(2, 11), Sampling(max_tokens=6, ignore_eos=True)

    def ask(eng, name):
        eng.cache.clear()
        return [g.output for g in eng.generate(prompts, s, adapters=[name] * 2)]

    want = {n: ask(_engine(_weights(), f"x={paths[n]}" if n else "", **kw), "x" if n else None) for n in ("all", "root", None)}
    w = _weights()
    made = []
    for name in (None, "all", "root", None):
        made.append((_engine(w, f"x={paths[name]}" if name else "", **kw), name))
        for eng, own in made:  # (every engine that is there, after each new one)
            assert ask(eng, "x" if own else None) == want[own]
            assert ask(eng, None) == want[None]
    assert all(lw.in_lora is None and lw.out_lora is None for lw in w.layers)
    # adapters attached to the weights are those of the models made from then on, and of no engine
    model = made[1][0].model
    attach_adapters(w, {"narrow": paths["narrow"]})
    assert made[1][0].model is model and ask(made[1][0], "x") == want["all"] and ask(_engine(w, **kw), None) == want[None]


# (what PEFT writes for an ordinary adapter, defaults of its newer versions among them)
_USUAL = dict(alpha_pattern={}, arrow_config=None, auto_mapping=None, base_model_name_or_path="some/model", corda_config=None, ensure_weight_tying=False,
              eva_config=None, exclude_modules=None, fan_in_fan_out=False, inference_mode=True, init_lora_weights=True, layer_replication=None, layers_pattern=None,
              layers_to_transform=None, loftq_config={}, lora_bias=False, lora_dropout=0.05, megatron_config=None, megatron_core="megatron.core",
              modules_to_save=None, peft_version="0.18.0", qalora_group_size=16, rank_pattern={}, revision=None, target_modules=["q_proj"],
              target_parameters=None, task_type="CAUSAL_LM", trainable_token_indices=None, use_dora=False, use_qalora=False, use_rslora=False,
              alora_invocation_tokens=None, a_later_switch=None)


@pytest.mark.parametrize("conf", [
    {"alora_invocation_tokens": [5, 6]}, {"use_qalora": True}, {"layer_replication": [[0, 2], [1, 3]]}, {"target_parameters": ["experts.w"]}, {"lora_bias": True},
    {"fan_in_fan_out": True}, {"arrow_config": {"top_k": 3}}, {"megatron_config": {"x": 1}}, {"loftq_config": {"loftq_bits": 4}}, {"a_later_switch": True},
    {"corda_config": {"x": 1}}, *({"init_lora_weights": v} for v in ("pissa", "pissa_niter_16", "olora", "corda", "loftq", "something", 1, ["gaussian"]))])
def test_adapters_of_another_kind_are_refused(tmp_path, conf):
    """What is not known to leave the formula and the base weights as they are is refused, not read as a plain adapter."""
    cfg = ModelConfig.tiny()
    write_adapter(tmp_path / "a", cfg, 0, **{**_USUAL, **conf})
    with pytest.raises(ValueError, match=f"adapter .*{next(iter(conf))}"):
        read_adapter(tmp_path / "a", cfg)


@pytest.mark.parametrize("init", [True, False, None, "gaussian", "eva", "orthogonal"])
def test_usual_configurations_are_read(tmp_path, init):
    cfg = ModelConfig.tiny()
    parts = write_adapter(tmp_path / "a", cfg, 0, **{**_USUAL, "init_lora_weights": init, "eva_config": {"rho": 2.0} if init == "eva" else None})
    got = read_adapter(tmp_path / "a", cfg)
    assert got.scale == 2.0 and got.parts.keys() == parts.keys()


def _with_state(path, edit):
    from safetensors.torch import load_file, save_file

    f = str(path / "adapter_model.safetensors")
    state = load_file(f)
    edit(state)
    save_file(state, f)


@pytest.mark.parametrize("prefix", ["mtp", "base_model.model.mtp", "base_model.model.model.visual", "base_model.model.model.layers.1.sub"])
def test_other_stacks_of_layers_are_not_the_models(tmp_path, prefix):
    """The draft block has a layer 0 as well: its adapter is not one of the model's first layer."""
    cfg = ModelConfig.tiny()
    write_adapter(tmp_path / "a", cfg, 0)
    _with_state(tmp_path / "a", lambda s: s.update({f"{prefix}.layers.0.linear_attn.out_proj.lora_A.weight": torch.ones(4, cfg.gdn_value_dim),
                                                    f"{prefix}.layers.0.linear_attn.out_proj.lora_B.weight": torch.ones(cfg.hidden_size, 4)}))
    with pytest.raises(ValueError, match="no module"):
        read_adapter(tmp_path / "a", cfg)


@pytest.mark.parametrize("prefix", ["", "model.", "model.language_model.", "base_model.model.", "base_model.model.model.", "base_model.model.model.language_model.",
                                    "base_model.model.language_model.model."])
def test_names_of_the_models_layers(tmp_path, prefix):
    cfg = ModelConfig.tiny()
    parts = write_adapter(tmp_path / "a", cfg, 0)

    def rename(s):
        for k in list(s):
            s[prefix + k[k.index("layers."):].replace("lora_A.weight", "lora_A.default.weight" if "model.l" in prefix else "lora_A.weight")] = s.pop(k)

    _with_state(tmp_path / "a", rename)
    got = read_adapter(tmp_path / "a", cfg).parts
    assert got.keys() == parts.keys() and all(torch.equal(got[k][i], parts[k][i]) for k in parts for i in (0, 1))


def test_a_module_is_given_once(tmp_path):
    cfg = ModelConfig.tiny()
    write_adapter(tmp_path / "a", cfg, 0)
    _with_state(tmp_path / "a", lambda s: s.update({"layers." + k.split(".layers.")[1]: v + 1 for k, v in list(s.items())[:1]}))
    with pytest.raises(ValueError, match="twice"):
        read_adapter(tmp_path / "a", cfg)


@pytest.mark.parametrize("conf", [{"r": 0}, {"r": -4}, {"r": None}, {"r": "four"}, {"r": 4.5}, {"r": True}, {"lora_alpha": None}, {"lora_alpha": "x"}, {"lora_alpha": [1]}])
def test_numbers_of_a_configuration(tmp_path, conf):
    cfg = ModelConfig.tiny()
    write_adapter(tmp_path / "a", cfg, 0)
    f = tmp_path / "a" / "adapter_config.json"
    f.write_text(json.dumps({**json.loads(f.read_text()), **conf}))
    if conf.get("r") == 0:
        _with_state(tmp_path / "a", lambda s: s.update({k: v[:0].contiguous() if "lora_A" in k else v[:, :0].contiguous() for k, v in s.items()}))
    with pytest.raises(ValueError, match="adapter"):
        read_adapter(tmp_path / "a", cfg)


@pytest.mark.parametrize("text", ["{", "[]", "3", "null", "\xff"])
def test_broken_files(tmp_path, text):
    cfg = ModelConfig.tiny()
    write_adapter(tmp_path / "a", cfg, 0)
    (tmp_path / "a" / "adapter_config.json").write_bytes(text.encode("latin-1"))
    with pytest.raises(ValueError, match="adapter .*a"):
        read_adapter(tmp_path / "a", cfg)
    write_adapter(tmp_path / "b", cfg, 0)
    (tmp_path / "b" / "adapter_model.safetensors").write_bytes(text.encode("latin-1") * 20)
    with pytest.raises(ValueError, match="adapter .*b"):
        read_adapter(tmp_path / "b", cfg)


def test_every_prompt_has_its_adapter(dirs):
    """A list that is too short would leave requests out without a word."""
    paths, _, _ = dirs
    eng, s = _engine(_weights(), f"all={paths['all']}"), Sampling(max_tokens=2, ignore_eos=True)
    prompts = [[5, 6], [7, 8], [9, 10]]
    for adapters in (["all"], ["all", None], [None] * 4):
        with pytest.raises(ValueError, match="adapters"):
            eng.generate(prompts, s, adapters=adapters)
    assert not eng.has_work()
    assert [len(g.output) for g in eng.generate(iter(prompts), s, adapters=["all", None, "all"])] == [2, 2, 2]
    assert eng.generate([], s, adapters=[]) == [] and len(eng.generate(prompts, s, adapters=[])) == 3


def test_adapters_move_with_their_weights(dirs):
    paths, _, _ = dirs
    w = _weights()
    bare = w.nbytes()
    attach_adapters(w, {"all": paths["all"]})
    pairs = [ad for lw in w.layers for ad in (lw.in_lora, lw.out_lora)]
    assert w.nbytes() - bare == sum(t.numel() * t.element_size() for ad in pairs for t in ad)
    moved = w.to(dtype=torch.bfloat16)
    for lw, old in zip(moved.layers, w.layers):
        for ad, was in ((lw.in_lora, old.in_lora), (lw.out_lora, old.out_lora)):
            assert isinstance(ad, LoraWeights) and [t.dtype for t in ad] == [torch.bfloat16, torch.bfloat16, torch.float32]
            assert torch.equal(ad.a, was.a.bfloat16()) and torch.equal(ad.b, was.b.bfloat16()) and torch.equal(ad.scale, was.scale)
    assert {t.device.type for lw in w.to("meta").layers for t in (*lw.in_lora, *lw.out_lora)} == {"meta"}
