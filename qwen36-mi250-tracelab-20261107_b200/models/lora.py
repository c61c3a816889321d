"""Low-rank adapters from disk: what requests of different fine-tunings share a server with.

An adapter is a directory as PEFT writes it: ``adapter_config.json`` (rank, alpha, target modules) and ``adapter_model.safetensors`` with
``...layers.N.<module>.lora_A.weight [r, in]`` and ``lora_B.weight [out, r]``. Modules that may have one are the mixers' projections:
``self_attn.{q,k,v,o}_proj`` and ``linear_attn.{in_proj_qkv, in_proj_z, in_proj_b, in_proj_a, out_proj}``. The model runs the input projections of a layer
as one product, so their adapters become one as well: the modules' ranks side by side, each with zeros in the outputs of the others.
"""

from __future__ import annotations

import json
import math
import re
from dataclasses import dataclass
from pathlib import Path

import torch

from ..config import ModelConfig
from ..ops.lora import MAX_ADAPTERS, MAX_RANK, RANK_STEP, LoraWeights
from .checkpoint import Weights

# (a draft block, or an encoder beside the text model, has layers of its own, under other names)
_NAME = re.compile(r"^(?:(?:base_model|model|language_model)\.)*layers\.(\d+)\.((?:self_attn|linear_attn)\.\w+)\.lora_([AB])(?:\.default)?\.weight$")

# The keys of a configuration that may be set: those read here, and those that change neither the formula nor which weights it is added to. Any
# other one that is set, of this format's later versions too, stands for something else than a plain low-rank product.
_PLAIN = frozenset(("peft_type", "r", "lora_alpha", "use_rslora", "bias", "init_lora_weights", "auto_mapping", "base_model_name_or_path", "revision",
                    "inference_mode", "task_type", "lora_dropout", "target_modules", "exclude_modules", "layers_to_transform", "layers_pattern", "eva_config",
                    "megatron_core", "qalora_group_size", "runtime_config", "peft_version"))
_PLAIN_INIT = frozenset(("gaussian", "eva", "orthogonal"))  # starting points that leave the base weights alone


def modules(cfg: ModelConfig, kind: str) -> tuple[list[tuple[str, int]], list[tuple[str, int]]]:
    """``(name, outputs)`` of the modules in a layer's input projection, in its order, and in its output projection."""
    if kind == "linear_attention":
        n = cfg.linear_num_value_heads
        return [("linear_attn.in_proj_qkv", cfg.gdn_conv_dim), ("linear_attn.in_proj_z", cfg.gdn_value_dim), ("linear_attn.in_proj_b", n),
                ("linear_attn.in_proj_a", n)], [("linear_attn.out_proj", cfg.hidden_size)]
    return [("self_attn.q_proj", cfg.attn_q_rows), ("self_attn.k_proj", cfg.attn_kv_rows), ("self_attn.v_proj", cfg.attn_kv_rows)], \
        [("self_attn.o_proj", cfg.hidden_size)]


def parse_adapters(spec: str) -> dict[str, str]:
    """``NAME=DIR[,NAME=DIR...]``"""
    out: dict[str, str] = {}
    for part in spec.split(","):
        name, eq, path = part.strip().partition("=")
        if not part.strip():
            continue
        if not eq or not name or not path:
            raise ValueError(f"an adapter is given as NAME=DIR, not {part.strip()!r}")
        if name in out:
            raise ValueError(f"two adapters are called {name!r}")
        out[name] = path
    return out


@dataclass
class _Adapter:
    scale: float
    parts: dict[tuple[int, str], tuple[torch.Tensor, torch.Tensor]]  # (layer, module) -> A [r, in], B [out, r]


def read_adapter(path: str | Path, cfg: ModelConfig) -> _Adapter:
    """One adapter directory, refused where it asks for what this engine does not do."""
    from safetensors import SafetensorError
    from safetensors.torch import load_file

    path = Path(path)
    try:
        conf = json.loads((path / "adapter_config.json").read_text())
        state = load_file(str(path / "adapter_model.safetensors"))
    except (OSError, ValueError, SafetensorError) as e:
        raise ValueError(f"adapter {path}: {e}") from None
    if not isinstance(conf, dict):
        raise ValueError(f"adapter {path}: its configuration is no object")
    for key, value in conf.items():
        if value and key not in _PLAIN:
            raise ValueError(f"adapter {path}: {key} is not supported")
    init = conf.get("init_lora_weights")
    if not (init is None or isinstance(init, bool) or isinstance(init, str) and init in _PLAIN_INIT):
        raise ValueError(f"adapter {path}: init_lora_weights {init!r}, which may belong to other base weights, is not supported")
    if conf.get("peft_type", "LORA") != "LORA" or conf.get("bias", "none") != "none":
        raise ValueError(f"adapter {path}: a {conf.get('peft_type')} adapter with bias {conf.get('bias')!r} is not supported")
    r = conf.get("r")
    alpha = conf.get("lora_alpha", r)
    if type(r) is not int or r < 1 or type(alpha) not in (int, float):
        raise ValueError(f"adapter {path}: rank {r!r} and alpha {alpha!r} are not a whole number from 1 on and a number")
    found: dict[tuple[int, str], dict[str, torch.Tensor]] = {}
    for name, t in state.items():
        m = _NAME.match(name)
        known = m is not None and int(m.group(1)) < cfg.num_hidden_layers
        if known:
            layer, module = int(m.group(1)), m.group(2)
            ins, outs = modules(cfg, cfg.layer_types[layer])
            known = module in dict(ins + outs)
        if not known:
            raise ValueError(f"adapter {path}: {name} is of no module that can have one")
        part = found.setdefault((layer, module), {})
        if m.group(3) in part:
            raise ValueError(f"adapter {path}: {name} gives layer {layer} {module} lora_{m.group(3)} twice")
        part[m.group(3)] = t
    if not found:
        raise ValueError(f"adapter {path}: it holds nothing")
    parts = {}
    for (layer, module), ab in found.items():
        if set(ab) != {"A", "B"}:
            raise ValueError(f"adapter {path}: layer {layer} {module} has no lora_{'B' if 'A' in ab else 'A'}")
        a, b = ab["A"].float(), ab["B"].float()
        low, high = torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max  # (what rounds to infinity in bf16 is as bad)
        ins, outs = modules(cfg, cfg.layer_types[layer])
        n = dict(ins + outs)[module]
        k = cfg.hidden_size if module in dict(ins) else mixer_width(cfg, cfg.layer_types[layer])
        if a.shape != (r, k) or b.shape != (n, r):
            raise ValueError(f"adapter {path}: layer {layer} {module} has {tuple(a.shape)} and {tuple(b.shape)}, not {(r, k)} and {(n, r)}")
        if not all(((t >= low) & (t <= high)).all() for t in (a, b)):
            raise ValueError(f"adapter {path}: layer {layer} {module} holds numbers that are not finite, or not in bf16")
        parts[layer, module] = (a, b)
    scale = alpha / math.sqrt(r) if conf.get("use_rslora") else alpha / r
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"adapter {path}: alpha {alpha}")
    return _Adapter(scale, parts)


def mixer_width(cfg: ModelConfig, kind: str) -> int:
    """Inputs of a layer's output projection."""
    return cfg.gdn_value_dim if kind == "linear_attention" else cfg.num_attention_heads * cfg.head_dim


def _merge(adapters: list[_Adapter], layer: int, mods: list[tuple[str, int]], K: int, what: str, device, dtype) -> LoraWeights | None:
    """The adapters of one projection of one layer: the modules' ranks side by side."""
    ranks = [sum(a.parts[layer, m][0].shape[0] for m, _ in mods if (layer, m) in a.parts) for a in adapters]
    if not any(ranks):
        return None
    R = (max(ranks) + RANK_STEP - 1) // RANK_STEP * RANK_STEP
    if R > MAX_RANK:
        raise ValueError(f"adapters of rank {max(ranks)} in layer {layer}'s {what} projection, at most {MAX_RANK} in all its modules")
    N, L = sum(n for _, n in mods), len(adapters)
    a, b = torch.zeros(L, R, K), torch.zeros(L, N, R)
    for i, ad in enumerate(adapters):
        at = row = 0
        for m, n in mods:
            if (layer, m) in ad.parts:
                pa, pb = ad.parts[layer, m]
                r = pa.shape[0]
                a[i, at : at + r], b[i, row : row + n, at : at + r] = pa, pb
                at += r
            row += n
    scale = torch.tensor([ad.scale for ad in adapters], dtype=torch.float32)
    return LoraWeights(a.to(device, dtype), b.to(device, dtype), scale.to(device))


def load_adapters(weights: Weights, paths: dict[str, str]) -> list[tuple[LoraWeights | None, LoraWeights | None]]:
    """The adapters of every layer's input and output projection, numbered in the order of ``paths``. ``weights`` stay as they are: engines that
    share them have adapters of their own."""
    if len(paths) > MAX_ADAPTERS:
        raise ValueError(f"{len(paths)} adapters, at most {MAX_ADAPTERS}")
    cfg = weights.config
    adapters = [read_adapter(p, cfg) for p in paths.values()]
    layers = []
    for i, lw in enumerate(weights.layers):
        ins, outs = modules(cfg, lw.kind)
        layers.append((_merge(adapters, i, ins, cfg.hidden_size, "input", weights.device, weights.dtype),
                       _merge(adapters, i, outs, mixer_width(cfg, lw.kind), "output", weights.device, weights.dtype)))
    return layers


def attach_adapters(weights: Weights, paths: dict[str, str]) -> list[str]:
    """Load the adapters into ``weights``' layers (``LayerWeights.in_lora``, ``out_lora``), for every ``Model`` that is made of them from then on;
    their names, in the order of their numbers."""
    for lw, pair in zip(weights.layers, load_adapters(weights, paths)):
        lw.in_lora, lw.out_lora = pair
    return list(paths)
