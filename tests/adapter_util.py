"""Adapter directories as PEFT writes them, with random numbers."""

import json

import torch

from b200serve.models.lora import mixer_width, modules


def write_adapter(path, cfg, seed, r=4, alpha=8.0, only=None, dtype=torch.float32, std=0.15, **conf):
    """``only``: the modules that have one (all if None). Returns what it wrote: (layer, module) -> (A, B)."""
    from safetensors.torch import save_file

    g = torch.Generator().manual_seed(seed)
    state, parts = {}, {}
    for layer, kind in enumerate(cfg.layer_types):
        ins, outs = modules(cfg, kind)
        for group, k in ((ins, cfg.hidden_size), (outs, mixer_width(cfg, kind))):
            for m, n in group:
                if only is not None and m.split(".")[-1] not in only:
                    continue
                a, b = (torch.randn(r, k, generator=g) * std).to(dtype), (torch.randn(n, r, generator=g) * std).to(dtype)
                parts[layer, m] = (a, b)
                for x, t in (("A", a), ("B", b)):
                    state[f"base_model.model.model.language_model.layers.{layer}.{m}.lora_{x}.weight"] = t
    path.mkdir(parents=True, exist_ok=True)
    save_file(state, str(path / "adapter_model.safetensors"))
    (path / "adapter_config.json").write_text(json.dumps({"peft_type": "LORA", "r": r, "lora_alpha": alpha, "bias": "none", **conf}))
    return parts


def merged(weights, parts, scale):
    """``weights`` with an adapter's products added to its projections (in place)."""
    cfg = weights.config
    for layer, lw in enumerate(weights.layers):
        for group, name in zip(modules(cfg, lw.kind), ("in_proj", "out_proj")):
            row, w = 0, getattr(lw, name)
            for m, n in group:
                if (layer, m) in parts:
                    a, b = parts[layer, m]
                    w[row : row + n] += (scale * b.float() @ a.float()).to(w)
                row += n
    return weights
