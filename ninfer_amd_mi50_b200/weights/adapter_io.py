"""Reading a low-rank adapter from a folder: ``adapter_model.safetensors`` with a pair ``<module>.lora_A.weight`` [r, in] and
``<module>.lora_B.weight`` [out, r] for each adapted module, and ``adapter_config.json`` with ``r`` and ``lora_alpha``
(the scale is alpha / r, or alpha / sqrt(r) with ``use_rslora``)."""

from __future__ import annotations

import json
import math
import os
from typing import Dict, Tuple

import torch

from .safetensors_io import SafetensorsError, SafetensorsFile

_PREFIX = "base_model.model."


def read_adapter(folder: str) -> Tuple[Dict[str, Tuple[torch.Tensor, torch.Tensor]], float]:
    """(weights by the checkpoint's tensor name, scale), as `Engine.load_adapter` takes them."""
    with open(os.path.join(folder, "adapter_config.json")) as fh:
        cfg = json.load(fh)
    try:
        r, alpha = int(cfg["r"]), float(cfg["lora_alpha"])
    except (KeyError, TypeError, ValueError):
        raise SafetensorsError(f"{folder}/adapter_config.json: r and lora_alpha must be numbers") from None
    if r < 1:
        raise SafetensorsError(f"{folder}/adapter_config.json: r={r}")
    # what would change the product beyond scale B A: scales of single tensors, norms, tokens from which it counts, other base weights
    for key in ("rank_pattern", "alpha_pattern", "modules_to_save", "use_dora", "alora_invocation_tokens", "trainable_token_indices",
                "layer_replication"):
        if cfg.get(key):
            raise SafetensorsError(f"{folder}/adapter_config.json: {key} is not supported")
    start = str(cfg.get("init_lora_weights", True)).lower()
    if start.startswith(("pissa", "olora", "corda", "loftq")):
        raise SafetensorsError(f"{folder}/adapter_config.json: init_lora_weights {start!r} goes with base weights of its own")
    found: Dict[str, Dict[str, torch.Tensor]] = {}
    f = SafetensorsFile(os.path.join(folder, "adapter_model.safetensors"))
    try:
        for name in f.names():
            for side in "AB":
                end = f".lora_{side}.weight"
                if name.endswith(end):
                    module = name[:-len(end)]
                    module = module[len(_PREFIX):] if module.startswith(_PREFIX) else module
                    found.setdefault(module + ".weight", {})[side] = f.read(name).clone()
                    break
            else:
                raise SafetensorsError(f"{f.path}: {name} is not half of a low-rank pair")
    finally:
        f.close()
    for name, pair in found.items():
        if len(pair) != 2:
            raise SafetensorsError(f"{f.path}: {name} has only one half of its pair")
    return {n: (p["A"], p["B"]) for n, p in found.items()}, alpha / (math.sqrt(r) if cfg.get("use_rslora") else r)
