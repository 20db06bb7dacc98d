"""Random adapters for the tests' models, and the model with one of them added to its weights."""

import torch


def adapted_names(cfg, layers=None):
    """(name, out, in) of the checkpoint's tensors that take adapters: attention's, and a dense layer's feed-forward."""
    H, D = cfg["hidden_size"], cfg.get("head_dim", cfg["hidden_size"] // cfg["num_attention_heads"])
    q, kv, I = cfg["num_attention_heads"] * D, cfg["num_key_value_heads"] * D, cfg["intermediate_size"]
    out = []
    for l in range(cfg["num_hidden_layers"]) if layers is None else layers:
        p = f"model.layers.{l}."
        out += [(p + "self_attn.q_proj.weight", q, H), (p + "self_attn.k_proj.weight", kv, H), (p + "self_attn.v_proj.weight", kv, H),
                (p + "self_attn.o_proj.weight", H, q)]
        if l in cfg["mlp_only_layers"]:
            out += [(p + "mlp.gate_proj.weight", I, H), (p + "mlp.up_proj.weight", I, H), (p + "mlp.down_proj.weight", H, I)]
    return out


def random_adapter(cfg, seed, rank, keep=1.0):
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, n, k in adapted_names(cfg):
        if torch.rand((), generator=g) < keep:
            r = int(torch.randint(1, rank + 1, (1,), generator=g))
            # (numbers that bfloat16 holds, so that both modes have the same adapter)
            a, b = torch.randn(r, k, generator=g) / k ** 0.5, torch.randn(n, r, generator=g) * 0.1
            out[name] = (a.bfloat16().float(), b.bfloat16().float())
    return out


def merged(weights, adapter, scale):
    """The plain model's weights with scale B A added."""
    out = dict(weights)
    for name, (a, b) in adapter.items():
        out[name] = weights[name].float() + scale * (b @ a)
    return out
