"""Adapters beside projections whose float32 sums go on to a rotation or an activation: rounded as often as without adapters."""

import pytest
import torch

from plain_requests import HALF_F32, outside_rounded, plain_adapter
from test_adapter_gpu import SIZES, check, make
from test_parts_gpu import fetcher, random_tensors, simple_ctx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,K,widths,n,R", SIZES + [(9, 7, [33, 20], 3, 16), (150, 130, [33, 20], 3, 16), (300, 264, [255, 1, 77], 4, 32)])
def test_sums_against_the_plain_form(T, K, widths, n, R):
    from ninfer_amd_mi50_b200 import kernels
    args = make(T, K, widths, n, R, torch.bfloat16, seed=T + K)
    sums = kernels.adapter_linear(*args, widths, out_dtype=torch.float32)
    assert sums.dtype == torch.float32
    check(args, widths, sums)
    assert torch.equal(sums.bfloat16(), kernels.adapter_linear(*args, widths))       # what is rounded is the same
    kernels.check_status("adapter")


def test_types_of_the_result():
    from ninfer_amd_mi50_b200 import kernels
    args = make(5, 64, [64], 2, 16, torch.bfloat16)
    out = torch.empty((5, 64), dtype=torch.float32).cuda()
    assert kernels.adapter_linear(*args, out=out, out_dtype=torch.float32) is out
    with pytest.raises(TypeError):
        kernels.adapter_linear(*args, out=out)
    with pytest.raises(TypeError):
        kernels.adapter_linear(*args, out_dtype=torch.float16)
    args = make(5, 64, [64], 2, 16, torch.float32)
    with pytest.raises(TypeError):
        kernels.adapter_linear(*args, out_dtype=torch.bfloat16)


def turned(y, off, positions, inv_freq, heads, D):
    """Half-split rotation of [T, heads * D] in float64 and how far float32 (cosine and sine to two units in the last place, two
    products and a sum) may be off."""
    T, half = y.shape[0], D // 2
    angle = (positions.float()[:, None] * inv_freq.cpu().float()[None]).double()      # the angle is float32's
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = y.view(T, heads, D)[..., :half], y.view(T, heads, D)[..., half:]
    ea, eb = off.view(T, heads, D)[..., :half], off.view(T, heads, D)[..., half:]
    e = ea + eb + (a.abs() + b.abs()) * 5 * HALF_F32
    return torch.cat([a * c - b * s, a * s + b * c], -1).reshape(T, -1), torch.cat([e, e], -1).reshape(T, -1)


def pool(part, which, R, seed):
    from ninfer_amd_mi50_b200.parts.adapters import ProjectionAdapters
    g = torch.Generator().manual_seed(seed)
    p = part.projections()[which]
    out = ProjectionAdapters(p, 2, R, torch.bfloat16, "cuda", torch.tensor([1.25, 0.5]).cuda())
    out.a.copy_(torch.randn(out.a.shape, generator=g) / p.in_features ** 0.5)
    out.b.copy_(torch.randn(out.b.shape, generator=g) * 0.2)
    return out


@pytest.mark.parametrize("Hq,Hkv,D,bias", [(6, 2, 48, True), (4, 1, 128, False), (16, 16, 64, True)])
def test_keys_and_values_of_a_decode_step_are_rounded_once(Hq, Hkv, D, bias):
    from ninfer_amd_mi50_b200 import kernels
    from ninfer_amd_mi50_b200.config import PartSpec
    from ninfer_amd_mi50_b200.parts.attention import PagedGqaAttention
    from ninfer_amd_mi50_b200.parts.base import CacheView
    H, page, seg_lens = 520, 16, [9, 3, 4]
    T = sum(seg_lens)
    att = PagedGqaAttention(hidden_size=H, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, qkv_bias=bias,
                            position=PartSpec.make("rotary_half_split", head_dim=D, theta=5e4), prefix="a.")
    att.load(fetcher(random_tensors(att.tensor_specs(), 2), torch.bfloat16)(att.tensor_specs()))
    att.adapters = {w: pool(att, w, 16, 5) for w in ("qkv", "o")}
    ctx, bt, n_pages = simple_ctx(torch.bfloat16, seg_lens, page)
    ids = torch.tensor([-1] * 9 + [0] * 3 + [1, 1, -1, 0], dtype=torch.int32)
    ctx.row_adapter = ids.cuda()
    pages = torch.zeros((n_pages + 1, 2, Hkv, page, D), dtype=torch.bfloat16, device="cuda")
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(1)).bfloat16()
    att.forward(x.cuda(), ctx, CacheView(att.cache_spec(), pages, bt, page, True), None)
    kernels.check_status("attention")
    p = att.adapters["qkv"]
    y, off = plain_adapter(x, att.w_qkv, p.a, p.b, p.scale, ids, p.projection.widths)
    if bias:
        y = y + att.b_qkv.double().cpu()
        off = off + y.abs() * HALF_F32
    q, k = att.q_width, att.kv_width
    inv_freq, rot = att.position.rotary_table(torch.device("cuda"))
    k_want, k_off = turned(y[:, q:q + k], off[:, q:q + k], ctx.positions.cpu(), inv_freq, Hkv, D)
    for what, (want, e) in enumerate(((k_want, k_off), (y[:, q + k:], off[:, q + k:]))):
        got = torch.stack([pages[int(bt[s, pos // page]), what, :, pos % page].reshape(-1)
                           for s, pos in zip(ctx.row_seg.tolist(), ctx.positions.tolist())])
        wrong = outside_rounded(got, want, e)
        assert not wrong.any(), (what, int(wrong.sum()), wrong.numel(), wrong.any(1).tolist())
    # the queries, by the kernel alone
    sums = p.linear(x.cuda(), att.w_qkv, ctx.row_adapter, torch.float32)
    b = att.b_qkv if bias else None
    turned_q = kernels.rope_append_sums(sums, b, ctx.positions, ctx.row_seg, inv_freq, Hq, Hkv, D, pages, bt, page, False)
    q_want, q_off = turned(y[:, :q], off[:, :q], ctx.positions.cpu(), inv_freq, Hq, D)
    assert not outside_rounded(turned_q[:, :q].contiguous(), q_want, q_off).any()


@pytest.mark.parametrize("activation,T", [(("silu",), 12), (("gelu_tanh",), 12), (("capped", 0.75, 1.702), 12), (("capped", 0.75, 1.702), 40),
                                          (("capped", 0.75, 1.702), 150)])
def test_the_activation_takes_sums_where_it_does_without_adapters(activation, T, monkeypatch):
    from ninfer_amd_mi50_b200 import kernels
    from ninfer_amd_mi50_b200.parts.feedforward import DenseSwiglu
    H, I = 520, 232
    ff = DenseSwiglu(hidden_size=H, intermediate_size=I, prefix="m.", activation=activation)
    ff.load(fetcher(random_tensors(ff.tensor_specs(), 3), torch.bfloat16)(ff.tensor_specs()))
    ff.adapters = {w: pool(ff, w, 32, 6) for w in ("gate_up", "down")}
    ctx, _, _ = simple_ctx(torch.bfloat16, [T])
    ids = torch.tensor([-1, 0, 1, 1] * T, dtype=torch.int32)[:T].contiguous()
    ctx.row_adapter = ids.cuda()
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(1)).bfloat16()
    seen, project = [], ff.project
    monkeypatch.setattr(ff, "project", lambda which, v, *a: (seen.append(v), project(which, v, *a))[1])
    out = ff.forward(x.cuda(), ctx)
    assert out.dtype == (torch.float32 if activation[0] == "capped" else torch.bfloat16)
    kernels.check_status("feed-forward")
    p = ff.adapters["gate_up"]
    y, off = plain_adapter(x, ff.w_gate_up, p.a, p.b, p.scale, ids, p.projection.widths)
    g, u, eg, eu = y[:, :I], y[:, I:], off[:, :I], off[:, I:]
    if activation[0] == "capped":
        _, limit, alpha = activation
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
        gate, eu = g * torch.sigmoid(alpha * g), eu + u.abs() * HALF_F32
        own = gate.abs() * (16 + 8 * g.abs()) * HALF_F32
    elif activation[0] == "silu":
        gate = g * torch.sigmoid(g)
        own = gate.abs() * (16 + 4 * g.abs()) * HALF_F32       # an exponential to 2 + 1.2 |g| units, a sum, a quotient, a product
    else:
        gate = torch.nn.functional.gelu(g, approximate="tanh")
        own = gate.abs() * 8 * HALF_F32 + g.abs() * 16 * HALF_F32       # 1 + tanh cancels below 0: two units of 1, times g / 2
    # neither gate's slope exceeds 1.13
    want, e = gate * u, (1.13 * eg + own) * u.abs() + (gate.abs() + 1.13 * eg + own) * eu + 4 * HALF_F32 * (gate * u).abs()
    wrong = outside_rounded(seen[1], want, e)
    assert not wrong.any(), (int(wrong.sum()), wrong.numel(), wrong.any(1).tolist())
