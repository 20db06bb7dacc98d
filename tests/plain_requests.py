"""Plain forms, in 64 bits and one row at a time, of the operators that a request brings to a step: adapters beside a
projection, penalties, biases and masks on logits; and bounds for what the kernels may be off."""

import math
from collections import Counter

import torch

HALF_F32 = 2.0 ** -24      # the most that a rounding to float32 takes from a number, relative


def plain_adapter(x, w, a, b, scale, ids, widths):
    """(y, bound): y[t] = x w^T + scale (x a^T) b^T in float64, and how far the kernels' float32 sums, the representation of
    x a^T in two bfloat16 parts and the last rounding may take a result from it."""
    x, w, a, b, s = (t.detach().cpu().double() for t in (x, w, a, b, scale))
    ids = ids.cpu().tolist()
    K, R, n = x.shape[1], b.shape[2], b.shape[0]
    y = x @ w.t()
    size = x.abs() @ w.abs().t()                 # what float32 sums round against
    off = (K + 8) * HALF_F32 * size
    for t, i in enumerate(ids):
        if not 0 <= i < n:
            continue
        h = (x[t] @ a[i].t()) * s[i]
        hs = (x[t].abs() @ a[i].abs().t()) * s[i].abs()
        h_off = (K + 8) * HALF_F32 * hs + 2.0 ** -17 * h.abs()
        lo = 0
        for j, width in enumerate(widths):
            part, sl = slice(j * R, (j + 1) * R), slice(lo, lo + width)
            y[t, sl] += b[i, sl] @ h[part]
            off[t, sl] += b[i, sl].abs() @ h_off[part] + (K + R + 8) * HALF_F32 * (b[i, sl].abs() @ h[part].abs() + size[t, sl])
            lo += width
    return y, off


def outside_rounded(got, y, off):
    """Where `got` is not the rounding, to its own type, of a number between y - off and y + off (rounding keeps order)."""
    got, dtype = got.cpu().double(), got.dtype
    rounded = lambda v: v.to(torch.float32).to(dtype).double()      # (twice rounded only a hair from the edge, outwards here)
    edge = off + 2 * HALF_F32 * y.abs()
    return ~((rounded(y - edge) <= got) & (got <= rounded(y + edge)))


def plain_rules(logits, history, slots, lengths, starts, penalties, tokens=None, bias=None, mask=None):
    """(out, bound, history afterwards), out in float64 but -inf, inf and overflow as float32 has them."""
    l, h = logits.detach().cpu().double().clone(), history.cpu().clone()
    R, V = l.shape
    off = torch.zeros_like(l)
    for r in range(R):
        n, start, slot = int(lengths[r]), int(starts[r]), int(slots[r])
        if tokens is not None:
            h[slot, n - 1] = int(tokens[r])
        log = h[slot, :n].tolist()
        p, f, q = (float(v) for v in penalties[r].cpu().double())
        every, made = Counter(log), Counter(log[max(start, 0):])
        for i in every:
            if not 0 <= i < V:
                continue
            c, g, v = every[i], made[i], float(l[r, i])
            err = 0.0
            if v != 0 and not math.isinf(v) and not math.isnan(v) and p != 1.0:
                e = c * math.log(p)
                v = math.copysign(math.exp(min(max(math.log(abs(v)) + (-e if v > 0 else e), -800), 700)), v)
                err = 12 * HALF_F32 * abs(v) + 1e-38           # a power (4 units at most), a quotient or a product
            v2 = v - g * f - (q if g else 0.0)
            err += 3 * HALF_F32 * (abs(v) + abs(g * f) + abs(q)) if math.isfinite(v2) else 0.0
            l[r, i], off[r, i] = v2, err
        if bias is not None:
            lo, hi = int(bias[0][r]), int(bias[0][r + 1])
            for i, v in zip(bias[1][lo:hi].tolist(), bias[2][lo:hi].tolist()):
                off[r, i] += 2 * HALF_F32 * (abs(float(l[r, i])) + abs(v)) if math.isfinite(float(l[r, i])) and math.isfinite(v) else 0.0
                l[r, i] += v
        if mask is not None and int(mask[1][r]) >= 0:
            words, i = mask[0][int(mask[1][r])].cpu().long(), torch.arange(V)
            left_out = (words[i // 32] >> (i % 32)) & 1 == 0
            l[r, left_out], off[r, left_out] = -math.inf, 0.0
    most = torch.finfo(torch.float32).max
    l[l > most], l[l < -most] = math.inf, -math.inf
    return l, off, h


# ---- twins of the kernels, for CPU tests of the engine's logic --------------------------------------------------------------

def adapter_linear(x, w, a, b, scale, ids, widths=None, out=None):
    y = x.float() @ w.float().t()
    R = b.shape[2]
    for t, i in enumerate(ids.tolist()):
        lo = 0
        for j, width in enumerate(widths or [w.shape[0]]):
            if i >= 0:
                h = (a[i, j * R:(j + 1) * R].float() @ x[t].float()) * scale[i]
                y[t, lo:lo + width] += b[i, lo:lo + width].float() @ h
            lo += width
    return y.to(x.dtype)


def append_history(history, slots, positions, tokens):
    history[slots.long(), positions.long()] = tokens


def adjust_logits(logits, history, slots, lengths, starts, penalties, tokens=None, bias=None, mask=None, out=None):
    y, _, h = plain_rules(logits, history, slots, lengths, starts, penalties, tokens, bias, mask)
    history.copy_(h)
    if out is not None:
        return out.copy_(y)
    return y.float()


def install(monkeypatch):
    import ninfer_amd_mi50_b200.kernels as K
    for name in ("adapter_linear", "append_history", "adjust_logits"):
        monkeypatch.setattr(K, name, globals()[name])
