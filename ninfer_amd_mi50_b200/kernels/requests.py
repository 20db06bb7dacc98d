"""Python faces of the kernels for what a request brings of its own to a step that it shares: a low-rank adapter beside a
projection, and penalties, biases and a mask on its logits.  Everything is indexed by the step's rows on the device, so
that a step captured into a graph serves whichever requests its index tensors name.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import lib as _lib
from .ops import TUNING, _chk, _dt, _p, _stream, c_int, linear

__all__ = ["ADAPTER_RANKS", "MAX_ADAPTER_SLICES", "adapter_linear", "adapter_rank", "adjust_logits", "append_history",
           "request_status"]

ADAPTER_RANKS = (16, 32, 64, 128)       # ranks that adapters are laid out for; a smaller one is padded with zeros
MAX_ADAPTER_SLICES = 8


def adapter_rank(rank: int) -> int:
    """The rank that a pool of adapters of up to `rank` is laid out for."""
    for r in ADAPTER_RANKS:
        if 1 <= rank <= r:
            return r
    raise ValueError(f"adapter rank {rank} is not supported (1..{ADAPTER_RANKS[-1]})")


def adapter_linear(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, ids: torch.Tensor,
                   widths: Optional[Sequence[int]] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [T, K] times w [N, K] transposed, plus every row's adapter -> [T, N]:

        out[t] = x[t] w^T + scale[i] (x[t] a[i]^T) b[i]^T,   i = ids[t];   ids[t] = -1: no adapter

    `widths`: the parts that the N features are stacked of (query, key and value, say), each with rows of `a` of its own;
    [N] if left out.  a [n, len(widths) * R, K] (the parts' rows one after the other), b [n, N, R], R one of
    `ADAPTER_RANKS`, scale float32 [n], ids int32 [T].  Sums are float32 and rounded once, to x's type.  An id outside
    [-1, n) is served like -1 and reported by `check_status`.  The weights of all adapters have to be finite: rows of
    several requests share a product, in which another request's adapter is multiplied by zero."""
    for t, name in ((x, "x"), (w, "w"), (a, "a"), (b, "b"), (scale, "scale"), (ids, "ids")):
        if t.device != x.device:
            raise ValueError(f"adapter_linear: {name} lies on {t.device}, x on {x.device}")
    _chk(x, "x"); _chk(w, "w", x.dtype); _chk(a, "a", x.dtype); _chk(b, "b", x.dtype)
    _chk(scale, "scale", torch.float32); _chk(ids, "ids", torch.int32)
    dt = _dt(x)
    if x.dim() != 2 or w.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError("adapter_linear takes x [T, K], w [N, K], a [n, slices * R, K] and b [n, N, R]")
    T, K = x.shape
    N = w.shape[0]
    widths = [N] if widths is None else [int(v) for v in widths]
    n, R, S = b.shape[0], b.shape[2], len(widths)
    if w.shape[1] != K:
        raise ValueError(f"adapter_linear: x has {K} columns, w has {w.shape[1]}")
    if not 1 <= S <= MAX_ADAPTER_SLICES or min(widths) < 1 or sum(widths) != N:
        raise ValueError(f"adapter_linear: widths {widths} are not 1 to {MAX_ADAPTER_SLICES} positive parts of {N} features")
    if R not in ADAPTER_RANKS:
        raise ValueError(f"adapter_linear: rank {R} is not one of {ADAPTER_RANKS}; pad with zeros")
    if n < 1 or a.shape != (n, S * R, K) or b.shape[1] != N:
        raise ValueError(f"adapter_linear: a {tuple(a.shape)} and b {tuple(b.shape)} do not fit {S} parts, rank {R} and w "
                         f"{tuple(w.shape)}")
    if scale.shape != (n,) or ids.shape != (T,):
        raise ValueError(f"adapter_linear: scale {tuple(scale.shape)} and ids {tuple(ids.shape)} for {n} adapters and {T} rows")
    if out is None:
        out = torch.empty((T, N), dtype=x.dtype, device=x.device)
    else:
        _chk(out, "out", x.dtype)
        if out.shape != (T, N) or out.device != x.device:
            raise ValueError(f"adapter_linear: out is {tuple(out.shape)} on {out.device}, not {(T, N)} on {x.device}")
    if T == 0:
        return out
    ends, e = [], 0
    for v in widths:
        e += v
        ends.append(e)
    ends = (c_int * S)(*ends)
    if x.dtype == torch.bfloat16 and K % 8 == 0 and TUNING["adapter"] == "auto":
        lib = _lib.load()
        h = torch.empty((lib.nf_adapter_parts(c_int(T), c_int(K)), T, S * R), dtype=torch.float32, device=x.device)
        _lib.call("nf_adapter_linear", _p(x), _p(w), _p(a), _p(b), _p(scale), _p(ids), _p(h), _p(out), c_int(T), c_int(N), c_int(K),
                  c_int(R), c_int(n), c_int(S), ends, _stream())
        return out
    # float32, or rows that TMA cannot fetch: the shared product by itself, the adapters added to its float32 sums
    h = torch.empty((T, S * R), dtype=torch.float32, device=x.device)
    z = linear(x, w, out_dtype=torch.float32)
    _lib.call("nf_adapter_add", _p(x), _p(a), _p(b), _p(scale), _p(ids), _p(z), _p(h), _p(out), c_int(T), c_int(N), c_int(K),
              c_int(R), c_int(n), c_int(S), ends, c_int(dt), _stream())
    return out


def append_history(history: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, tokens: torch.Tensor) -> None:
    """history[slots[i], positions[i]] = tokens[i].  history int32 [slots, capacity]; entries with a negative slot are left
    out, others outside the log too, and reported by `check_status`."""
    _chk(history, "history", torch.int32)
    for t, name in ((slots, "slots"), (positions, "positions"), (tokens, "tokens")):
        _chk(t, name, torch.int32)
        if t.dim() != 1 or t.shape != tokens.shape or t.device != history.device:
            raise ValueError(f"append_history: {name} is {tuple(t.shape)} on {t.device}; slots, positions and tokens are lists of "
                             f"one length on {history.device}")
    if history.dim() != 2:
        raise ValueError("append_history: history is [slots, capacity]")
    if tokens.numel():
        _lib.call("nf_append_history", _p(history), _p(slots), _p(positions), _p(tokens), c_int(tokens.numel()),
                  c_int(history.shape[0]), c_int(history.shape[1]), _stream())


def adjust_logits(logits: torch.Tensor, history: torch.Tensor, slots: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
                  penalties: torch.Tensor, tokens: Optional[torch.Tensor] = None,
                  bias: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                  mask: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties for repeated tokens, biases and a mask on float32 logits [R, V] (rows may lie further apart) -> float32 [R, V].

    Row r belongs to the request whose tokens are history[slots[r], :lengths[r]] (history int32 [slots, capacity],
    capacity a multiple of 4), of which those from starts[r] on were generated.  With p, f, q = penalties[r] (float32
    [R, 3]), c and g the times that a token occurs among all and among the generated ones:

        v = logit;  v = v > 0 ? v / p^c : v p^c;  v -= f g + q [g > 0];  v += bias;  out = allowed ? v : -inf

    (1, 0, 0 changes nothing.)  `tokens` int32 [R]: the last token of each row, which is written to its log here, at
    lengths[r] - 1; left out, the log holds it already.  `bias` = (offsets int32 [R + 1], ids int32, values float32): the
    entries of row r are those from offsets[r] to offsets[r + 1], each id once.  `mask` = (bits int32 [M, (V + 31) // 32],
    index int32 [R]): bit i % 32 of word i // 32 of row index[r] is set where token i is allowed; index -1: no mask.  A
    row whose mask allows nothing is -inf throughout.  `out` may be `logits` itself.  A slot, a length or a mask row
    outside its tensor changes that row as if it had no tokens or no mask, and is reported by `check_status`."""
    _chk(logits, "logits", torch.float32, contiguous=False); _chk(history, "history", torch.int32)
    if logits.dim() != 2 or history.dim() != 2:
        raise ValueError("adjust_logits takes logits [R, V] and history [slots, capacity]")
    R, V = logits.shape
    _chk(penalties, "penalties", torch.float32)
    if penalties.shape != (R, 3):
        raise ValueError(f"adjust_logits: penalties are {tuple(penalties.shape)}, not {(R, 3)}")
    lists = [(slots, "slots", R), (lengths, "lengths", R), (starts, "starts", R)]
    if tokens is not None:
        lists.append((tokens, "tokens", R))
    offsets = ids = values = bits = index = None
    if bias is not None:
        offsets, ids, values = bias
        lists += [(offsets, "bias offsets", R + 1), (ids, "bias ids", ids.numel())]
        _chk(values, "bias values", torch.float32)
        if values.shape != ids.shape:
            raise ValueError(f"adjust_logits: {tuple(ids.shape)} bias ids, {tuple(values.shape)} values")
    if mask is not None:
        bits, index = mask
        lists.append((index, "mask index", R))
        _chk(bits, "mask bits", torch.int32)
        if bits.dim() != 2 or bits.shape[0] < 1 or bits.shape[1] != (V + 31) // 32:
            raise ValueError(f"adjust_logits: mask bits are {tuple(bits.shape)}, not [M, {(V + 31) // 32}]")
    for t, name, n in lists:
        _chk(t, name, torch.int32)
        if t.shape != (n,):
            raise ValueError(f"adjust_logits: {name} are {tuple(t.shape)}, not {(n,)}")
    for t in (history, penalties, values, bits, *(v[0] for v in lists)):
        if t is not None and t.device != logits.device:
            raise ValueError(f"adjust_logits: a tensor lies on {t.device}, the logits on {logits.device}")
    if out is None:
        out = torch.empty((R, V), dtype=torch.float32, device=logits.device)
    _chk(out, "out", torch.float32, contiguous=False)
    if out.shape != (R, V) or out.device != logits.device:
        raise ValueError(f"adjust_logits: out is {tuple(out.shape)} on {out.device}, not {(R, V)} on {logits.device}")
    strides = []
    for t, name in ((logits, "logits"), (out, "out")):
        step = t.stride(0) if R > 1 else V
        if V > 1 and t.stride(1) != 1 or step < V:
            raise ValueError(f"adjust_logits: the rows of {name} must be runs of their own, got strides {t.stride()}")
        strides.append(step)
    if R == 0 or V == 0:
        return out
    if history.shape[0] < 1 or history.shape[1] < 4 or history.shape[1] % 4:
        raise ValueError(f"adjust_logits: history is {tuple(history.shape)}; its capacity must be a multiple of 4")
    _lib.call("nf_logit_rules", _p(logits), _p(out), _p(history), _p(slots), _p(lengths), _p(starts), _p(tokens), _p(penalties),
              _p(offsets), _p(ids), _p(values), c_int(0 if ids is None else ids.numel()), _p(bits), _p(index),
              c_int(0 if bits is None else bits.shape[0]), c_int(R), c_int(V), c_int(strides[0]), c_int(strides[1]),
              c_int(history.shape[0]), c_int(history.shape[1]), _stream())
    return out


def request_status() -> int:
    """0, or what these kernels met since the last call: 1 to 14 a bounded wait that ran out, 101 + a row whose adapter was
    outside the pool, 10000001 + a row whose log or mask did not fit.  Synchronises the device."""
    lib = _lib.load()
    tc, ad, ru = int(lib.nf_adapter_tc_status()), int(lib.nf_adapter_index_status()), int(lib.nf_rules_index_status())
    return tc if tc else (100 + ad if ad else (10000000 + ru if ru else 0))
