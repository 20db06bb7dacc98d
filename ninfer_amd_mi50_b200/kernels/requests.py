"""Python faces of the kernels for what a request brings of its own to a step that it shares: a low-rank adapter beside a
projection, and penalties, biases and a mask on its logits.  Everything is indexed by the step's rows on the device, so
that a step captured into a graph serves whichever requests its index tensors name.

These calls come many times a step and take a few microseconds on the device, so the host's part is kept short: one
condition over all operands, and a second look, for the message, only where it fails.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import lib as _lib
from .ops import TUNING, _DT, _chk, _dt, linear

__all__ = ["ADAPTER_RANKS", "MAX_ADAPTER_SLICES", "adapter_linear", "adapter_rank", "adjust_logits", "append_history",
           "request_status"]

ADAPTER_RANKS = (16, 32, 64, 128)       # ranks that adapters are laid out for; a smaller one is padded with zeros
MAX_ADAPTER_SLICES = 8

_I, _P = ctypes.c_int, ctypes.c_void_p
_F32, _BF16 = _DT[torch.float32], _DT[torch.bfloat16]
_SIGNATURES = {
    "nf_adapter_add": [_P] * 8 + [_I] * 6 + [_P, _I, _I, _P],
    "nf_adapter_linear": [_P] * 8 + [_I] * 6 + [_P, _I, _P],
    "nf_adapter_rows_f32": [_P] * 8 + [_I] * 6 + [_P, _P],
    "nf_append_history": [_P] * 4 + [_I] * 3 + [_P],
    "nf_adapter_scratch": [_I] * 3,
    "nf_logit_rules": [_P] * 11 + [_I] + [_P] * 2 + [_I] * 7 + [_P],
}
_functions = {}
_slices = {}            # widths -> (their ends for the C call, how many, their sum)
_used = False           # whether any of these kernels was called: until then there is no status to read


def _function(name: str):
    f = _functions.get(name)
    if f is None:
        f = getattr(_lib.load(), name)
        f.argtypes = _SIGNATURES[name]
        if name == "nf_adapter_scratch":
            f.restype = ctypes.c_longlong
        _functions[name] = f
    return f


def _begin(name: str):
    """The C function, about to be called."""
    global _used
    _used = True
    _lib.count_launches(1)
    return _functions.get(name) or _function(name)


def _failed(name: str) -> None:
    raise _lib.KernelError(f"{name}: {_lib.load().nf_last_error().decode(errors='replace')}")


def _stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _parts(widths: Sequence[int]) -> Tuple[ctypes.Array, int, int]:
    """The ends of stacked parts as the kernels take them, their number and the last end; no parts where a width is none."""
    key = tuple(widths)
    got = _slices.get(key)
    if got is None:
        ends, e = (_I * max(1, len(key)))(), 0
        ok = all(int(v) > 0 for v in key)
        for i, v in enumerate(key if ok else ()):
            e += int(v)
            ends[i] = e
        got = (ends, len(key) if ok else 0, e)
        if len(_slices) < 1024:
            _slices[key] = got
    return got


def adapter_rank(rank: int) -> int:
    """The rank that a pool of adapters of up to `rank` is laid out for."""
    for r in ADAPTER_RANKS:
        if 1 <= rank <= r:
            return r
    raise ValueError(f"adapter rank {rank} is not supported (1..{ADAPTER_RANKS[-1]})")


def _overlap(s: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    p, q = s.data_ptr(), t.data_ptr()
    return p < q + t.numel() * t.element_size() and q < p + s.numel() * s.element_size()


def _refuse_adapter(x, w, a, b, scale, ids, widths, out, out_dtype) -> None:
    """Says what is wrong with the operands of adapter_linear."""
    _chk(x, "x")
    for t, name in ((w, "w"), (a, "a"), (b, "b"), (scale, "scale"), (ids, "ids"), (out, "out")):
        if t is not None and t.device != x.device:
            raise ValueError(f"adapter_linear: {name} lies on {t.device}, x on {x.device}")
    _chk(w, "w", x.dtype); _chk(a, "a", x.dtype); _chk(b, "b", x.dtype)
    _chk(scale, "scale", torch.float32); _chk(ids, "ids", torch.int32)
    _dt(x)
    if x.dim() != 2 or w.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError("adapter_linear takes x [T, K], w [N, K], a [n, slices * R, K] and b [n, N, R]")
    T, K = x.shape
    N, n, R, S = w.shape[0], b.shape[0], b.shape[2], len(widths)
    if w.shape[1] != K:
        raise ValueError(f"adapter_linear: x has {K} columns, w has {w.shape[1]}")
    if not 1 <= S <= MAX_ADAPTER_SLICES or min(widths) < 1 or sum(widths) != N:
        raise ValueError(f"adapter_linear: widths {list(widths)} are not 1 to {MAX_ADAPTER_SLICES} positive parts of {N} features")
    if R not in ADAPTER_RANKS:
        raise ValueError(f"adapter_linear: rank {R} is not one of {ADAPTER_RANKS}; pad with zeros")
    if n < 1 or K < 1 or a.shape != (n, S * R, K) or b.shape[1] != N:
        raise ValueError(f"adapter_linear: a {tuple(a.shape)} and b {tuple(b.shape)} do not fit {S} parts, rank {R} and w "
                         f"{tuple(w.shape)}")
    if scale.numel() != n or ids.numel() != T:
        raise ValueError(f"adapter_linear: scale {tuple(scale.shape)} and ids {tuple(ids.shape)} for {n} adapters and {T} rows")
    if out_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"adapter_linear: out_dtype is {out_dtype}, not {x.dtype} or {torch.float32}")
    if out is not None:
        _chk(out, "out", out_dtype)
        if out.shape != (T, N):
            raise ValueError(f"adapter_linear: out is {tuple(out.shape)}, not {(T, N)}")
        if T and _overlap(x, out):
            raise ValueError("adapter_linear: out shares memory with x")
    for t, name in ((x, "x"), (w, "w"), (a, "a"), (b, "b"), (out, "out")):
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"adapter_linear: {name} does not start on a 16-byte boundary")


def adapter_linear(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, ids: torch.Tensor,
                   widths: Optional[Sequence[int]] = None, out: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [T, K] times w [N, K] transposed, plus every row's adapter -> [T, N]:

        out[t] = x[t] w^T + scale[i] (x[t] a[i]^T) b[i]^T,   i = ids[t];   ids[t] = -1: no adapter

    `widths`: the parts that the N features are stacked of (query, key and value, say), each with rows of `a` of its own;
    [N] if left out.  a [n, len(widths) * R, K] (the parts' rows one after the other), b [n, N, R], R one of
    `ADAPTER_RANKS`, scale float32 [n], ids int32 [T].  Sums are float32 and rounded once, to x's type, or
    left as they are with `out_dtype` float32.  An id outside
    [-1, n) is served like -1 and, from n on, reported by `check_status`.  The weights of all adapters have to be finite:
    rows of several requests share a product, in which another request's adapter is multiplied by zero."""
    if widths is None:
        widths = (w.shape[0],)
    dtype, dev = x.dtype, x.get_device()
    if out_dtype is None:
        out_dtype = dtype
    xs, ws, bs = x.shape, w.shape, b.shape
    ends, S, total = _parts(widths)
    if not (dev >= 0 and len(xs) == 2 and len(ws) == 2 and len(bs) == 3 and (dtype is torch.bfloat16 or dtype is torch.float32)
            and w.dtype is dtype and a.dtype is dtype and b.dtype is dtype and scale.dtype is torch.float32
            and ids.dtype is torch.int32 and w.get_device() == dev and a.get_device() == dev and b.get_device() == dev
            and scale.get_device() == dev and ids.get_device() == dev and x.is_contiguous() and w.is_contiguous()
            and a.is_contiguous() and b.is_contiguous() and scale.is_contiguous() and ids.is_contiguous()):
        _refuse_adapter(x, w, a, b, scale, ids, widths, out, out_dtype)
    T, K = xs
    N, (n, b_rows, R) = ws[0], bs
    if not (K > 0 and ws[1] == K and n > 0 and b_rows == N and R in ADAPTER_RANKS and 1 <= S <= MAX_ADAPTER_SLICES
            and total == N and a.shape == (n, S * R, K) and scale.numel() == n and ids.numel() == T
            and (out_dtype is dtype or out_dtype is torch.float32)):
        _refuse_adapter(x, w, a, b, scale, ids, widths, out, out_dtype)
    if out is None:
        out = x.new_empty((T, N)) if out_dtype is dtype else x.new_empty((T, N), dtype=out_dtype)
    elif not (out.dtype is out_dtype and out.get_device() == dev and out.is_contiguous() and out.shape == (T, N)) or _overlap(x, out):
        _refuse_adapter(x, w, a, b, scale, ids, widths, out, out_dtype)
    if T == 0:
        return out
    px, pw, pa, pb, po = x.data_ptr(), w.data_ptr(), a.data_ptr(), b.data_ptr(), out.data_ptr()
    if (px | pw | pa | pb | po) & 15:
        _refuse_adapter(x, w, a, b, scale, ids, widths, out, out_dtype)
    bf16 = dtype is torch.bfloat16
    if TUNING["adapter"] == "auto" and (K % 8 == 0 if bf16 else K % 4 == 0 and T <= TUNING["adapter_f32_max_rows"]):
        # (h of a few rows lies row by row, see nf_adapter_scratch)
        h = scale.new_empty(_function("nf_adapter_scratch")(T, S * R, n) if bf16 and T > 16 else T * S * R)
        if bf16:
            if _begin("nf_adapter_linear")(px, pw, pa, pb, scale.data_ptr(), ids.data_ptr(), h.data_ptr(), po, T, N, K, R, n, S, ends,
                                           _BF16 if out_dtype is dtype else _F32, _stream(dev)):
                _failed("nf_adapter_linear")
        elif _begin("nf_adapter_rows_f32")(px, pw, pa, pb, scale.data_ptr(), ids.data_ptr(), h.data_ptr(), po, T, N, K, R, n, S, ends,
                                           _stream(dev)):
            _failed("nf_adapter_rows_f32")
        return out
    # many float32 rows, or rows that TMA cannot fetch: the shared product by itself, the adapters added to its float32 sums
    h = scale.new_empty(T * S * R)
    z = linear(x, w, out_dtype=torch.float32)
    if _begin("nf_adapter_add")(px, pa, pb, scale.data_ptr(), ids.data_ptr(), z.data_ptr(), h.data_ptr(), po, T, N, K, R, n, S, ends, _dt(x),
                                _dt(out), _stream(dev)):
        _failed("nf_adapter_add")
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
    if tokens.numel() and _begin("nf_append_history")(history.data_ptr(), slots.data_ptr(), positions.data_ptr(), tokens.data_ptr(),
                                                      tokens.numel(), history.shape[0], history.shape[1], _stream(history.get_device())):
        _failed("nf_append_history")


def _rows_apart(t: torch.Tensor, R: int, V: int) -> int:
    """Elements between two rows of [R, V], or -1 where the rows are not runs of their own, or too far apart for the kernel's
    32-bit step."""
    step, one = t.stride()
    if R <= 1:
        step = V
    return step if (one == 1 or V <= 1) and V <= step < 1 << 31 else -1


def _clash(p: int, apart: int, q: int, apart_q: int, R: int, V: int) -> bool:
    """Whether float32 rows at p and at q share memory otherwise than as the same rows."""
    if (p == q and (apart == apart_q or R == 1)) or p + 4 * ((R - 1) * apart + V) <= q or q + 4 * ((R - 1) * apart_q + V) <= p:
        return False
    between = (q - p) // 4 % apart                    # rows of one tensor may lie between those of the other
    return apart != apart_q or not V <= between <= apart - V


def _refuse_logits(logits, history, slots, lengths, starts, penalties, tokens, bias, mask, out) -> None:
    """Says what is wrong with the operands of adjust_logits."""
    _chk(logits, "logits", torch.float32, contiguous=False); _chk(history, "history", torch.int32)
    if logits.dim() != 2 or history.dim() != 2:
        raise ValueError("adjust_logits takes logits [R, V] and history [slots, capacity]")
    R, V = logits.shape
    _chk(penalties, "penalties", torch.float32)
    if penalties.numel() != 3 * R:
        raise ValueError(f"adjust_logits: penalties are {tuple(penalties.shape)}, not {(R, 3)}")
    lists = [(slots, "slots", R), (lengths, "lengths", R), (starts, "starts", R)]
    if tokens is not None:
        lists.append((tokens, "tokens", R))
    others = [history, penalties]
    if bias is not None:
        offsets, ids, values = bias
        lists += [(offsets, "bias offsets", R + 1), (ids, "bias ids", ids.numel())]
        _chk(values, "bias values", torch.float32)
        if values.numel() != ids.numel():
            raise ValueError(f"adjust_logits: {tuple(ids.shape)} bias ids, {tuple(values.shape)} values")
        others.append(values)
    if mask is not None:
        bits, index = mask
        lists.append((index, "mask index", R))
        _chk(bits, "mask bits", torch.int32)
        if bits.dim() != 2 or bits.shape[0] < 1 or bits.shape[1] != (V + 31) // 32:
            raise ValueError(f"adjust_logits: mask bits are {tuple(bits.shape)}, not [M, {(V + 31) // 32}]")
        others.append(bits)
    for t, name, n in lists:
        _chk(t, name, torch.int32)
        if t.numel() != n:
            raise ValueError(f"adjust_logits: {name} are {tuple(t.shape)}, not {(n,)}")
    if out is not None:
        _chk(out, "out", torch.float32, contiguous=False)
        if out.shape != (R, V):
            raise ValueError(f"adjust_logits: out is {tuple(out.shape)}, not {(R, V)}")
        others.append(out)
    for t in others + [v[0] for v in lists]:
        if t.device != logits.device:
            raise ValueError(f"adjust_logits: a tensor lies on {t.device}, the logits on {logits.device}")
    for t, name in ((logits, "logits"), (out, "out")):
        if t is not None and R and V and _rows_apart(t, R, V) < 0:
            raise ValueError(f"adjust_logits: the rows of {name} must be runs of their own, less than 2^31 apart, got strides {t.stride()}")
    if out is not None and R and V and _clash(logits.data_ptr(), _rows_apart(logits, R, V), out.data_ptr(), _rows_apart(out, R, V), R, V):
        raise ValueError("adjust_logits: out shares memory with the logits without being the logits")
    if history.shape[0] < 1 or history.shape[1] < 4 or history.shape[1] % 4 or history.data_ptr() % 16:
        raise ValueError(f"adjust_logits: history is {tuple(history.shape)}; its capacity must be a multiple of 4, its start a "
                         f"16-byte boundary")


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
    lengths[r] - 1; left out, the log holds it already.  No two rows may write to one slot.  `bias` = (offsets int32
    [R + 1], ids int32, values float32): the entries of row r are those from offsets[r] to offsets[r + 1], each id once.
    `mask` = (bits int32 [M, (V + 31) // 32], index int32 [R]): bit i % 32 of word i // 32 of row index[r] is set where
    token i is allowed; index -1: no mask.  A row whose mask allows nothing is -inf throughout.  `out` may be `logits`
    itself, but not overlap it otherwise.  A slot, a length or a mask row outside its tensor changes that row as if it had no tokens or no mask; a start
    counts as the nearest place from 0 to the length, an offset as the nearest entry: all are reported by `check_status`."""
    dev = logits.get_device()
    ls, hs = logits.shape, history.shape
    good = (dev >= 0 and len(ls) == 2 and len(hs) == 2 and logits.dtype is torch.float32 and history.dtype is torch.int32
            and slots.dtype is torch.int32 and lengths.dtype is torch.int32 and starts.dtype is torch.int32
            and penalties.dtype is torch.float32 and history.get_device() == dev and slots.get_device() == dev
            and lengths.get_device() == dev and starts.get_device() == dev and penalties.get_device() == dev
            and history.is_contiguous() and slots.is_contiguous() and lengths.is_contiguous() and starts.is_contiguous()
            and penalties.is_contiguous())
    R, V = ls if good else (0, 0)
    p_history = history.data_ptr()
    good = (good and slots.numel() == R and lengths.numel() == R and starts.numel() == R and penalties.numel() == 3 * R
            and hs[0] > 0 and hs[1] > 0 and hs[1] % 4 == 0 and p_history % 16 == 0)
    if good and tokens is not None:
        good = tokens.dtype is torch.int32 and tokens.get_device() == dev and tokens.is_contiguous() and tokens.numel() == R
    p_off = p_ids = p_values = p_bits = p_index = None
    n_bias = n_masks = 0
    if good and bias is not None:
        offsets, ids, values = bias
        n_bias = ids.numel()
        good = (offsets.dtype is torch.int32 and ids.dtype is torch.int32 and values.dtype is torch.float32
                and offsets.get_device() == dev and ids.get_device() == dev and values.get_device() == dev
                and offsets.is_contiguous() and ids.is_contiguous() and values.is_contiguous() and offsets.numel() == R + 1
                and values.numel() == n_bias)
        p_off, p_ids, p_values = offsets.data_ptr(), ids.data_ptr(), values.data_ptr()
    if good and mask is not None:
        bits, index = mask
        n_masks = bits.shape[0] if bits.dim() == 2 else 0
        good = (bits.dtype is torch.int32 and index.dtype is torch.int32 and bits.get_device() == dev and index.get_device() == dev
                and bits.is_contiguous() and index.is_contiguous() and n_masks > 0 and bits.shape[1] == (V + 31) // 32
                and index.numel() == R)
        p_bits, p_index = bits.data_ptr(), index.data_ptr()
    if good and out is not None:
        good = out.dtype is torch.float32 and out.get_device() == dev and out.shape == ls
    if not good:
        _refuse_logits(logits, history, slots, lengths, starts, penalties, tokens, bias, mask, out)
    given = out is not None
    if given:
        apart_out = _rows_apart(out, R, V)
    else:
        out = penalties.new_empty((R, V))
        apart_out = V
    if R == 0 or V == 0:
        return out
    apart = _rows_apart(logits, R, V)
    p_in, p_out = logits.data_ptr(), out.data_ptr()
    if apart < 0 or apart_out < 0 or (given and _clash(p_in, apart, p_out, apart_out, R, V)):
        _refuse_logits(logits, history, slots, lengths, starts, penalties, tokens, bias, mask, out)
    if _begin("nf_logit_rules")(p_in, p_out, p_history, slots.data_ptr(), lengths.data_ptr(), starts.data_ptr(),
                                None if tokens is None else tokens.data_ptr(), penalties.data_ptr(), p_off, p_ids, p_values, n_bias, p_bits,
                                p_index, n_masks, R, V, apart, apart_out, hs[0], hs[1], _stream(dev)):
        _failed("nf_logit_rules")
    return out


def request_status() -> int:
    """0, or what these kernels met since the last call: 1 to 14 a bounded wait that ran out, 101 + a row whose adapter was
    outside the pool, 10000001 + a row whose log, mask or biases did not fit.  Synchronises the device; where none of them was ever
    called there is nothing to read."""
    if not _used:
        return 0
    lib = _lib.load()
    tc, ad, ru = int(lib.nf_adapter_tc_status()), int(lib.nf_adapter_index_status()), int(lib.nf_rules_index_status())
    return tc if tc else (100 + ad if ad else (10000000 + ru if ru else 0))
