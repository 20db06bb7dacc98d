"""Python faces of the kernels by which a request tries several continuations at once: attention of a tree of drafted
tokens over its cache, which of them the model's probabilities let stand, the cache's rows of those moved up behind what
the request held, and pages copied for a request that is forked.

A step's nodes are rows, a request's rows lie together: `row0` int32 [S + 1] says where each request's begin.  Node 0 of a
request is its tree's root, the newest token that it has; the others are drafted.  Keys and values of node i go into the
request's pages at position lengths[s] + i, whatever its depth: `rope_append` turns them by their depth and takes these
positions as `places`.  Everything is on the device, so that a captured step serves any trees.
"""

from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

from . import lib as _lib
from .ops import TUNING, _chk, _dt, check_head_dim

__all__ = ["MAX_TREE_NODES", "MAX_VERIFY_NODES", "compact_cache", "copy_pages", "draft_status", "tree_attention", "verify_drafts"]

MAX_TREE_NODES = 256          # nodes of a request that tree attention takes
MAX_VERIFY_NODES = 1024       # ... and verification
MAX_TREE_CONTEXT = 1 << 30
# of a scale, with which the kernels multiply as a float32 number: beyond, it or its product with log2(e) is 0 (which a hidden
# score of -inf must not meet), infinite, or has lost bits
LEAST_SCALE, MOST_SCALE = 2.0 ** -126, 2.0 ** 126

_I, _L, _P = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p
_SIGNATURES = {
    "nf_tree_attention_plan": [_I] * 8 + [_L] + [_I] * 3,
    "nf_tree_attention_workspace": [_L] + [_I] * 5,
    "nf_tree_attention": [_P],
    "nf_verify_drafts": [_P, _L, _P, _L] + [_P] * 7 + [_I] * 4 + [_P],
    "nf_compact_cache": [_P, _L] + [_I] * 5 + [_P, _I] + [_P] * 3 + [_I] * 2 + [_P],
    "nf_copy_pages": [_P, _L] + [_I] * 5 + [_P] * 3 + [_I, _P],
}
_TREE_CALL = struct.Struct("=20qd2q")          # TreeCall of tree_attention.cu
_plans = {}             # sizes -> how a call of these is served, as nf_tree_attention_plan says, and its workspace
_int32, _float32 = torch.int32, torch.float32
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_functions = {}
_used = False           # whether any of these kernels was called: until then there is no status to read


def _function(name: str):
    f = _functions.get(name)
    if f is None:
        f = getattr(_lib.load(), name)
        f.argtypes = _SIGNATURES[name]
        if name in ("nf_tree_attention_plan", "nf_tree_attention_workspace"):
            f.restype = _L
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


def _ints(what: str, device, **tensors) -> None:
    """Refuses index tensors that are not contiguous int32 ones on `device`."""
    for name, t in tensors.items():
        _chk(t, name, torch.int32)
        if t.device != device:
            raise ValueError(f"{what}: {name} lies on {t.device}, not on {device}")


def _same_memory(s: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether the memory that two tensors span overlaps."""
    def span(v):
        return v.data_ptr(), v.data_ptr() + v.element_size() * (1 + sum((n - 1) * d for n, d in zip(v.shape, v.stride())))
    (a, b), (c, d) = span(s), span(t)
    return s.numel() > 0 and t.numel() > 0 and a < d and c < b


def _refuse_tree(qkv, Hq, Hkv, D, pages, block_table, page_size, lengths, row0, mask, max_context, scale, out) -> None:
    """Says what is wrong with the operands of tree_attention."""
    what = "tree_attention"
    _chk(qkv, "qkv", contiguous=False)
    _dt(qkv)
    _chk(pages, "pages", qkv.dtype)
    check_head_dim(D)
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"{what}: {Hq} query heads do not divide into {Hkv} groups")
    if qkv.dim() != 2 or qkv.shape[1] < Hq * D or qkv.stride(1) != 1 or (qkv.shape[0] > 1 and qkv.stride(0) < qkv.shape[1]):
        raise ValueError(f"{what}: qkv is {tuple(qkv.shape)} with strides {qkv.stride()}; rows of {Hq} heads of {D} are wanted")
    if page_size < 1 or pages.dim() != 5 or pages.shape[1:] != (2, Hkv, page_size, D) or not 1 <= pages.shape[0] < 1 << 31:
        raise ValueError(f"{what}: pages are {tuple(pages.shape)}, not [pages, 2, {Hkv}, {page_size}, {D}]")
    if pages.device != qkv.device:
        raise ValueError(f"{what}: pages lie on {pages.device}, qkv on {qkv.device}")
    _ints(what, qkv.device, block_table=block_table, lengths=lengths, row0=row0, mask=mask)
    T = qkv.shape[0]
    if block_table.dim() != 2 or block_table.shape[1] < 1 or lengths.shape != block_table.shape[:1] or row0.shape != (lengths.numel() + 1,):
        raise ValueError(f"{what}: block table {tuple(block_table.shape)}, lengths {tuple(lengths.shape)} and row0 {tuple(row0.shape)} "
                         f"are not of one number of requests (row0: one more)")
    if mask.dim() != 2 or mask.shape[0] != T or not 1 <= mask.shape[1] <= MAX_TREE_NODES // 32:
        raise ValueError(f"{what}: mask is {tuple(mask.shape)}, not [{T}, 1 to {MAX_TREE_NODES // 32}]")
    if not LEAST_SCALE <= scale <= MOST_SCALE:
        raise ValueError(f"{what}: scale={scale} must be positive, within 2^-126 and 2^126")
    if not 1 <= max_context <= MAX_TREE_CONTEXT:
        raise ValueError(f"{what}: max_context={max_context} is not within 1 and {MAX_TREE_CONTEXT}")
    if pages.data_ptr() % 16:
        raise ValueError(f"{what}: pages do not start on a 16-byte boundary")
    if out is not None:
        _chk(out, "out", qkv.dtype)
        if out.shape != (T, Hq * D) or out.device != qkv.device:
            raise ValueError(f"{what}: out is {tuple(out.shape)} on {out.device}, not {(T, Hq * D)} on {qkv.device}")
        for t, name in ((qkv, "qkv"), (pages, "pages")):
            if _same_memory(out, t):
                raise ValueError(f"{what}: out shares memory with {name}")


def tree_attention(qkv: torch.Tensor, Hq: int, Hkv: int, D: int, pages: torch.Tensor, block_table: torch.Tensor, page_size: int,
                   lengths: torch.Tensor, row0: torch.Tensor, mask: torch.Tensor, max_context: int, scale: float,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the (rotated) queries of trees of drafted tokens over the cache -> [T, Hq * D].

    qkv [T, at least Hq * D] (rows may lie further apart): queries in the first columns.  Request s holds lengths[s] keys;
    its rows row0[s] .. row0[s + 1] - 1 are its nodes, whose keys and values are in its pages already, node i's at position
    lengths[s] + i.  A row sees all keys that the request held, and node k's where bit k % 32 of word k // 32 of its mask
    (int32 [T, words], words for as many nodes as a request may have) is set: its ancestors and itself, as a rule, but any
    set will do.  A row that sees nothing is zero.  pages [pages, 2, Hkv, page_size, D], block_table int32 [S, width];
    `max_context`: what lengths[s] and a request's nodes add up to at most.  All of a page's rows must hold finite numbers,
    as they do in a cache manager's pool.

    Rows that belong to no request stay as they were in `out`.  Rows, lengths or nodes outside the bounds count as if they
    ended there, keys whose page is not in the pool as if no row saw them; both are reported by `check_status`."""
    dev, dtype = qkv.get_device(), qkv.dtype
    qs, bs, ms, ps = qkv.shape, block_table.shape, mask.shape, pages.shape
    good = (dev >= 0 and len(qs) == 2 and len(bs) == 2 and len(ms) == 2 and len(ps) == 5 and (dtype is torch.bfloat16 or dtype is _float32)
            and pages.dtype is dtype and block_table.dtype is _int32 and lengths.dtype is _int32 and row0.dtype is _int32 and mask.dtype is _int32
            and pages.get_device() == dev and block_table.get_device() == dev and lengths.get_device() == dev and row0.get_device() == dev
            and mask.get_device() == dev and pages.is_contiguous() and block_table.is_contiguous() and lengths.is_contiguous()
            and row0.is_contiguous() and mask.is_contiguous() and Hkv > 0 and Hq > 0 and Hq % Hkv == 0 and D % 16 == 0 and 16 <= D <= 256
            and page_size > 0 and 1 <= max_context <= MAX_TREE_CONTEXT and LEAST_SCALE <= scale <= MOST_SCALE)
    if good:
        (T, width), (S, table_width), (rows, words), (n_pages, two, heads, size, dim) = qs, bs, ms, ps
        step, one = qkv.stride()
        if T <= 1:
            step = -(-width // 8) * 8
        p_pages = pages.data_ptr()
        good = (width >= Hq * D and one == 1 and step >= width and 1 <= n_pages < 1 << 31 and two == 2 and heads == Hkv and size == page_size
                and dim == D and table_width > 0 and lengths.shape == (S,) and row0.shape == (S + 1,) and rows == T
                and 1 <= words <= MAX_TREE_NODES // 32 and p_pages % 16 == 0)
    if not good or out is not None:
        _refuse_tree(qkv, Hq, Hkv, D, pages, block_table, page_size, lengths, row0, mask, max_context, scale, out)
        if dev != _current_device():
            with torch.cuda.device(dev):
                return tree_attention(qkv, Hq, Hkv, D, pages, block_table, page_size, lengths, row0, mask, max_context, scale, out)
    elif dev != _current_device():
        with torch.cuda.device(dev):
            return tree_attention(qkv, Hq, Hkv, D, pages, block_table, page_size, lengths, row0, mask, max_context, scale)
    if out is None:
        out = qkv.new_empty((T, Hq * D))
    if T == 0 or S == 0:
        return out
    p_q, p_out = qkv.data_ptr(), out.data_ptr()
    code = 1 if dtype is torch.bfloat16 else 0
    key = (S, T, Hq, Hkv, D, page_size, n_pages, words, max_context, code, (p_q | p_out | 2 * step) & 15 == 0, TUNING["tree_attention"])
    plan = _plans.get(key)
    if plan is None:
        form = key[-1]
        plan = _function("nf_tree_attention_plan")(-1 if form == "auto" else form, code, S, T, Hq, Hkv, D, page_size, n_pages, words, max_context, key[-2])
        plan = plan, _function("nf_tree_attention_workspace")(plan, S, T, Hq, D, max_context)
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    plan, floats = plan
    # (kept until the call has been made; what comes after it on the stream may have the memory)
    ws = lengths.new_empty(floats) if floats else None
    if _begin("nf_tree_attention")(_TREE_CALL.pack(p_q, step, p_pages, block_table.data_ptr(), table_width, lengths.data_ptr(), row0.data_ptr(),
                                                   mask.data_ptr(), words, p_out, 0 if ws is None else ws.data_ptr(), S, T, Hq, Hkv, D, page_size,
                                                   n_pages, max_context, plan, scale, code, _raw_stream(dev))):
        _failed("nf_tree_attention")
    return out


def _rows_apart(t: torch.Tensor, T: int, V: int) -> int:
    """Numbers between two rows of [T, V], or -1 where the rows are not runs of their own."""
    step, one = t.stride()
    if T <= 1:
        step = V
    return step if (one == 1 or V <= 1) and step >= V else -1


def _refuse_verify(probs, tokens, parents, row0, draws, most, draft) -> None:
    """Says what is wrong with the operands of verify_drafts."""
    what = "verify_drafts"
    _chk(probs, "probs", torch.float32, contiguous=False)
    if probs.dim() != 2 or probs.shape[1] < 1:
        raise ValueError(f"{what}: probs are {tuple(probs.shape)}, not [rows, vocabulary]")
    T, V = probs.shape
    dev = probs.device
    _ints(what, dev, tokens=tokens, parents=parents, row0=row0)
    _chk(draws, "draws", torch.float32)
    if draws.device != dev:
        raise ValueError(f"{what}: draws lie on {draws.device}, not on {dev}")
    for t, name in ((tokens, "tokens"), (parents, "parents"), (draws, "draws")):
        if t.shape != (T,):
            raise ValueError(f"{what}: {name} are {tuple(t.shape)}, not {(T,)}")
    if row0.dim() != 1 or row0.numel() < 1:
        raise ValueError(f"{what}: row0 is {tuple(row0.shape)}, not [requests + 1]")
    if not 1 <= most <= MAX_VERIFY_NODES:
        raise ValueError(f"{what}: most={most} is not within 1 and {MAX_VERIFY_NODES}")
    if draft is not None:
        _chk(draft, "draft", torch.float32, contiguous=False)
        if draft.device != dev or draft.shape != (T, V):
            raise ValueError(f"{what}: draft is {tuple(draft.shape)} on {draft.device}, not {(T, V)} on {dev}")
    for t, name in ((probs, "probs"), (draft, "draft")):
        if t is not None and _rows_apart(t, T, V) < 0:
            raise ValueError(f"{what}: the rows of {name} must be runs of their own, got strides {t.stride()}")
    if row0.numel() > 1 and not T:
        raise ValueError(f"{what}: {row0.numel() - 1} requests without a row")


def verify_drafts(probs: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, row0: torch.Tensor, draws: torch.Tensor, most: int,
                  draft: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which drafted tokens stand, and the token after them -> (accepted int32 [S], path int32 [S, most], said int32
    [S, most + 1]).

    probs float32 [T, V] (rows may lie further apart): row t is the model's distribution behind node t's token.  Rows
    row0[s] .. row0[s + 1] - 1 are the nodes of request s (1 to `MAX_VERIFY_NODES`); node i's token is tokens[row0[s] + i],
    its parent, a node before it, parents[row0[s] + i] (the root's is not read).  draws float32 [T] are uniform numbers in
    [0, 1).  draft float32 [T, V]: the distributions that the tokens were drawn from, row t that of node t's; left out,
    drafted tokens stand for themselves (they were looked up, or are a model's likeliest).

    From v = 0 on, with r = probs[v] and z = 1, v's children c are asked in ascending order: where
    draws[c] z draft[c][x_c] < r[x_c] (left out: draws[c] z < r[x_c]), c is accepted and takes v's place; else
    r = max(r - z draft[c], 0) and z = sum(r) (left out: z -= r[x_c], r[x_c] = 0).  Where no child is left, or `most` are
    accepted, the next token is the lowest whose running sum of r passes draws[root] sum(r).  Tokens are then distributed as
    the model's own, one after the other.  Sums are 64 bits wide.

    `path[s]` lists the accepted nodes, `said[s]` their tokens and the next one, both with -1 behind; accepted[s] counts
    the drafted ones.  What is no positive number counts as a probability of 0; a row that holds nothing, or
    something infinite, gives -1.  Nodes whose token or parent makes no sense are nobody's children.  Both are reported by
    `check_status`."""
    dev, shape = probs.get_device(), probs.shape
    good = (dev >= 0 and len(shape) == 2 and shape[1] > 0 and probs.dtype is _float32 and draws.dtype is _float32 and tokens.dtype is _int32
            and parents.dtype is _int32 and row0.dtype is _int32 and tokens.get_device() == dev and parents.get_device() == dev
            and row0.get_device() == dev and draws.get_device() == dev and tokens.is_contiguous() and parents.is_contiguous()
            and row0.is_contiguous() and draws.is_contiguous() and row0.dim() == 1 and tokens.dim() == 1 and parents.dim() == 1
            and draws.dim() == 1 and 1 <= most <= MAX_VERIFY_NODES)
    if good:
        T, V = shape
        S = row0.numel() - 1
        probs_ld, draft_ld, p_draft = _rows_apart(probs, T, V), 0, None
        good = tokens.numel() == T and parents.numel() == T and draws.numel() == T and S >= 0 and probs_ld >= 0 and (T > 0 or S == 0)
        if good and draft is not None:
            good = draft.dtype is _float32 and draft.get_device() == dev and draft.shape == shape
            if good:
                draft_ld, p_draft = _rows_apart(draft, T, V), draft.data_ptr()
                good = draft_ld >= 0
    if not good:
        _refuse_verify(probs, tokens, parents, row0, draws, most, draft)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return verify_drafts(probs, tokens, parents, row0, draws, most, draft)
    accepted, path, said = tokens.new_empty(S * (2 * most + 2)).split_with_sizes((S, S * most, S * (most + 1)))
    if S and _begin("nf_verify_drafts")(probs.data_ptr(), probs_ld, p_draft, draft_ld, tokens.data_ptr(), parents.data_ptr(), row0.data_ptr(),
                                        draws.data_ptr(), accepted.data_ptr(), path.data_ptr(), said.data_ptr(), S, T, V, most, _raw_stream(dev)):
        _failed("nf_verify_drafts")
    return accepted, path.view(S, most), said.view(S, most + 1)


def _refuse_pages(what: str, pages: torch.Tensor) -> None:
    """Says what is wrong with a cache group's pages."""
    _chk(pages, "pages", contiguous=False)
    if pages.dim() not in (3, 4, 5, 6):
        raise ValueError(f"{what}: pages are {tuple(pages.shape)}, not (layers,) pages, (2, heads,) page_size, width")
    layered = pages if pages.dim() in (4, 6) else pages.unsqueeze(0)
    if layered.numel() == 0:
        raise ValueError(f"{what}: pages are {tuple(pages.shape)}")
    if not layered[0].is_contiguous() or (layered.shape[0] > 1 and layered.stride(0) < layered[0].numel()):
        raise ValueError(f"{what}: a layer's pages must be contiguous, got strides {pages.stride()}")
    raise ValueError(f"{what}: rows of {layered.shape[-1]} numbers of {layered.element_size()} bytes, in pages {tuple(pages.shape)}")


def _pages(what: str, pages: torch.Tensor) -> Tuple[int, ...]:
    """(address, bytes between two layers, layers, pages, planes, page size, row bytes) of a cache group's pages: one layer's
    [pages, 2, heads, page_size, D] or [pages, page_size, width], or with the layers before that."""
    shape, size = pages.shape, pages.element_size()
    n = len(shape)
    if n == 6 or n == 5:
        planes = shape[-4] * shape[-3]
    elif n == 4 or n == 3:
        planes = 1
    else:
        _refuse_pages(what, pages)
    layers, P = (shape[0], shape[1]) if n % 2 == 0 else (1, shape[0])
    rows, width = shape[-2], shape[-1]
    layer = P * planes * rows * width
    apart = layer
    if pages.is_contiguous():
        good = True
    elif n % 2 == 0:
        apart = pages.stride(0) if layers > 1 else layer
        good = layers > 0 and pages[0].is_contiguous() and apart >= layer
    else:
        good = False
    row = width * size
    if not (good and pages.is_cuda and layer > 0 and layers > 0 and row % 2 == 0 and row < 1 << 31 and P < 1 << 31 and planes < 1 << 31
            and rows < 1 << 31 and layers < 1 << 31 and planes * rows * row < 1 << 40):
        _refuse_pages(what, pages)
    return pages.data_ptr(), apart * size, layers, P, planes, rows, row


def compact_cache(pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor) -> None:
    """In every layer of `pages`, the cache's rows of the nodes that were kept move up behind what their request held:

        row lengths[s] + 1 + j  takes the place of  row lengths[s] + path[s, j],    j < accepted[s]

    so that they lie as if they alone had been run behind the root, whose row, lengths[s], stays.  pages: a cache group's
    [layers, pages, 2, heads, page_size, D] or [layers, pages, page_size, width], or one layer's; block_table int32
    [S, width]; path int32 [S, most] (rising) and accepted int32 [S] as `verify_drafts` gives them.  No two requests may have
    a page that rows move in, so none is listed twice.  A request whose path does
    not rise keeps its rows as they are, a row whose page is not in the pool stays: both are reported by `check_status`."""
    shape, dev = _pages("compact_cache", pages), pages.get_device()
    ts, ps = block_table.shape, path.shape
    if not (block_table.dtype is _int32 and lengths.dtype is _int32 and path.dtype is _int32 and accepted.dtype is _int32
            and block_table.get_device() == dev and lengths.get_device() == dev and path.get_device() == dev and accepted.get_device() == dev
            and block_table.is_contiguous() and lengths.is_contiguous() and path.is_contiguous() and accepted.is_contiguous() and len(ts) == 2
            and len(ps) == 2 and ts[1] > 0 and lengths.dim() == 1 and lengths.numel() == ts[0] and accepted.shape == lengths.shape and ps[0] == ts[0]):
        _ints("compact_cache", pages.device, block_table=block_table, lengths=lengths, path=path, accepted=accepted)
        raise ValueError(f"compact_cache: block table {tuple(block_table.shape)}, lengths {tuple(lengths.shape)}, path {tuple(path.shape)} and "
                         f"accepted {tuple(accepted.shape)} are not of one number of requests")
    if dev != _current_device():
        with torch.cuda.device(dev):
            return compact_cache(pages, block_table, lengths, path, accepted)
    S, most = ps
    if S and most and _begin("nf_compact_cache")(*shape, block_table.data_ptr(), ts[1], lengths.data_ptr(), path.data_ptr(), accepted.data_ptr(), S,
                                                 most, _raw_stream(dev)):
        _failed("nf_compact_cache")


def copy_pages(pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
    """In every layer of `pages` (as `compact_cache` takes them), page dst[i] becomes page src[i]: its first rows[i] rows
    where `rows` is given, the others then stay.  src, dst and rows are int32 lists of one length; no page may be written
    twice, or be read and written.  An entry that is outside the pool, or has more rows than a page, is left out and
    reported by `check_status`."""
    shape, dev, n = _pages("copy_pages", pages), pages.get_device(), src.numel()
    if not (src.dtype is _int32 and dst.dtype is _int32 and src.get_device() == dev and dst.get_device() == dev and src.is_contiguous()
            and dst.is_contiguous() and src.dim() == 1 and dst.dim() == 1 and dst.numel() == n
            and (rows is None or (rows.dtype is _int32 and rows.get_device() == dev and rows.is_contiguous() and rows.dim() == 1 and rows.numel() == n))):
        _ints("copy_pages", pages.device, src=src, dst=dst, **({} if rows is None else {"rows": rows}))
        raise ValueError(f"copy_pages: src {tuple(src.shape)}, dst {tuple(dst.shape)}"
                         + ("" if rows is None else f" and rows {tuple(rows.shape)}") + " are not lists of one length")
    if dev != _current_device():
        with torch.cuda.device(dev):
            return copy_pages(pages, src, dst, rows)
    if n and _begin("nf_copy_pages")(*shape, src.data_ptr(), dst.data_ptr(), None if rows is None else rows.data_ptr(), n, _raw_stream(dev)):
        _failed("nf_copy_pages")


def draft_status() -> int:
    """0, or what these kernels met since the last call: 1000001 + a request whose lengths, rows or pages did not fit tree
    attention, 2000001 + one whose tree or probabilities made no sense to verification, 3000001 + a request or an entry whose
    path or pages did not fit a copy, 4000000 + a code of tree attention on tensor cores (2 to 11: a bounded wait that ran out,
    101 + a request that did not fit), 5000000 + one of its form for few pairs (1 and 2, 101 + a request).  Synchronises the device; where none was ever called there is nothing to read."""
    if not _used:
        return 0
    lib = _lib.load()
    for k, name in enumerate(("nf_tree_attention_status", "nf_verify_drafts_status", "nf_cache_pages_status",
                              "nf_tree_attention_tc_status", "nf_tree_attention_mma_status"), 1):
        v = int(getattr(lib, name)())
        if v:
            return k * 1000000 + v
    return 0
