"""What is timed of the operators by which a request tries several continuations at once: attention of a tree of drafted
tokens over the paged cache, the verification of those tokens against the model's probabilities, the cache's rows of the
path that was kept moved up behind what the request held, and pages copied for a request that is forked.

Four kinds of case.  "attention": one layer of a step in which every request brings a tree of drafted tokens behind its
newest one (node 0, the tree's root).  "verify": which drafted tokens stand, and the token after them.  "compact": after
that, the cache of all layers.  "copy": the pages that a fork cannot share, of all layers.
Head layouts, layer counts and vocabularies are those of the engine's main design at the two sizes that its benchmark
names, and generic ones.
"""

from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 151936
SMALL, LARGE = (16, 16, 128), (28, 4, 128)          # query heads, key heads and head size at the two sizes


# ---- the cases --------------------------------------------------------------------------------------------------

def _attention(name, requests, nodes, longest, heads, page_size=64, shape="tree", dtype="bfloat16"):
    """`requests` requests of up to `longest` tokens, each with a tree of up to `nodes` nodes, its root among them."""
    return {"name": name, "kind": "attention", "requests": requests, "nodes": nodes, "longest": longest, "heads": heads[0],
            "kv_heads": heads[1], "head_dim": heads[2], "page_size": page_size, "shape": shape, "dtype": dtype}


def _verify(name, requests, nodes, vocab, shape, draft):
    """`draft`: tokens were drawn from a draft model's probabilities; else they were looked up, and stand for themselves."""
    return {"name": name, "kind": "verify", "requests": requests, "nodes": nodes, "vocab": vocab, "shape": shape, "draft": draft}


def _compact(name, requests, nodes, longest, layers, kv_heads, head_dim, page_size=64, dtype="bfloat16"):
    return {"name": name, "kind": "compact", "requests": requests, "nodes": nodes, "longest": longest, "layers": layers,
            "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size, "dtype": dtype}


def _copy(name, pages, layers, kv_heads, head_dim, partial, page_size=64, dtype="bfloat16"):
    """`partial`: pages that are filled in part, as a fork's last ones are; else whole ones."""
    return {"name": name, "kind": "copy", "pages": pages, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim,
            "partial": partial, "page_size": page_size, "dtype": dtype}


def listed():
    return [
        # one chat, a few looked-up tokens in a row
        _attention("one chat, 8 in a row", 1, 8, 300, SMALL, shape="chain"),
        # one request at the larger size, a tree of an odd number of nodes
        _attention("one request, 27 nodes", 1, 27, 4097, LARGE),
        # a step of eight requests at the smaller size
        _attention("8 requests, 32 nodes", 8, 32, 8192, SMALL),
        # many requests with large trees at the larger size: the products' turn
        _attention("16 requests, 64 nodes", 16, 64, 16384, LARGE),
        # the all-32-bit path
        _attention("2 requests, float32", 2, 12, 1000, SMALL, dtype="float32"),
        # one chat with a few looked-up tokens
        _verify("one chain of 5", 1, 5, VOCAB, "chain", False),
        # trees from a draft model's best tokens, which stand for themselves
        _verify("8 trees of 32", 8, 32, VOCAB, "tree", False),
        # a full step of chains that a draft model has drawn
        _verify("64 chains of 6, drawn", 64, 6, VOCAB, "chain", True),
        # one request after its step
        _compact("one request kept", 1, 27, 700, 24, 16, 128),
        # a full step at the larger size
        _compact("64 requests kept", 64, 32, 150, 28, 4, 128),
        # one fork of a request
        _copy("one fork", 1, 24, 16, 128, True),
        # prompts copied whole for requests that go on without sharing
        _copy("160 whole pages", 160, 28, 4, 128, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    kind = rng.choice(["attention", "attention", "attention", "verify", "verify", "compact", "copy"])
    shape = rng.choice(["tree", "tree", "chain"])
    if kind == "attention":
        narrow = rng.random() < 0.2
        heads = rng.choice([SMALL, LARGE, (16, 4, 64), (8, 1, 128), (12, 12, 64), (32, 8, 128)])
        while True:
            requests, nodes, longest = _log(rng, 1, 4 if narrow else 32), _log(rng, 1, 24 if narrow else 100), _log(rng, 16, 4096 if narrow else 65536)
            if requests * nodes * longest * heads[0] * heads[2] <= 16 * 64 * 16384 * 28 * 128 // 2 and \
                    requests * longest * heads[1] * heads[2] <= 16 * 16384 * 512:
                break
        case = _attention("", requests, nodes, longest, heads, rng.choice([16, 32, 64, 64]), shape, "float32" if narrow else "bfloat16")
    elif kind == "verify":
        while True:
            requests, nodes, vocab = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1000, 160000)
            if requests * nodes * vocab <= 64 * 6 * VOCAB:
                break
        case = _verify("", requests, nodes, vocab, shape, rng.random() < 0.5)
    elif kind == "compact":
        while True:
            requests, nodes, longest, layers = _log(rng, 1, 64), _log(rng, 2, 64), _log(rng, 1, 700), _log(rng, 1, 28)
            kv_heads, head_dim = rng.choice([(16, 128), (4, 128), (4, 64), (2, 32)])
            if requests * (longest + nodes) * layers * kv_heads * head_dim <= 64 * 182 * 28 * 4 * 128:
                break
        case = _compact("", requests, nodes, longest, layers, kv_heads, head_dim, rng.choice([16, 32, 64]), rng.choice(["bfloat16", "bfloat16", "float32"]))
    else:
        while True:
            pages, layers = _log(rng, 1, 300), _log(rng, 1, 28)
            kv_heads, head_dim = rng.choice([(16, 128), (4, 128), (4, 64), (2, 32)])
            if pages * layers * kv_heads * head_dim <= 160 * 28 * 4 * 128:
                break
        case = _copy("", pages, layers, kv_heads, head_dim, rng.random() < 0.5, rng.choice([16, 32, 64]), rng.choice(["bfloat16", "bfloat16", "float32"]))
    del case["name"]
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tree(rnd, n, shape):
    """Parents of n nodes, level by level: a few tokens at the first, the likelier ones with more below them."""
    if shape == "chain":
        return list(range(-1, n - 1))
    parents, level = [-1], [0]
    while len(parents) < n:
        below = []
        for i, v in enumerate(level):
            for _ in range(min(n - len(parents), max(1 if i == 0 else 0, rnd.randint(1, 6) - i))):
                below.append(len(parents))
                parents.append(v)
        level = below
    return parents


def _trees(case, rnd):
    """Each request's parents, and where its nodes begin among all.  The first request has as many as there may be, the
    others down to half of that."""
    sizes = [case["nodes"] - 5 * s % (case["nodes"] // 2 + 1) for s in range(case["requests"])]
    trees, row0 = [_tree(rnd, n, case["shape"]) for n in sizes], [0]
    for n in sizes:
        row0.append(row0[-1] + n)
    return trees, row0


def _tables(lengths, page_size, rnd):
    """A block table of pages in any order for requests of so many tokens; the number of pages, which is what all of them
    would take at the longest one's length, and two more."""
    need = [-(-n // page_size) for n in lengths]
    pool = list(range(len(need) * max(need) + 2))
    rnd.shuffle(pool)
    table, at = [[-1] * max(need) for _ in need], 0
    for s, n in enumerate(need):
        table[s][:n] = pool[at:at + n]
        at += n
    return _ints(table), len(pool)


def prepare(case, seed):
    rnd = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)
    state = {"case": case}
    if case["kind"] == "attention":
        dtype, ps = getattr(torch, case["dtype"]), case["page_size"]
        Hq, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
        trees, row0 = _trees(case, rnd)
        longest = case["longest"]
        lengths = [longest] + [rnd.randint(longest // 2, longest) for _ in trees[1:]]
        words = (case["nodes"] + 31) // 32
        bits = []
        for parents in trees:
            seen = []
            for i, v in enumerate(parents):
                seen.append((seen[v] if v >= 0 else 0) | 1 << i)           # its ancestors and itself
            bits += [[(b >> 32 * w & 0xffffffff) - ((b >> 32 * w + 31 & 1) << 32) for w in range(words)] for b in seen]
        ends = [n + len(p) for n, p in zip(lengths, trees)]
        table, pages = _tables(ends, ps, rnd)
        state.update(qkv=normal(row0[-1], (Hq + 2 * Hkv) * D).to(dtype), pages=normal(pages, 2, Hkv, ps, D, dtype=dtype), table=table,
                     lengths=_ints(lengths), row0=_ints(row0), mask=_ints(bits), longest=max(ends), scale=1.5 / math.sqrt(D))
    elif case["kind"] == "verify":
        V = case["vocab"]
        trees, row0 = _trees(case, rnd)
        T = row0[-1]
        logits = normal(T, V) * 2.5
        probs = torch.softmax(logits * 1.4, -1)
        parent = torch.tensor([row0[s] + max(v, 0) for s, p in enumerate(trees) for v in p], device="cuda")
        # a draft model is near the target where it was trained well
        draft = torch.softmax(logits[parent] * 1.4 + normal(T, V) * 0.6, -1) if case["draft"] else None
        if case["draft"]:
            tokens = torch.multinomial(draft, 1, generator=gen)[:, 0]
        else:
            # siblings are a node's likeliest tokens, one after the other, or now and then one that was merely looked up
            rank, seen = [], {}
            for s, p in enumerate(trees):
                for v in p:
                    rank.append(seen.get((s, v), 0))
                    seen[s, v] = rank[-1] + 1
            best = torch.topk(probs[parent], max(rank) + 1, -1)[1]
            tokens = best.gather(1, torch.tensor(rank, device="cuda")[:, None])[:, 0]
            looked = torch.rand(T, generator=gen, device="cuda") < 0.2
            tokens = torch.where(looked, torch.randint(V, (T,), generator=gen, device="cuda"), tokens)
        state.update(probs=probs, draft=draft, tokens=tokens.to(torch.int32), parents=_ints([v for p in trees for v in p]), row0=_ints(row0),
                     draws=torch.rand(T, generator=gen, device="cuda"), most=max(1, case["nodes"] - 1), sizes=[len(p) for p in trees])
    elif case["kind"] == "compact":
        dtype, ps, R, most = getattr(torch, case["dtype"]), case["page_size"], case["requests"], case["nodes"] - 1
        lengths = [case["longest"]] + [rnd.randint(0, case["longest"]) for _ in range(R - 1)]
        table, pages = _tables([n + case["nodes"] for n in lengths], ps, rnd)
        kept, paths = [], []
        for s in range(R):
            n = min(most, rnd.choice([0, 1, 1, 2, 3, 4, 5, 7]) if s else 4)
            path, at = [], 0
            for j in range(n):
                # the first child of the first, or one of the tree's later nodes
                at = j + 1 if at == j and rnd.random() < 0.4 else rnd.randint(max(at, n) + 1, max(at, n) + 1 + (most - max(at, n)) // 2) \
                    if max(at, n) < most else 0
                if not at:
                    break
                path.append(at)
            kept.append(len(path))
            # (a later node's row lies behind every row that is written, so that the same call made again finds what it found before)
            if any(p != j + 1 and p <= len(path) for j, p in enumerate(path)):
                kept[-1], path = 0, []
            paths.append(path + [-1] * (most - len(path)))
        state.update(pages=normal(case["layers"], pages, 2, case["kv_heads"], ps, case["head_dim"], dtype=dtype), table=table,
                     lengths=_ints(lengths), path=_ints(paths), accepted=_ints(kept))
    else:
        dtype, ps, n = getattr(torch, case["dtype"]), case["page_size"], case["pages"]
        order = list(range(2 * n + 3))
        rnd.shuffle(order)
        state.update(pages=normal(case["layers"], len(order), 2, case["kv_heads"], ps, case["head_dim"], dtype=dtype), src=_ints(order[:n]),
                     dst=_ints(order[n:2 * n]), rows=_ints([rnd.randint(1, ps - 1) for _ in range(n)]) if case["partial"] else None)
    return state


# ---- the operators ------------------------------------------------------------------------------------------------

def _plain_attention(s):
    """All requests at once, each with as many keys and nodes as the longest has; what is not its own is masked."""
    c, qkv, lengths, row0 = s["case"], s["qkv"], s["lengths"].long(), s["row0"].long()
    ps, Hq, Hkv, D, N = c["page_size"], c["heads"], c["kv_heads"], c["head_dim"], c["nodes"]
    S, dev = lengths.numel(), qkv.device
    kv = s["pages"][s["table"].long().clamp_min(0)].float()                             # [S, pages, 2, Hkv, ps, D]
    k, v = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, S, Hkv, -1, D)
    row = row0[:-1, None] + torch.arange(N, device=dev)
    real = row < row0[1:, None]
    row = torch.where(real, row, 0)
    q = qkv[row][:, :, :Hq * D].float().view(S, N, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    scores = (q @ k.transpose(2, 3)).view(S, Hkv, Hq // Hkv, N, -1) * s["scale"]
    at = torch.arange(k.shape[2], device=dev) - lengths[:, None, None]                  # a key's place in the tree
    word = s["mask"][row].gather(2, (at // 32).clamp(0, s["mask"].shape[1] - 1).expand(S, N, -1))
    seen = (at < 0) | (at < 32 * s["mask"].shape[1]) & ((word >> (at % 32)) & 1 > 0)
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).view(S, Hkv, Hq // Hkv, N, D).permute(0, 3, 1, 2, 4).reshape(S, N, Hq * D)
    return o[real].to(qkv.dtype)


def _plain_verify(s):
    """Nodes in their order, all requests at once: a child of the node that its request has come to is accepted, or its part
    is taken off what is left of that node's probabilities.  (One node's turn decides whether the next one has one.)  In 64
    bits, as a draw may fall next to a border."""
    probs, row0, most, V = s["probs"], s["row0"].long(), s["most"], s["case"]["vocab"]
    S, dev = row0.numel() - 1, probs.device
    first, sizes = row0[:-1], row0[1:] - row0[:-1]
    at = torch.arange(S, device=dev)
    cur, left, mass = torch.zeros_like(first), probs[first].double(), torch.ones(S, dtype=torch.float64, device=dev)
    accepted, path = torch.zeros_like(first), torch.full((S, most + 1), -1, dtype=torch.int64, device=dev)
    tokens = path.clone()
    for i in range(1, max(s["sizes"])):
        row = torch.minimum(first + i, row0[1:] - 1)
        turn = (i < sizes) & (s["parents"][row] == cur)
        x = s["tokens"][row].long()
        have = left.gather(1, x[:, None])[:, 0]
        ask = s["draws"][row].double() * mass
        if s["draft"] is not None:
            ask = ask * s["draft"][row].gather(1, x[:, None])[:, 0].double()
        yes, no = turn & (ask < have), turn & ~(ask < have)
        path[at, torch.where(yes, accepted, most)] = torch.where(yes, i, path[:, most])
        tokens[at, torch.where(yes, accepted, most)] = torch.where(yes, x, tokens[:, most])
        accepted, cur = accepted + yes, torch.where(yes, i, cur)
        if s["draft"] is not None:
            rest = (left - mass[:, None] * s["draft"][row].double()).clamp_min(0)
        else:
            rest = left.scatter(1, x[:, None], 0.0)
        less = rest.sum(-1) if s["draft"] is not None else mass - have
        left = torch.where(yes[:, None], probs[row].double(), torch.where(no[:, None], rest, left))
        mass = torch.where(yes, 1.0, torch.where(no, less, mass))
    run = left.cumsum(-1)
    new = ((run > s["draws"][first].double()[:, None] * run[:, -1:]) & (left > 0)).long().argmax(-1)
    tokens[:, most] = -1
    tokens[at, accepted] = new
    small = lambda t: t.to(torch.int32)
    return {"accepted": small(accepted), "path": small(path[:, :most]), "tokens": small(tokens)}


def _plain_compact(s):
    pages, table, ps, most = s["pages"], s["table"].long(), s["case"]["page_size"], s["path"].shape[1]
    j = torch.arange(most, device=pages.device)[None, :]
    src = torch.where(j < s["accepted"][:, None], s["path"], j + 1) + s["lengths"][:, None]     # (rows that stay go where they are)
    dst = (j + 1 + s["lengths"][:, None]).expand_as(src)
    page = lambda at: table.gather(1, at.long() // ps)
    moved = pages[:, page(src), :, :, src.long() % ps]
    pages[:, page(dst), :, :, dst.long() % ps] = moved
    return pages


def _plain_copy(s):
    pages, src, dst = s["pages"], s["src"].long(), s["dst"].long()
    if s["rows"] is None:
        pages[:, dst] = pages[:, src]
    else:
        filled = torch.arange(s["case"]["page_size"], device=pages.device) < s["rows"][:, None]
        pages[:, dst] = torch.where(filled[None, :, None, None, :, None], pages[:, src], pages[:, dst])
    return pages


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"attention": _plain_attention, "verify": _plain_verify, "compact": _plain_compact, "copy": _plain_copy}[kind](s)
    from ninfer_amd_mi50_b200 import kernels
    c = s["case"]
    if kind == "attention":
        return kernels.tree_attention(s["qkv"], c["heads"], c["kv_heads"], c["head_dim"], s["pages"], s["table"], c["page_size"],
                                      s["lengths"], s["row0"], s["mask"], s["longest"], s["scale"])
    if kind == "verify":
        accepted, path, tokens = kernels.verify_drafts(s["probs"], s["tokens"], s["parents"], s["row0"], s["draws"], s["most"], s["draft"])
        return {"accepted": accepted, "path": path, "tokens": tokens}
    if kind == "compact":
        kernels.compact_cache(s["pages"], s["table"], s["lengths"], s["path"], s["accepted"])
    else:
        kernels.copy_pages(s["pages"], s["src"], s["dst"], s["rows"])
    return s["pages"]


# ---- what a pass cannot do without, and its outputs in 64 bits -----------------------------------------------------

def work(case):
    R = case.get("requests", 0)
    size = 4 if case.get("dtype") == "float32" else 2
    if case["kind"] == "attention":
        Hq, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
        nodes = case["nodes"] + (R - 1) * 0.75 * case["nodes"]
        keys = case["longest"] + case["nodes"] + (R - 1) * 0.75 * (case["longest"] + case["nodes"])
        return {"bytes": size * (2.0 * keys * Hkv * D + 2 * nodes * Hq * D), "flops": 4.0 * Hq * D * keys * nodes / R}
    if case["kind"] == "verify":
        return {"bytes": 4.0 * R * case["vocab"] * (2 if case["draft"] else 1), "flops": 2.0 * R * case["vocab"]}
    row = 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * size
    if case["kind"] == "compact":
        return {"bytes": 2.0 * row * (1 + 2 * R), "flops": 0}
    return {"bytes": 2.0 * row * case["pages"] * case["page_size"] * (0.5 if case["partial"] else 1), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        Hq, Hkv, D, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
        out = torch.zeros(s["qkv"].shape[0], Hq, D, dtype=torch.float64, device="cuda")
        table, lengths, row0 = s["table"].cpu(), s["lengths"].tolist(), s["row0"].tolist()
        for i, (n, lo, hi) in enumerate(zip(lengths, row0, row0[1:])):
            at = torch.arange(n + hi - lo)
            page, place = table[i, at // ps].long().cuda(), (at % ps).cuda()
            words = s["mask"][lo:hi].cpu().long() & 0xffffffff
            hidden = torch.tensor([[not words[r, k // 32] >> k % 32 & 1 for k in range(hi - lo)] for r in range(hi - lo)], device="cuda")
            for g in range(Hkv):
                k, v = (s["pages"][page, w, g, place].double() for w in (0, 1))
                for h in range(g * (Hq // Hkv), (g + 1) * (Hq // Hkv)):
                    scores = s["qkv"][lo:hi, h * D:(h + 1) * D].double() @ k.t() * s["scale"]
                    scores[:, n:].masked_fill_(hidden, -math.inf)
                    out[lo:hi, h] = torch.softmax(scores, -1) @ v
        return out.flatten(1)
    if case["kind"] == "verify":
        most, row0, parents = s["most"], s["row0"].tolist(), s["parents"].tolist()
        tokens, draws = s["tokens"].tolist(), s["draws"].double().tolist()
        accepted, path, said = [], [], []
        for lo, hi in zip(row0, row0[1:]):
            node, kept = 0, []
            while True:
                left, total, step = s["probs"][lo + node].double(), 1.0, None
                for child in (i for i in range(1, hi - lo) if parents[lo + i] == node):
                    x = tokens[lo + child]
                    q = s["draft"][lo + child].double() if s["draft"] is not None else None
                    if draws[lo + child] * total * (1.0 if q is None else q[x].item()) < left[x].item():
                        step = child
                        break
                    if q is None:
                        total -= left[x].item()
                        left[x] = 0.0
                    else:
                        left = torch.relu(left - total * q)
                        total = left.sum().item()
                if step is None:
                    break
                kept.append(step)
                node = step
            upto = left.cpu().cumsum(0)
            new = int(torch.searchsorted(upto, torch.tensor([draws[lo] * upto[-1].item()], dtype=torch.float64), right=True))
            accepted.append(len(kept))
            path.append(kept + [-1] * (most - len(kept)))
            said.append([tokens[lo + i] for i in kept] + [new] + [-1] * (most - len(kept)))
        return {"accepted": _ints(accepted), "path": _ints(path), "tokens": _ints(said)}
    pages = s["pages"]
    if case["kind"] == "compact":
        before, table, ps = pages.clone(), s["table"].tolist(), case["page_size"]
        for t, n, path, kept in zip(table, s["lengths"].tolist(), s["path"].tolist(), s["accepted"].tolist()):
            for j in range(kept):
                a, b = n + path[j], n + 1 + j
                pages[:, t[b // ps], :, :, b % ps] = before[:, t[a // ps], :, :, a % ps]
        return pages.double()
    rows = s["rows"].tolist() if s["rows"] is not None else [case["page_size"]] * case["pages"]
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), rows):
        pages[:, b, :, :, :n] = pages[:, a, :, :, :n]
    return pages.double()
