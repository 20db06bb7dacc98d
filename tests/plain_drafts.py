"""Trees of drafted tokens in their plain form, in 64 bits on the CPU: attention over the cache, verification, and the
cache's rows moved and copied."""

import math
import random

import torch


def tree(rnd, n, shape="tree"):
    """Parents of n nodes; each below any node before it, or all in a row."""
    return [-1] + [i - 1 if shape == "chain" else rnd.randrange(max(0, i - 9), i) for i in range(1, n)]


def masks(parents, words):
    """int32 [nodes, words]: a node's ancestors and itself."""
    seen, out = [], []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        out.append([(seen[i] >> 32 * w & 0xffffffff) - ((seen[i] >> 32 * w + 31 & 1) << 32) for w in range(words)])
    return torch.tensor(out, dtype=torch.int64).reshape(len(out), words).to(torch.int32)


def block_tables(lengths, page_size, rnd, spare=1):
    """(int32 [S, width], number of pages): pages in any order, -1 behind a request's last."""
    need = [-(-n // page_size) for n in lengths]
    pool = list(range(sum(need) + spare))
    rnd.shuffle(pool)
    table, at = torch.full((len(need), max(1, max(need))), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(pool[at:at + n], dtype=torch.int32)
        at += n
    return table, len(pool)


def plain_attention(qkv, Hq, Hkv, D, pages, table, page_size, lengths, row0, mask, scale):
    """-> (out, weight): the result [T, Hq * D], and the weighted sum of the values' sizes, by which errors are measured; both
    NaN in rows that belong to no request.  Also the largest sum of |q||k| that a score was added up of."""
    T = qkv.shape[0]
    out, weight = (torch.full((T, Hq, D), math.nan, dtype=torch.float64) for _ in range(2))
    size = 0.0
    for s, (n, lo, hi) in enumerate(zip(lengths, row0, row0[1:])):
        at = torch.arange(n + hi - lo)
        page = table[s, at // page_size].long() if len(at) else at
        k, v = (pages[page, w, :, at % page_size].double() for w in (0, 1))             # [keys, Hkv, D]
        for t in range(lo, hi):
            seen = [j < n or bool(int(mask[t, (j - n) // 32]) >> (j - n) % 32 & 1) for j in range(len(at))]
            for h in range(Hq):
                g, q = h // (Hq // Hkv), qkv[t, h * D:(h + 1) * D].double()
                kk, vv = k[seen][:, g], v[seen][:, g]
                if not len(kk):
                    out[t, h] = weight[t, h] = 0.0
                    continue
                size = max(size, float((kk.abs() @ q.abs()).max()) * scale)
                p = torch.softmax(kk @ q * scale, 0)
                out[t, h], weight[t, h] = p @ vv, p @ vv.abs()
    return out.flatten(1), weight.flatten(1), size


def plain_verify(probs, tokens, parents, row0, draws, most, draft=None):
    """-> (accepted, path, said) as lists."""
    accepted, path, said = [], [], []
    for lo, hi in zip(row0, row0[1:]):
        v, kept = 0, []
        while True:
            r, z, step = probs[lo + v].double().clone(), 1.0, None
            for c in range(1, hi - lo):
                if parents[lo + c] != v or len(kept) == most:
                    continue
                x = int(tokens[lo + c])
                q = 1.0 if draft is None else float(draft[lo + c, x])
                if float(draws[lo + c]) * z * q < float(r[x]):
                    step = c
                    break
                if draft is None:
                    z -= float(r[x])
                    r[x] = 0.0
                else:
                    r = (r - z * draft[lo + c].double()).clamp_min(0.0)
                    z = float(r.sum())
            if step is None:
                break
            kept.append(step)
            v = step
        if not float(r.sum()) > 0.0:
            r = probs[lo + v].double()
        run = r.cumsum(0)
        past = ((run > float(draws[lo]) * float(run[-1])) & (r > 0)).nonzero()
        new = int(past[0]) if len(past) else -1
        accepted.append(len(kept))
        path.append(kept + [-1] * (most - len(kept)))
        said.append([int(tokens[lo + c]) for c in kept] + [new] + [-1] * (most - len(kept)))
    return accepted, path, said


def plain_compact(pages, table, lengths, path, accepted):
    """[layers, pages, planes, page_size, width] on the CPU, a copy in which the kept rows have moved."""
    out, ps = pages.clone(), pages.shape[3]
    for s, n in enumerate(accepted):
        for j in range(n):
            a, b = lengths[s] + path[s][j], lengths[s] + 1 + j
            out[:, table[s, b // ps], :, b % ps] = pages[:, table[s, a // ps], :, a % ps]
    return out


def make_attention(sizes, lengths, heads, page_size=16, words=None, seed=0, shape="tree", sharp=1.0):
    """CPU tensors of a step: qkv float32 [T, (Hq + 2 Hkv) D], pages, block table, lengths, row0, mask, the largest context."""
    Hq, Hkv, D = heads
    rnd, g = random.Random(seed), torch.Generator().manual_seed(seed)
    row0 = [0]
    for n in sizes:
        row0.append(row0[-1] + n)
    words = words or max(1, (max(sizes) + 31) // 32)
    mask = torch.cat([masks(tree(rnd, n, shape), words) if n else torch.zeros(0, words, dtype=torch.int32) for n in sizes])
    table, pages = block_tables([a + b for a, b in zip(lengths, sizes)], page_size, rnd)
    return {"qkv": torch.randn(row0[-1], (Hq + 2 * Hkv) * D, generator=g) * sharp, "pages": torch.randn(pages, 2, Hkv, page_size, D, generator=g),
            "table": table, "lengths": list(lengths), "row0": row0, "mask": mask, "longest": max(1, max(a + b for a, b in zip(lengths, sizes)))}


def make_verify(sizes, V, draft, seed=0, shape="tree", near=0.5):
    """CPU tensors of a verification; siblings now and then name one token twice."""
    rnd, g = random.Random(seed), torch.Generator().manual_seed(seed)
    row0, parents = [0], []
    for n in sizes:
        parents += tree(rnd, n, shape)
        row0.append(row0[-1] + n)
    T = row0[-1]
    logits = torch.randn(T, V, generator=g) * 3
    up = torch.tensor([lo + max(p, 0) for lo, hi in zip(row0, row0[1:]) for p in parents[lo:hi]])
    q = torch.softmax(logits[up] + torch.randn(T, V, generator=g) * near, -1)
    return {"probs": torch.softmax(logits, -1), "tokens": torch.multinomial(q, 1, generator=g)[:, 0].int(), "draft": q if draft else None,
            "parents": torch.tensor(parents, dtype=torch.int32), "row0": row0, "draws": torch.rand(T, generator=g)}
