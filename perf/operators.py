"""What is timed of the operators by which requests of one step differ from one another: their adapters beside a shared
projection, and the penalties, biases and masks on their logits.

Two kinds of case.  "adapter": a projection of a step's rows, every row with the low-rank adapter of its request (or
none) beside it.  "rules": the tokens that a decode step has drawn go into the requests' logs, and the logits of the
step after it get each request's penalties for repeated tokens, its biases and its mask of allowed tokens.
Layer sizes are those of the engine's main design at the two sizes that its benchmark names, and generic ones.
"""

from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 151936


# ---- the cases --------------------------------------------------------------------------------------------------

def _adapter(name, rows, k, widths, adapters, rank, mix, none, dtype="bfloat16"):
    """`rows` rows of `k` numbers through a projection to the stacked `widths`; a pool of `adapters` adapters of up to
    `rank`; `mix` "rows": every row is a request of its own, "prompts": a few requests with many rows each, "both";
    `none`: the share of requests without an adapter."""
    return {"name": name, "kind": "adapter", "rows": rows, "k": k, "widths": ",".join(map(str, widths)), "adapters": adapters,
            "rank": rank, "mix": mix, "none": none, "dtype": dtype}


def _rules(name, rows, vocab, longest, repetition, frequency, biases, masks, capacity):
    """`rows` requests with up to `longest` tokens each, logs of `capacity`; `repetition`: some have a penalty for every
    occurrence; `frequency`: some pay for what they have generated; up to `biases` biased tokens a row; `masks`: "none",
    "some" or "all" rows under a mask of allowed tokens."""
    return {"name": name, "kind": "rules", "rows": rows, "vocab": vocab, "longest": longest, "repetition": repetition,
            "frequency": frequency, "biases": biases, "masks": masks, "capacity": capacity}


def listed():
    return [
        # one request decodes: the attention's output projection at the smaller size
        _adapter("one row", 1, 2048, [2048], 8, 16, "rows", 0.0),
        # eight requests decode, each with an adapter of its own: queries, keys and values at the smaller size
        _adapter("8 rows, qkv", 8, 2048, [2048, 2048, 2048], 16, 16, "rows", 0.0),
        # a full decode step at the larger size, some requests without an adapter
        _adapter("64 rows, wide", 64, 3584, [3584], 48, 32, "rows", 0.25),
        # a step that mixes prompt portions and decoded tokens, an odd number of rows: gate and up of a feed-forward
        _adapter("777 rows, gate up", 777, 2048, [5632, 5632], 12, 64, "both", 0.1),
        # the portion of prompts that the engine runs by default: queries, keys and values at the smaller size
        _adapter("2048 rows, qkv", 2048, 2048, [2048, 2048, 2048], 8, 16, "prompts", 0.0),
        # the longest portions: queries, keys and values at the larger size
        _adapter("8192 rows, qkv wide", 8192, 3584, [3584, 512, 512], 8, 16, "prompts", 0.0),
        # the all-32-bit path, a few requests
        _adapter("16 rows, float32", 16, 2048, [2048], 4, 8, "rows", 0.2, "float32"),
        # one chat: penalties over a short log
        _rules("one chat", 1, VOCAB, 200, True, True, 8, "none", 4096),
        # eight requests, all of them under grammars
        _rules("8 grammars", 8, VOCAB, 2000, False, True, 0, "all", 4096),
        # a full decode step, everything at once
        _rules("64 mixed", 64, VOCAB, 8192, True, True, 300, "some", 8192),
        # long logs over a small vocabulary of odd size
        _rules("5 long logs", 5, 32003, 131072, False, True, 40, "some", 131072),
        # the largest step
        _rules("256 rows", 256, VOCAB, 4096, True, True, 64, "some", 4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random):
    if rng.random() < 0.6:
        narrow = rng.random() < 0.2
        while True:
            rows = _log(rng, 1, 48 if narrow else 8192)
            k = 8 * _log(rng, 16, 1024)
            widths = [_log(rng, 128, 8192) for _ in range(rng.choice([1, 1, 2, 3]))]
            if rng.random() < 0.6:
                widths = [16 * (-(-w // 16)) for w in widths]
            if rows * k * sum(widths) <= 8192 * 3584 * 4608 // 2:
                break
        case = _adapter("", rows, k, widths, _log(rng, 1, 48), rng.choice([8, 16, 32, 64, 128]),
                        rng.choice(["rows", "both", "prompts"]) if rows <= 256 else rng.choice(["both", "prompts"]),
                        rng.choice([0.0, 0.2, 0.5]), "float32" if narrow else "bfloat16")
    else:
        vocab = _log(rng, 1000, 160000)
        rows = _log(rng, 1, min(256, 256 * VOCAB // vocab))
        longest = _log(rng, 1, 131072 if rows <= 8 else 8192)
        case = _rules("", rows, vocab, longest, rng.random() < 0.5, rng.random() < 0.7, rng.choice([0, 5, 300]),
                      rng.choice(["none", "some", "all"]), 1 << max(4, (longest - 1).bit_length()))
    del case["name"]
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------

def _padded(rank):
    """The rank that a pool is laid out for: the next of 16, 32, 64, 128."""
    return max(16, 1 << (rank - 1).bit_length())


def _row_adapters(case, rnd):
    """The adapter of every row: one choice a request, requests one after the other."""
    choose = lambda: -1 if rnd.random() < case["none"] else rnd.randrange(case["adapters"])
    T, ids = case["rows"], []
    if case["mix"] != "prompts":
        single = T if case["mix"] == "rows" else min(T, rnd.randint(1, 64))
        # a request for every row; the first ones take the pool in turn, as a step full of distinct requests does
        ids += [i % case["adapters"] if rnd.random() >= case["none"] else -1 for i in range(single)]
    while len(ids) < T:
        n = min(T - len(ids), rnd.randint(max(1, T // 8), max(1, T // 2)))
        ids += [choose()] * n
    return ids


def prepare(case, seed):
    rnd = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    if case["kind"] == "adapter":
        dtype = getattr(torch, case["dtype"])
        T, K, n, R = case["rows"], case["k"], case["adapters"], _padded(case["rank"])
        widths = [int(w) for w in case["widths"].split(",")]
        N, S = sum(widths), len(widths)
        a = normal(n, S * R, K) / math.sqrt(K)
        b = normal(n, N, R) * 0.15
        # adapters of several ranks in one pool: what lies beyond an adapter's own rank holds zeros
        ranks = ints([max(1, case["rank"] >> rnd.randrange(3)) for _ in range(n)])
        dead = torch.arange(R, device="cuda")[None, :] >= ranks[:, None]
        a.view(n, S, R, K).masked_fill_(dead[:, None, :, None], 0.0)
        b.masked_fill_(dead[:, None, :], 0.0)
        return {"case": case, "x": normal(T, K).to(dtype), "w": (normal(N, K) * 0.5 / math.sqrt(K)).to(dtype), "a": a.to(dtype),
                "b": b.to(dtype), "scale": torch.rand(n, generator=gen, device="cuda") + 0.5, "ids": ints(_row_adapters(case, rnd)),
                "widths": widths, "slice": ints([s for s, w in enumerate(widths) for _ in range(w)])}
    R, V, cap = case["rows"], case["vocab"], case["capacity"]
    rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")
    # requests of many lengths, in slots that are handed out in any order; tokens of a text: few frequent ones, many rare ones
    slots = rnd.sample(range(R + 2), R)
    lengths = [case["longest"]] + [rnd.randint(1, case["longest"]) for _ in range(R - 1)]
    starts = [rnd.randint(0, n) for n in lengths]
    order = torch.randperm(V, generator=gen, device="cuda")
    text = lambda *shape: order[(V ** rand(*shape) - 1).long().clamp_(0, V - 1)].to(torch.int32)
    tail = (text(R + 2, cap), text(R))
    penalties = torch.tensor([[rnd.choice([1.0, 1.02, 1.05]) if case["repetition"] else 1.0,
                               rnd.choice([0.0, 0.1, 0.4]) if case["frequency"] else 0.0,
                               rnd.choice([0.0, 0.5, -0.25]) if case["frequency"] else 0.0] for _ in range(R)], device="cuda")
    state = {"case": case, "logits": normal(R, V) * 3.0, "history": tail[0], "slots": ints(slots), "lengths": ints(lengths),
             "starts": ints(starts), "tokens": tail[1], "penalties": penalties, "bias": None, "mask": None}
    if case["biases"]:
        per = [sorted(rnd.sample(range(V), rnd.randint(0, min(V, case["biases"])))) for _ in range(R)]
        offsets = [0]
        for p in per:
            offsets.append(offsets[-1] + len(p))
        ids = ints([i for p in per for i in p])
        values = torch.where(rand(len(ids)) < 0.1, torch.tensor(-100.0, device="cuda"), normal(len(ids)) * 4.0)
        state["bias"] = (ints(offsets), ids, values)
    if case["masks"] != "none":
        # a few grammar states; some rows share one.  Few tokens are allowed, a third, or nearly all
        M, words = max(1, (R + 1) // 2), (V + 31) // 32
        keep = torch.tensor([rnd.choice([0.002, 0.3, 0.97]) for _ in range(M)], device="cuda")
        allowed = rand(M, words, 32) < keep[:, None, None]
        bits = (allowed.long() << torch.arange(32, device="cuda")).sum(-1)
        bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
        index = [rnd.randrange(M) if case["masks"] == "all" or rnd.random() < 0.5 else -1 for _ in range(R)]
        state["mask"] = (bits, ints(index))
    return state


# ---- the operators ------------------------------------------------------------------------------------------------

def _plain_adapter(s):
    """Every adapter on every row, and all but the row's own multiplied by nothing: two products more beside the shared one."""
    x, ids, n, R = s["x"].float(), s["ids"].long(), s["a"].shape[0], s["b"].shape[2]
    T, S = x.shape[0], len(s["widths"])
    mine = (ids[:, None] == torch.arange(n, device=x.device)).float() * s["scale"]
    h = (x @ s["a"].float().flatten(0, 1).t()).view(T, n, S * R) * mine[:, :, None]
    in_slice = (s["slice"][:, None] == torch.arange(S, device=x.device)).float()                # [N, S]
    spread = s["b"].float()[:, :, None, :] * in_slice[:, :, None]                               # [n, N, S, R]
    y = x @ s["w"].float().t() + h.flatten(1) @ spread.permute(0, 2, 3, 1).reshape(n * S * R, -1)
    return y.to(s["x"].dtype)


def _plain_rules(s):
    logits, slots, lengths, starts = s["logits"], s["slots"].long(), s["lengths"].long(), s["starts"].long()
    R, V = logits.shape
    s["history"][slots, lengths - 1] = s["tokens"]
    log = s["history"][slots].long()
    at = torch.arange(log.shape[1], device=log.device)[None, :]
    known = (at < lengths[:, None]).float()
    zeros = torch.zeros_like(logits)
    count = zeros.scatter_add(1, log, known)
    made = zeros.scatter_add(1, log, known * (at >= starts[:, None]).float())
    p, f, q = s["penalties"][:, :, None].unbind(1)
    times = torch.pow(p, count)
    v = torch.where(count > 0, torch.where(logits > 0, logits / times, logits * times), logits)
    v = v - made * f - (made > 0).float() * q
    if s["bias"] is not None:
        offsets, ids, values = s["bias"]
        row = torch.repeat_interleave(torch.arange(R, device=log.device), (offsets[1:] - offsets[:-1]).long(), output_size=ids.numel())
        v = v.index_put((row, ids.long()), values, accumulate=True)
    if s["mask"] is not None:
        bits, index = s["mask"]
        words = bits[index.long().clamp_min(0)]
        on = ((words[:, :, None] >> torch.arange(32, device=log.device, dtype=torch.int32)) & 1).flatten(1)[:, :V] > 0
        v = torch.where(on | (index < 0)[:, None], v, -math.inf)
    return v


def run(s):
    if s["case"]["kind"] == "adapter":
        if not own:
            return _plain_adapter(s)
        from ninfer_amd_mi50_b200 import kernels
        return kernels.adapter_linear(s["x"], s["w"], s["a"], s["b"], s["scale"], s["ids"], s["widths"])
    if not own:
        return {"logits": _plain_rules(s), "history": s["history"]}
    from ninfer_amd_mi50_b200 import kernels
    out = kernels.adjust_logits(s["logits"], s["history"], s["slots"], s["lengths"], s["starts"], s["penalties"],
                                tokens=s["tokens"], bias=s["bias"], mask=s["mask"])
    return {"logits": out, "history": s["history"]}


# ---- what a pass cannot do without, and its outputs in 64 bits -----------------------------------------------------

def work(case):
    if case["kind"] == "adapter":
        T, K, R = case["rows"], case["k"], _padded(case["rank"])
        widths = [int(w) for w in case["widths"].split(",")]
        N, S, size = sum(widths), len(widths), 4 if case["dtype"] == "float32" else 2
        served = T * (1.0 - case["none"])
        if case["mix"] == "rows":
            used = min(case["adapters"], T) * (1.0 - case["none"])
        elif case["mix"] == "both":
            used = min(case["adapters"], min(T, 32) + 3) * (1.0 - case["none"])
        else:
            used = min(case["adapters"], 3, T) * (1.0 - case["none"])
        return {"bytes": size * (T * K + N * K + used * (S * R * K + N * R) + T * N) + 4 * T,
                "flops": 2.0 * T * K * N + 2.0 * served * (S * R * K + N * R)}
    R, V = case["rows"], case["vocab"]
    known = case["longest"] + (R - 1) * (1 + case["longest"]) / 2
    masked = {"none": 0, "some": 0.5, "all": 1}[case["masks"]] * R
    return {"bytes": 8.0 * R * V + 4 * known + 8 * (case["biases"] / 2) * R + min(masked, (R + 1) // 2) * V / 8, "flops": 4.0 * R * V}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adapter":
        x, R, ends, begin = s["x"].double(), s["b"].shape[2], [], 0
        y = x @ s["w"].double().t()
        for w in s["widths"]:
            ends.append((begin, begin + w))
            begin += w
        for a in sorted(set(s["ids"].tolist()) - {-1}):
            rows = (s["ids"] == a).nonzero()[:, 0]
            h = (x[rows] @ s["a"][a].double().t()) * s["scale"][a].double()
            for i, (lo, hi) in enumerate(ends):
                y[rows, lo:hi] += h[:, i * R:(i + 1) * R] @ s["b"][a, lo:hi].double().t()
        return y
    logits, V = s["logits"].double(), case["vocab"]
    slots, lengths, starts = s["slots"].tolist(), s["lengths"].tolist(), s["starts"].tolist()
    penalties = s["penalties"].double().tolist()
    for r, (slot, n, start) in enumerate(zip(slots, lengths, starts)):
        s["history"][slot, n - 1] = s["tokens"][r]
        log = s["history"][slot, :n].long()
        count, made = (torch.bincount(t, minlength=V).double() for t in (log, log[start:]))
        p, f, q = penalties[r]
        v = logits[r]
        v = torch.where(v > 0, v * p ** -count, v * p ** count) - f * made - q * made.clamp(max=1)
        if s["bias"] is not None:
            offsets, ids, values = s["bias"]
            lo, hi = offsets[r].item(), offsets[r + 1].item()
            v[ids[lo:hi].long()] += values[lo:hi].double()
        if s["mask"] is not None and s["mask"][1][r] >= 0:
            words = s["mask"][0][s["mask"][1][r].item()].long()
            ids = torch.arange(V, device=v.device)
            v[(words[ids // 32] >> (ids % 32)) & 1 == 0] = -math.inf
        most = torch.finfo(torch.float32).max      # the result's type ends here
        v[v > most], v[v < -most] = math.inf, -math.inf
        logits[r] = v
    return {"logits": logits, "history": None}
