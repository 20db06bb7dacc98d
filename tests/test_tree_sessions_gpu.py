"""Sessions that decode, try trees, accept or leave them, fork and close in any order, in a cache that is now and then too small:
what each says is what its tokens run at once say, and no page is lost."""

import random

import pytest
import torch

from ninfer_amd_mi50_b200.api import Ninfer, NinferError
from ninfer_amd_mi50_b200.cache import OutOfPages
from test_trees_gpu import CONFIGS, close, path_to

pytestmark = pytest.mark.gpu

CFG = CONFIGS["A"]
VOCAB = CFG["vocab_size"]


def engine(sequences, tokens=None):
    return Ninfer(config=CFG, random_weights=11, dtype="float32", max_context=256, prefill_chunk=64, num_sequences=sequences, page_size=16,
                  cache_tokens=tokens)


def test_sessions_in_any_order():
    line = engine(1)

    def run_at_once(tokens):
        with line.session() as s:
            return s.prefill(tokens)

    counts = {"checked": 0, "accepted": 0, "refused": 0}
    for seed in range(8):
        rnd = random.Random(seed)
        eng, live = engine(5, 320), []                       # [session, its tokens, the tree that it may accept]
        tokens = lambda n: [rnd.randrange(VOCAB) for _ in range(n)]
        for _ in range(150):
            what = rnd.choice(["open", "fork", "decode", "decode", "tree", "trees", "batch", "close", "reset", "accept", "accept"])
            one = rnd.choice(live) if live else None
            try:
                if what == "open" or not live:
                    live.append([eng.session(), [], None])
                    new = tokens(rnd.randint(1, 60))
                    live[-1][0].prefill(new)
                    live[-1][1] = new
                elif what == "fork":
                    live.append([one[0].fork(), list(one[1]), None])
                elif what == "close":
                    one[0].close()
                    live.remove(one)
                elif what == "reset":
                    one[0].reset()
                    one[1:] = [], None
                elif what == "decode":
                    new = tokens(1)
                    got = one[0].decode(new[0])
                    one[1:] = one[1] + new, None
                    if rnd.random() < 0.2:
                        close(got, run_at_once(one[1]), "float32")
                        counts["checked"] += 1
                elif what == "batch":
                    some = rnd.sample(live, rnd.randint(1, len(live)))
                    new = tokens(len(some))
                    eng.decode_batch([s[0] for s in some], new)
                    for s, t in zip(some, new):
                        s[1:] = s[1] + [t], None
                elif what in ("tree", "trees"):
                    some = [one] if what == "tree" else rnd.sample(live, min(2, len(live)))
                    sizes = [rnd.randint(1, 40) for _ in some]
                    trees = [(tokens(n), [-1] + [rnd.randrange(max(0, i - 6), i) for i in range(1, n)]) for n in sizes]
                    logits = eng.decode_trees([(s[0], *t) for s, t in zip(some, trees)])
                    at = 0
                    for s, (drafted, parents) in zip(some, trees):
                        s[2] = drafted, parents
                        if rnd.random() < 0.2 and len(s[1]) < 200:
                            node = rnd.randrange(len(drafted))
                            close(logits[at + node], run_at_once(s[1] + [drafted[i] for i in path_to(node, parents)]), "float32")
                            counts["checked"] += 1
                        at += len(drafted)
                elif what == "accept" and one[2]:
                    drafted, parents = one[2]
                    path = path_to(rnd.randrange(len(drafted)), parents)
                    one[0].accept(path[1:])
                    one[1:] = one[1] + [drafted[i] for i in path], None
                    counts["accepted"] += 1
            except (OutOfPages, NinferError):                # (trees that were to be accepted still are)
                counts["refused"] += 1
            eng._runner.cache.check()
            for s, said, _ in live:
                assert s.length == len(said)
        for s, _, _ in live:
            s.close()
        assert eng.pages_free == [eng._runner.cache.groups[0].pool.num_pages]
    assert min(counts.values()) > 20, counts
