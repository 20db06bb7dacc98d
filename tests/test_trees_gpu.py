"""Trees of drafted tokens and forks through the engine's sessions: a tree's logits are those of its paths run one token
after the other, what is accepted goes on as if run in a line, and drafting, verification and the cache work together."""

import pytest
import torch

from tiny_configs import TINY_A, TINY_B, TINY_C, TINY_D, random_tokens

pytestmark = pytest.mark.gpu

# all layers dense: no choice of experts that a rounding could turn
CONFIGS = {"A": dict(TINY_A, mlp_only_layers=[0, 1]), "B": dict(TINY_B, mlp_only_layers=[0, 1, 2]), "D": dict(TINY_D, mlp_only_layers=[0, 1])}
# the same step in another form: float32 sums in another order, bfloat16 roundings of activations
BOUND = {"float32": 1e-4, "bfloat16": 1.5e-2}
PARENTS = [-1, 0, 0, 1, 1, 2, 3, 6, 5, 0]


def engine(cfg, dtype, sequences=8, **more):
    from ninfer_amd_mi50_b200.api import Ninfer
    return Ninfer(config=cfg, random_weights=11, dtype=dtype, max_context=512, prefill_chunk=128, num_sequences=sequences, **more)


def close(got, want, dtype):
    got, want = torch.as_tensor(got), torch.as_tensor(want)
    assert float((got - want).abs().max()) <= BOUND[dtype] * float(want.abs().max())


def path_to(node, parents):
    out = []
    while node >= 0:
        out.append(node)
        node = parents[node]
    return out[::-1]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["A", "B", "D"])
@pytest.mark.parametrize("length", [1, 63, 100])
def test_a_tree_is_its_paths(which, dtype, length):
    cfg = CONFIGS[which]
    eng = engine(cfg, dtype)
    prompt, drafted = random_tokens(length, cfg["vocab_size"], 3), random_tokens(len(PARENTS), cfg["vocab_size"], 4)
    s = eng.session()
    s.prefill(prompt)
    logits = s.decode_tree(drafted, PARENTS)
    assert s.length == length
    for leaf in (4, 7, 8, 9):
        with s.fork() as f:                          # (a fork knows nothing of a tree that was not accepted)
            for node in path_to(leaf, PARENTS):
                close(logits[node], f.decode(drafted[node]), dtype)
    # the path of the deepest leaf is kept; what follows is what would follow it in a line
    straight = s.fork()
    logits = s.decode_tree(drafted, PARENTS)
    s.accept([1, 3, 6, 7])
    for node in (0, 1, 3, 6, 7):
        want = straight.decode(drafted[node])
    close(logits[7], want, dtype)
    assert s.length == straight.length == length + 5
    for tok in random_tokens(5, cfg["vocab_size"], 5):
        close(s.decode(tok), straight.decode(tok), dtype)
    eng._runner.cache.check()
    s.close()
    straight.close()
    assert eng.pages_free == [eng._runner.cache.groups[0].pool.num_pages]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_trees_of_several_sessions_in_one_step(dtype):
    cfg = CONFIGS["B"]
    eng = engine(cfg, dtype, sequences=6)
    lengths, trees = (5, 64, 200), ([-1], PARENTS, [-1, 0, 1, 2, 3, 0, 5])
    sessions, drafted, alone = [], [], []
    for i, n in enumerate(lengths):
        s = eng.session()
        s.prefill(random_tokens(n, cfg["vocab_size"], 20 + i))
        sessions.append(s)
        drafted.append(random_tokens(len(trees[i]), cfg["vocab_size"], 30 + i))
        alone.append(s.decode_tree(drafted[i], trees[i]))
    got = eng.decode_trees(list(zip(sessions, drafted, trees)))
    at = 0
    for a in alone:
        close(got[at:at + len(a)], a, dtype)
        at += len(a)
    eng._runner.accept({sessions[0]._key: [], sessions[1]._key: [2, 5, 8], sessions[2]._key: [5]})
    assert [s.length for s in sessions] == [6, 68, 202]
    for i, (s, path) in enumerate(zip(sessions, ([0], [0, 2, 5, 8], [0, 5]))):
        straight = eng.session()
        straight.prefill(random_tokens(lengths[i], cfg["vocab_size"], 20 + i) + [drafted[i][n] for n in path])
        close(s.decode(7), straight.decode(7), dtype)
        straight.close()
    eng._runner.cache.check()


@pytest.mark.parametrize("lookup", [False, True], ids=["a line", "a tree"])
def test_drafting_verification_and_cache_together(lookup):
    """Greedy generation by drafts: certain probabilities make verification take exactly the tokens that decoding gives."""
    from ninfer_amd_mi50_b200 import kernels
    cfg = CONFIGS["A"]
    eng = engine(cfg, "float32")
    prompt = random_tokens(40, cfg["vocab_size"], 8)
    want = eng.generate([prompt], max_new_tokens=40, temperature=0.0)[0]
    s = eng.session()
    first = int(torch.as_tensor(s.prefill(prompt)).argmax())
    out, steps, ints = [first], 0, lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    rnd = torch.Generator().manual_seed(1)
    while len(out) < 40:
        # drafts: the right tokens, now and then with a wrong one among them, and wrong siblings before them
        right = (want + [0] * 8)[len(out):len(out) + 5]
        tokens, parents, at = [out[-1]], [-1], 0
        for t in right:
            wrong = int(torch.randint(cfg["vocab_size"], (1,), generator=rnd))
            if lookup:
                tokens.append(wrong)
                parents.append(at)
            tokens.append(wrong if float(torch.rand(1, generator=rnd)) < 0.2 else t)
            parents.append(at)
            at = len(tokens) - 1
        logits = torch.as_tensor(s.decode_tree(tokens, parents)).cuda()
        probs = torch.zeros_like(logits).scatter_(1, logits.argmax(1, keepdim=True), 1.0)
        accepted, path, said = kernels.verify_drafts(probs, ints(tokens), ints(parents), ints([0, len(tokens)]),
                                                     torch.rand(len(tokens), generator=rnd).cuda(), len(tokens) - 1)
        n = int(accepted[0])
        s.accept(path[0, :n].tolist())
        out += said[0, :n + 1].tolist()
        steps += 1
    assert out[:40] == want and steps < 39
    kernels.check_status()


def test_everything_captured_and_replayed():
    """The four operators in one graph, replayed for other trees, lengths and draws."""
    import random

    from ninfer_amd_mi50_b200 import kernels
    from plain_drafts import block_tables, make_attention, make_verify, plain_attention, plain_compact, plain_verify
    heads, ps, V, sizes = (8, 2, 64), 16, 700, [9, 6]
    a = make_attention(sizes, [40, 25], heads, ps, seed=1)
    v = make_verify(sizes, V, False, seed=1)
    cache = torch.randn(3, 10, 2, heads[1], ps, heads[2], generator=torch.Generator().manual_seed(9)).bfloat16()
    dev = {k: t.cuda() for k, t in dict(qkv=a["qkv"].bfloat16(), pages=cache, table=a["table"], lengths=torch.tensor(a["lengths"], dtype=torch.int32),
                                        row0=torch.tensor(a["row0"], dtype=torch.int32), mask=a["mask"], probs=v["probs"], tokens=v["tokens"],
                                        parents=v["parents"], draws=v["draws"], src=torch.tensor([0], dtype=torch.int32),
                                        dst=torch.tensor([cache.shape[1] - 1], dtype=torch.int32)).items()}

    def all_four():
        out = kernels.tree_attention(dev["qkv"], *heads, dev["pages"][0], dev["table"], ps, dev["lengths"], dev["row0"], dev["mask"], 64, 0.125)
        accepted, path, said = kernels.verify_drafts(dev["probs"], dev["tokens"], dev["parents"], dev["row0"], dev["draws"], 8)
        kernels.compact_cache(dev["pages"], dev["table"], dev["lengths"], path, accepted)
        kernels.copy_pages(dev["pages"], dev["src"], dev["dst"])
        return out, accepted, path, said

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_four()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_four()
    for seed in range(2, 6):
        rnd = random.Random(seed)
        lengths = [rnd.randint(0, 48), rnd.randint(0, 40)]
        a = make_attention(sizes, lengths, heads, ps, seed=seed)
        v = make_verify(sizes, V, False, seed=seed)
        table, n = block_tables([50 + 9, 50 + 6], ps, rnd, spare=0)
        pages = torch.randn(cache.shape, generator=torch.Generator().manual_seed(seed)).bfloat16()
        assert table.shape == tuple(dev["table"].shape) and n < cache.shape[1]
        for k, t in dict(qkv=a["qkv"].bfloat16(), pages=pages, table=table, lengths=torch.tensor(lengths, dtype=torch.int32), mask=a["mask"],
                         probs=v["probs"], tokens=v["tokens"], parents=v["parents"], draws=v["draws"]).items():
            dev[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want, weight, _ = plain_attention(a["qkv"].bfloat16().float(), *heads, pages[0].float(), table, ps, lengths, a["row0"], a["mask"], 0.125)
        assert bool(((got[0].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * weight).all())
        accepted, path, said = plain_verify(v["probs"], v["tokens"], v["parents"].tolist(), v["row0"], v["draws"], 8)
        assert (got[1].tolist(), got[2].tolist(), got[3].tolist()) == (accepted, path, said)
        moved = plain_compact(pages.flatten(2, 3), table, lengths, path, accepted).view(pages.shape)
        moved[:, -1] = moved[:, 0]
        assert torch.equal(dev["pages"].cpu(), moved)
    kernels.check_status()


def test_on_a_stream_of_its_own():
    from ninfer_amd_mi50_b200 import kernels
    from plain_drafts import make_attention, make_verify, plain_verify
    a = make_attention([20, 31], [900, 1500], (16, 4, 128), 64, seed=3)
    v = make_verify([20, 31], 9000, True, seed=3)
    args = [t.cuda() for t in (a["qkv"].bfloat16(), a["pages"].bfloat16(), a["table"], torch.tensor(a["lengths"], dtype=torch.int32),
                               torch.tensor(a["row0"], dtype=torch.int32), a["mask"])]
    call = lambda: kernels.tree_attention(args[0], 16, 4, 128, args[1], args[2], 64, *args[3:], a["longest"], 0.09)
    first = call()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    probs = [v[k].cuda() for k in ("probs", "tokens", "parents")] + [args[4], v["draws"].cuda(), 30, v["draft"].cuda()]
    torch.cuda.synchronize()
    for _ in range(5):                               # two calls at once
        for st in streams:
            with torch.cuda.stream(st):
                got.append((call(), kernels.verify_drafts(*probs)))
    torch.cuda.synchronize()
    want = plain_verify(v["probs"], v["tokens"], v["parents"].tolist(), v["row0"], v["draws"], 30, v["draft"])
    for out, said in got:
        assert torch.equal(out, first) and tuple(t.tolist() for t in said) == want
    kernels.check_status()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_trees_and_forks_of_sessions_with_adapters(dtype):
    """Trees of sessions with different adapters and with none, in one step; a fork keeps its adapter in its place."""
    from adapter_models import random_adapter
    cfg = CONFIGS["B"]
    eng = engine(cfg, dtype, adapters=2, adapter_rank=8)
    eng.load_adapter("a", random_adapter(cfg, 1, 8), 1.5)
    eng.load_adapter("b", random_adapter(cfg, 2, 5), -0.5)
    sessions = [eng.session(name) for name in ("a", None, "b")]
    drafted = [random_tokens(len(PARENTS), cfg["vocab_size"], 30 + i) for i in range(3)]
    for i, s in enumerate(sessions):
        s.prefill(random_tokens(20 + 50 * i, cfg["vocab_size"], i))
    logits = eng.decode_trees([(s, d, PARENTS) for s, d in zip(sessions, drafted)])
    for i, s in enumerate(sessions):
        s.accept([1, 4])
        f = s.fork()
        with pytest.raises(Exception, match="accept|not a tree"):
            f.accept([1])
        f.close()
    others = [s.fork() for s in sessions]
    for i, (s, f) in enumerate(zip(sessions, others)):
        close(s.decode(7), f.decode(7), dtype)
    # the same paths run in a line by sessions of their own
    for i, name in enumerate(("a", None, "b")):
        with eng.session(name) as line:
            line.prefill(random_tokens(20 + 50 * i, cfg["vocab_size"], i))
            for node in (0, 1, 4):
                close(logits[i * len(PARENTS) + node], line.decode(drafted[i][node]), dtype)
    for s in sessions:
        s.close()
    with pytest.raises(Exception, match="in use"):           # (by the fork)
        eng.drop_adapter("a")
    for f in others:
        f.close()
    eng.drop_adapter("a")
    eng._runner.cache.check()


def test_refusals():
    from ninfer_amd_mi50_b200.api import NinferError
    from ninfer_amd_mi50_b200.engine import BatchError
    eng = engine(CONFIGS["A"], "float32", sequences=2)
    s = eng.session()
    s.prefill([1, 2, 3])
    with pytest.raises(BatchError):
        s.accept()
    for tokens, parents in [([], None), ([1, 2], [-1, 1]), ([1] * 257, None), ([1, 5000], None)]:
        with pytest.raises(BatchError):
            s.decode_tree(tokens, parents)
    s.decode_tree([4, 5, 6], [-1, 0, 0])
    for path in ([3], [1, 2], [2, 1], [-1], [0]):
        with pytest.raises(BatchError):
            s.accept(path)
    s.decode(4)
    with pytest.raises(BatchError):                  # the tree's rows have been written over
        s.accept([1])
    s.decode_tree([4, 5, 6], [-1, 0, 0])
    s.reset()
    with pytest.raises(BatchError):
        s.accept([1])
    t = s.fork()
    with pytest.raises(NinferError):                 # no slot left
        s.fork()
    t.close()
    windowed = engine(dict(TINY_C, mlp_only_layers=[0, 1, 2, 3]), "float32", sequences=2)
    w = windowed.session()
    w.prefill([1, 2, 3])
    with pytest.raises(BatchError, match="cannot run a tree"):
        w.decode_tree([4, 5])
    f = w.fork()                                     # (forks are for every model)
    close(f.decode(9), w.decode(9), "float32")


@pytest.mark.parametrize("arch", ["vekasun", "difavik", "nolesun"])
def test_forks_of_models_with_states_and_windows(arch):
    import importlib
    configs = importlib.import_module(f"{arch}_configs")
    cfg, _ = next(iter(configs.CONFIGS.values()))
    eng = engine(cfg, "float32", sequences=3)
    vocab = cfg["vocab"]
    s = eng.session()
    s.prefill(random_tokens(90, vocab, 1))
    f = s.fork()
    for tok in random_tokens(20, vocab, 2):
        a, b = s.decode(tok), f.decode(tok)
        close(a, b, "float32")
    s.decode(1)
    g = f.fork()
    for tok in random_tokens(8, vocab, 3):
        close(g.decode(tok), f.decode(tok), "float32")
    eng._runner.cache.check()
