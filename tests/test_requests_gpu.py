"""What requests bring of their own, through the engine on the GPU: adapters beside the projections of prompt portions and of
decode steps replayed from graphs, and penalties, biases and allowed tokens on their logits."""

import pytest
import torch

import plain_model
from adapter_models import merged, random_adapter
from tiny_configs import TINY_A, TINY_B, TINY_D, random_tokens

pytestmark = pytest.mark.gpu

# all layers dense: no choice of experts that a rounding could turn
CONFIGS = {"B": dict(TINY_B, mlp_only_layers=[0, 1, 2]), "D": dict(TINY_D, mlp_only_layers=[0, 1])}
# as for the engine without adapters: float32 sums in another order, bfloat16 roundings of activations
BOUND = {"float32": 1e-4, "bfloat16": 1.5e-2}


@pytest.fixture(scope="module", params=["B", "D"])
def model(request, tmp_path_factory):
    from ninfer_amd_mi50_b200.weights import write_random_model
    cfg = CONFIGS[request.param]
    d = str(tmp_path_factory.mktemp("requests") / request.param)
    write_random_model(cfg, 7, d)
    return d, cfg, plain_model.read_model_folder(d)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_portions_and_replayed_decode_steps_with_adapters(model, dtype):
    from ninfer_amd_mi50_b200.config import EngineOptions
    from ninfer_amd_mi50_b200.engine import StepEntry, load_runner
    d, cfg, (pcfg, weights) = model
    runner = load_runner(d, options=EngineOptions(dtype=dtype, num_sequences=4, max_context=512, adapters=3, adapter_rank=20))
    bank = runner.adapters
    adapters = {n: (random_adapter(cfg, i, 20, keep), s) for i, (n, keep, s) in enumerate([("x", 1.0, 1.25), ("y", 0.5, -0.75), ("z", 1.0, 0.5)])}
    for n, (a, s) in adapters.items():
        bank.load(n, a, s)
    who = {"r0": "x", "r1": None, "r2": "z", "r3": "y"}
    reqs = {r: random_tokens(n, cfg["vocab_size"], 70 + n) for r, n in zip(who, (150, 33, 7, 90))}
    got = {r: [] for r in reqs}
    for r in reqs:
        runner.open(r)

    def step(parts):
        out = runner.step([StepEntry(r, reqs[r][lo:hi], list(range(hi - lo)), bank.slot(who[r])) for r, lo, hi in parts])
        at = 0
        for r, lo, hi in parts:
            got[r].append(out[at:at + hi - lo].float().cpu())
            at += hi - lo

    step([("r0", 0, 97), ("r2", 0, 1), ("r1", 0, 20)])
    step([("r2", 1, 2), ("r0", 97, 98), ("r3", 0, 80), ("r1", 20, 23)])
    step([("r0", 98, 140), ("r1", 23, 24)])
    for i in range(5):                       # single tokens: replayed from a graph; the last ones without an adapter among them
        step([("r1", 24 + i, 25 + i), ("r3", 80 + i, 81 + i), ("r2", 2 + i, 3 + i), ("r0", 140 + i, 141 + i)])
    for i in range(3):
        step([("r1", 29 + i, 30 + i)])
    assert sorted(len(k) for k in runner.graphs.graphs) == [2, 3]
    for r in reqs:
        w = weights if who[r] is None else merged(weights, *adapters[who[r]])
        have = torch.cat(got[r])
        want = plain_model.plain_forward(pcfg, w, reqs[r])[:len(have)]
        assert (have - want).abs().max() <= BOUND[dtype] * want.abs().max(), r
        if who[r] is not None:               # the adapter is no rounding
            assert (want - plain_model.plain_forward(pcfg, weights, reqs[r])[:len(have)]).abs().max() > 0.1 * want.abs().max()
    from ninfer_amd_mi50_b200 import kernels
    kernels.check_status("test")


def test_generation_with_everything_at_once(tmp_path):
    """Adapters, penalties, biases and allowed tokens in one batch, with decode steps ahead of the host where the rules allow it:
    each request as if it were alone."""
    from ninfer_amd_mi50_b200.api import Ninfer
    from ninfer_amd_mi50_b200.sampling import SamplingParams, sample_reference
    from ninfer_amd_mi50_b200.weights import write_random_model
    cfg = dict(TINY_A, mlp_only_layers=[0, 1])
    write_random_model(cfg, 5, str(tmp_path))
    pcfg, weights = plain_model.read_model_folder(str(tmp_path))
    V = cfg["vocab_size"]
    eng = Ninfer(str(tmp_path), max_context=256, num_sequences=8, dtype="float32", adapters=2, adapter_rank=8)
    ad = random_adapter(cfg, 9, 8)
    eng.load_adapter("a", ad, 1.5)
    evens = list(range(0, V, 2))
    asked = []

    def alternate(generated):
        asked.append(len(generated))
        return evens if len(generated) % 2 else [i + 1 for i in evens]

    params = [SamplingParams(0.0, max_new_tokens=12), SamplingParams(0.0, frequency_penalty=1.5, presence_penalty=0.5, max_new_tokens=12),
              SamplingParams(0.0, allowed_tokens=alternate, max_new_tokens=12),
              SamplingParams(0.0, logit_bias={11: -float("inf"), 3: 0.25}, allowed_tokens=evens + [11], max_new_tokens=12),
              SamplingParams(0.0, repetition_penalty=1.3, max_new_tokens=12)]
    prompts = [random_tokens(n, V, 60 + n) for n in (17, 9, 30, 5, 12)]
    names = [None, "a", None, "a", "a"]
    got = eng._engine.generate(prompts, params, adapter=names)
    for p, sp, n, g in zip(prompts, params, names, got):
        w = weights if n is None else merged(weights, ad, 1.5)
        tokens = list(p)
        logits = plain_model.plain_forward(pcfg, w, p + g)
        for i, tok in enumerate(g):
            row = logits[len(p) - 1 + i]
            if tok != sample_reference(row, sp, tokens, prompt_length=len(p)):
                # (two tokens within float32 roundings of one another)
                adjusted = row.clone()
                adjusted[tok] += 1e-4 * row.abs().max()
                assert tok == sample_reference(adjusted, sp, tokens, prompt_length=len(p)), (n, i)
            tokens.append(tok)
        assert len(g) == 12
    # alone, and with no rule that looks back: steps run ahead of the host
    before = eng.stats()["ahead_steps"]
    alone = eng.generate([prompts[3]], max_new_tokens=12, temperature=0.0, logit_bias=params[3].logit_bias,
                         allowed_tokens=evens + [11], adapter="a")
    assert alone[0] == got[3] and eng.stats()["ahead_steps"] > before
    with eng.session(adapter="a") as s:
        l = s.prefill(prompts[4])
        first = eng.sample(l, temperature=0.0, repetition_penalty=1.3, recent=prompts[4], prompt_length=len(prompts[4]))
        assert first == got[4][0]
    drawn = eng.generate([prompts[0]] * 3, max_new_tokens=8, temperature=0.9, allowed_tokens=[1, 2, 3], seed=4)
    assert all(t in (1, 2, 3) for g in drawn for t in g)
    eng.close()
