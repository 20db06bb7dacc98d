"""What requests bring of their own - adapters, penalties, biases, allowed tokens - through the engine's own logic on the
CPU, with the kernels replaced by their plain twins."""

import json
import math

import pytest
import torch

import plain_kernels
import plain_model
import plain_requests
from adapter_models import adapted_names, merged, random_adapter
from tiny_configs import CONFIGS, random_tokens

from ninfer_amd_mi50_b200 import kernels
from ninfer_amd_mi50_b200.config import EngineOptions
from ninfer_amd_mi50_b200.engine import Engine, StepEntry
from ninfer_amd_mi50_b200.engine.batch import BatchError
from ninfer_amd_mi50_b200.parts.adapters import AdapterError
from ninfer_amd_mi50_b200.sampling import Sampler, SamplingParams, check_params, sample_reference
from ninfer_amd_mi50_b200.weights import read_adapter, write_random_model, write_safetensors

CFG, SEED = CONFIGS["B"]          # (its second layer has a dense feed-forward)


@pytest.fixture
def engine(tmp_path, monkeypatch):
    d = str(tmp_path / "B")
    write_random_model(CFG, SEED, d)
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    eng = Engine(d, options=EngineOptions(dtype="float32", device="cpu", page_size=16, num_sequences=4, max_context=128,
                                          prefill_chunk=16, adapters=2, adapter_rank=9))
    return eng, plain_model.read_model_folder(d)


def test_every_request_has_its_own_adapter(engine):
    eng, (pcfg, weights) = engine
    A, B = random_adapter(CFG, 1, 9), random_adapter(CFG, 2, 5, keep=0.5)
    eng.load_adapter("a", A, 1.5)
    eng.load_adapter("b", B, 0.5)
    prompts = [random_tokens(n, CFG["vocab_size"], 20 + n) for n in (21, 3, 18, 9)]
    names = ["a", None, "b", "a"]
    got = eng.generate(prompts, SamplingParams(0.0, max_new_tokens=5), adapter=names)
    for p, g, n in zip(prompts, got, names):
        w = weights if n is None else merged(weights, A if n == "a" else B, 1.5 if n == "a" else 0.5)
        assert g == plain_model.plain_greedy(pcfg, w, p, 5), n


def test_a_slot_is_reused_without_what_it_held(engine):
    eng, (pcfg, weights) = engine
    A, B = random_adapter(CFG, 3, 9), random_adapter(CFG, 4, 4, keep=0.3)
    eng.load_adapter("a", A)
    eng.load_adapter("x", random_adapter(CFG, 5, 9))
    eng.drop_adapter("a")
    eng.load_adapter("b", B, 2.0)
    p = random_tokens(12, CFG["vocab_size"], 6)
    runner = eng.runner
    runner.open("r")
    got = runner.step([StepEntry("r", p, list(range(len(p))), eng.adapter_slot("b"))])
    want = plain_model.plain_forward(pcfg, merged(weights, B, 2.0), p)
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)
    runner.close("r")


def test_what_the_bank_refuses(engine):
    eng, _ = engine
    A = random_adapter(CFG, 1, 9)
    name = next(iter(A))
    a, b = A[name]
    bad = [({}, "nothing"), ({"model.norm.weight": (a, b)}, "take no adapters"), ({name: (a[:, 1:], b)}, "do not fit"),
           ({name: (a, b[:, :-1])}, "do not fit"), ({name: (torch.zeros(17, a.shape[1]), torch.zeros(b.shape[0], 17))}, "rank 17"),
           ({name: (a * math.nan, b)}, "finite"), ({name: (a, b * math.inf)}, "finite")]
    for weights, what in bad:
        with pytest.raises(AdapterError, match=what):
            eng.load_adapter("x", weights)
    with pytest.raises(AdapterError, match="scale"):
        eng.load_adapter("x", A, math.inf)
    assert not eng.runner.adapters.slots
    eng.load_adapter("x", A)
    with pytest.raises(AdapterError, match="already"):
        eng.load_adapter("x", A)
    eng.load_adapter("y", A)
    with pytest.raises(AdapterError, match="taken"):
        eng.load_adapter("z", A)
    with pytest.raises(AdapterError, match="no adapter"):
        eng.submit([1], adapter="z")
    eng.submit([1], SamplingParams(0.0, max_new_tokens=2), adapter="x")
    with pytest.raises(ValueError, match="in use"):
        eng.drop_adapter("x")
    eng.run_until_idle()
    eng.drop_adapter("x")
    eng.runner.open("r")
    with pytest.raises(BatchError, match="slot"):
        eng.runner.step([StepEntry("r", [1], [0], 0)])
    with pytest.raises(ValueError, match="2 prompts"):
        eng.generate([[1], [2]], adapter=["y"])


def test_an_engine_without_adapters(tmp_path, monkeypatch):
    d = str(tmp_path / "A")
    write_random_model(*CONFIGS["A"], d)
    plain_kernels.install(monkeypatch)
    eng = Engine(d, options=EngineOptions(dtype="float32", device="cpu", num_sequences=1, max_context=64))
    with pytest.raises(ValueError, match="keeps no adapters"):
        eng.load_adapter("x", {})
    with pytest.raises(ValueError, match="keeps no adapters"):
        eng.submit([1], adapter="x")
    with pytest.raises(ValueError):
        EngineOptions(adapters=-1)


def test_an_adapter_from_a_folder(engine, tmp_path):
    eng, (pcfg, weights) = engine
    A = {n: (torch.randn(4, k) / k ** 0.5, torch.randn(o, 4) * 0.1) for n, o, k in adapted_names(CFG, [0])}
    pairs = []
    for n, (a, b) in A.items():
        m = "base_model.model." + n[:-len(".weight")]
        pairs += [(m + ".lora_A.weight", a), (m + ".lora_B.weight", b)]
    write_safetensors(str(tmp_path / "adapter_model.safetensors"), pairs)
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 6}))
    got, scale = read_adapter(str(tmp_path))
    assert scale == 1.5 and got.keys() == A.keys() and all(torch.equal(got[n][i], A[n][i]) for n in A for i in (0, 1))
    eng.load_adapter("f", str(tmp_path))
    p = random_tokens(7, CFG["vocab_size"], 8)
    assert eng.generate([p], SamplingParams(0.0, max_new_tokens=4), adapter="f")[0] == plain_model.plain_greedy(
        pcfg, merged(weights, A, 1.5), p, 4)


@pytest.mark.parametrize("graphless", [True])
def test_penalties_biases_and_allowed_tokens_in_one_batch(engine, graphless):
    """Every request as it is generated alone, by the host's twin on the plain model's logits."""
    eng, (pcfg, weights) = engine
    V = CFG["vocab_size"]
    prompts = [random_tokens(n, V, 40 + n) for n in (11, 5, 8, 14)]

    def walk(generated):                       # ids that the last one says, none after four
        return None if not generated else [] if len(generated) == 4 else [(generated[-1] * 7 + i) % V for i in range(30)]

    params = [SamplingParams(0.0, repetition_penalty=1.1, frequency_penalty=0.8, presence_penalty=0.5, max_new_tokens=6),
              SamplingParams(0.0, logit_bias={3: 30.0, 4: 29.9}, frequency_penalty=4.0, max_new_tokens=6),
              SamplingParams(0.0, allowed_tokens=[5, 9, 1000], presence_penalty=50.0, max_new_tokens=6),
              SamplingParams(0.0, allowed_tokens=walk, max_new_tokens=6)]
    got = eng.generate(prompts, params)
    for p, sp, g in zip(prompts, params, got):
        tokens, want = list(p), []
        while len(want) < 6:
            if callable(sp.allowed_tokens) and sp.allowed_tokens(want) == []:
                break
            logits = plain_model.plain_forward(pcfg, weights, tokens)[-1]
            want.append(sample_reference(logits, sp, tokens, prompt_length=len(p)))
            tokens.append(want[-1])
        assert g == want
    assert set(got[2]) == {5, 9, 1000} and got[1][0] == 3 and got[1][1] == 4 and len(got[3]) == 4
    assert eng.requests["req-3"].finish_reason == "stop"


def test_a_function_that_fails_leaves_the_engine_as_it_was(engine):
    eng, (pcfg, weights) = engine
    calls = []

    def bad(generated):
        calls.append(len(generated))
        if len(calls) == 2:
            raise RuntimeError("grammar")
        return [1, 2, 3]

    p = random_tokens(6, CFG["vocab_size"], 2)
    rid = eng.submit(p, SamplingParams(0.0, allowed_tokens=bad, max_new_tokens=3))
    eng.step()
    with pytest.raises(RuntimeError, match="grammar"):
        eng.step()
    eng.run_until_idle()
    assert len(eng.requests[rid].generated) == 3 and set(eng.requests[rid].generated) <= {1, 2, 3}
    rid = eng.submit(p, SamplingParams(0.0, allowed_tokens=lambda g: [CFG["vocab_size"]], max_new_tokens=3))
    with pytest.raises(ValueError, match="outside"):
        eng.step()


def test_logs_are_sent_once_and_slots_change_hands(monkeypatch):
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    sent = []
    twin = kernels.append_history
    monkeypatch.setattr(kernels, "append_history", lambda h, s, p, t: (sent.append(len(t)), twin(h, s, p, t)))
    V, s, p = 50, Sampler(50, "cpu"), SamplingParams(0.0, presence_penalty=100.0)
    logits = torch.arange(V, dtype=torch.float32)[None]
    tokens = [[49, 48], [49]]
    for _ in range(3):
        out = s.sample(logits.expand(2, V).contiguous(), [p, p], recent=tokens, prompt_lengths=[0, 0], keys=["a", "b"]).tolist()
        assert out == [max(set(range(V)) - set(t)) for t in tokens]
        tokens = [t + [o] for t, o in zip(tokens, out)]
    assert sent == [3, 2, 2]
    for k in range(20):                                       # more requests than slots, none of them told to be done
        assert s.sample(logits, [p], recent=[[49, 47]], prompt_lengths=[0], keys=[k]).tolist() == [48]
    assert s.sample(logits, [p], recent=[tokens[0]], prompt_lengths=[1], keys=["a"]).tolist() == [49]      # the prompt's do not count
    long = list(range(40)) * 60                               # a longer log than there was room for
    assert s.sample(logits, [p], recent=[long], prompt_lengths=[0], keys=["a"]).tolist() == [49]
    s.forget("a")
    assert s.sample(logits, [p], recent=[[1]], prompt_lengths=[0], keys=["a"]).tolist() == [49]


def test_rows_without_rules_keep_their_results(monkeypatch):
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    monkeypatch.setattr(kernels, "repetition_penalty", lambda logits, ids, counts, row_of, pen: [
        logits.__setitem__((r, i), logits[r, i] / pen[r] ** c if logits[r, i] > 0 else logits[r, i] * pen[r] ** c)
        for i, c, r in zip(ids.tolist(), counts.tolist(), row_of.tolist())], raising=False)
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(3, 30, generator=g)
    ps = [SamplingParams(0.0, repetition_penalty=3.0), SamplingParams(0.0), SamplingParams(0.0, logit_bias={7: 99.0}, repetition_penalty=3.0)]
    recent = [[int(logits[0].argmax())] * 2, [], [7, 7]]
    got = Sampler(30, "cpu").sample(logits, ps, recent=recent, prompt_lengths=[0] * 3, keys=[0, 1, 2]).tolist()
    assert got == [sample_reference(logits[r], ps[r], recent[r]) for r in range(3)] and got[2] == 7


def test_parameters_that_are_refused():
    for bad in [dict(frequency_penalty=math.nan), dict(presence_penalty=math.inf), dict(logit_bias={50: 1.0}), dict(logit_bias={-1: 1.0}),
                dict(logit_bias={3: math.nan}), dict(logit_bias={3: math.inf}), dict(allowed_tokens=[]), dict(allowed_tokens=[1, 50]),
                dict(frequency_penalty=0.1, repetition_penalty=0.0)]:
        with pytest.raises(ValueError):
            check_params(SamplingParams(0.0, **bad), 50)
    check_params(SamplingParams(0.0, logit_bias={3: -math.inf}, allowed_tokens=range(4)), 50)


def test_ranks_and_cpu_tensors():
    assert [kernels.adapter_rank(r) for r in (1, 16, 17, 64, 65, 128)] == [16, 16, 32, 64, 128, 128]
    for r in (0, 129, -1):
        with pytest.raises(ValueError):
            kernels.adapter_rank(r)
