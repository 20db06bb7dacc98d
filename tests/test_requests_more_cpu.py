"""What requests bring of their own, where requests, sessions and functions come, go and fail: the engine's own logic on the CPU,
with the kernels replaced by their plain twins."""

import pytest
import torch

import plain_kernels
import plain_model
import plain_requests
from adapter_models import merged, random_adapter
from tiny_configs import CONFIGS, random_tokens

from ninfer_amd_mi50_b200 import kernels
from ninfer_amd_mi50_b200.api import Ninfer, NinferError
from ninfer_amd_mi50_b200.sampling import Sampler, SamplingParams, sample_reference
from ninfer_amd_mi50_b200.weights import write_random_model

CFG, SEED = CONFIGS["B"]
V = CFG["vocab_size"]


@pytest.fixture
def ninfer(tmp_path, monkeypatch):
    d = str(tmp_path / "B")
    write_random_model(CFG, SEED, d)
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    monkeypatch.setattr(kernels, "sample_rows", lambda logits, *a: kernels.argmax_rows(logits), raising=False)      # (some draw)
    return Ninfer(d, max_context=128, prefill_chunk=16, num_sequences=3, dtype="float32", device="cpu", page_size=16, adapters=1,
                  adapter_rank=9), plain_model.read_model_folder(d)


def test_an_adapter_stays_while_a_session_has_it(ninfer):
    eng, (pcfg, weights) = ninfer
    A, B = random_adapter(CFG, 1, 9), random_adapter(CFG, 2, 9)
    p = random_tokens(9, V, 3)
    eng.load_adapter("a", A)
    s, other = eng.session(adapter="a"), eng.session(adapter="a")
    for open_one in (s, other):
        with pytest.raises(ValueError, match="session"):
            eng.drop_adapter("a")
        with pytest.raises(ValueError):
            eng.load_adapter("b", B)                       # the only slot is taken still
        got = torch.from_numpy(open_one.prefill(p))
        torch.testing.assert_close(got, plain_model.plain_forward(pcfg, merged(weights, A, 1.0), p)[-1], rtol=1e-4, atol=1e-4)
        open_one.reset()                                   # (keeps its adapter)
        with pytest.raises(ValueError, match="session"):
            eng.drop_adapter("a")
        open_one.close()
        open_one.close()                                   # (gives it back once)
    plain = eng.session()
    eng.drop_adapter("a")
    eng.load_adapter("b", B)
    with eng.session(adapter="b") as t:
        got = torch.from_numpy(t.prefill(p))
        torch.testing.assert_close(got, plain_model.plain_forward(pcfg, merged(weights, B, 1.0), p)[-1], rtol=1e-4, atol=1e-4)
    plain.close()
    # a session that finds no place takes none of the adapter's uses with it
    full = [eng.session() for _ in range(3)]
    with pytest.raises(NinferError):
        eng.session(adapter="b")
    eng.drop_adapter("b")
    for f in full:
        f.close()


# ---- rules that together leave no token ---------------------------------------------------------------------------------------

INF = float("inf")


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_fixed_set_that_its_biases_empty_is_refused(ninfer, temperature):
    eng, _ = ninfer
    for rules in (dict(allowed_tokens=[7], logit_bias={7: -INF}), dict(allowed_tokens=[7, 7, 9], logit_bias={7: -INF, 9: -INF, 8: 1.0}),
                  dict(logit_bias={i: -INF for i in range(V)})):
        with pytest.raises(ValueError, match="leave"):
            eng.generate([[1, 2]], 3, temperature, **rules)
        with pytest.raises(ValueError, match="leave"):
            eng.sample([0.0] * V, temperature, **rules)
    drawn = eng.generate([[1, 2]], 3, temperature, allowed_tokens=[7, 9], logit_bias={7: -INF}, seed=3)
    assert drawn == [[9, 9, 9]]


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_an_answer_that_the_biases_empty_ends_the_request(ninfer, temperature):
    eng, _ = ninfer

    def answer(generated):
        return (t for t in ([5, 6] if len(generated) < 2 else [6]))

    p = SamplingParams(temperature, allowed_tokens=answer, logit_bias={6: -INF}, max_new_tokens=6, seed=1)
    rid = eng._engine.submit([1, 2, 3], p)
    eng._engine.run_until_idle()
    assert eng._engine.requests[rid].generated == [5, 5] and eng._engine.requests[rid].finish_reason == "stop"
    # by themselves, the sampler and its host twin say so instead of drawing what is not allowed
    with pytest.raises(ValueError, match="leave"):
        sample_reference([0.0] * V, p, [5, 5])
    with pytest.raises(ValueError, match="leave"):
        Sampler(V, "cpu").sample(torch.zeros(1, V), [p], recent=[[5, 5]])
    with pytest.raises(ValueError, match="leave"):
        Sampler(V, "cpu").sample(torch.zeros(1, V), [SamplingParams(temperature, allowed_tokens=lambda g: [])], recent=[[5, 5]])


# ---- logs of tokens of requests that come and go ------------------------------------------------------------------------------

def test_a_request_that_ran_out_of_cache_leaves_no_tokens_to_the_next_of_its_name(tmp_path, monkeypatch):
    d = str(tmp_path / "B")
    write_random_model(CFG, SEED, d)
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    eng = Ninfer(d, max_context=64, prefill_chunk=64, num_sequences=2, dtype="float32", device="cpu", page_size=16, cache_tokens=64)
    pcfg, weights = plain_model.read_model_folder(d)
    rules = SamplingParams(0.0, presence_penalty=100.0, frequency_penalty=1.0, max_new_tokens=30)
    s = eng.session()
    s.prefill(random_tokens(40, V, 1))                       # three of four pages
    first = eng._engine.submit(random_tokens(10, V, 2), rules, request_id="x")
    ended = []
    while not eng._engine.scheduler.idle:
        ended += eng._engine.step()
    assert [r.id for r in ended] == [first] and ended[0].finish_reason == "out_of_cache" and ended[0].generated
    assert not eng._engine.sampler.logs.slots
    s.close()
    # a prompt whose first tokens alone hold the token that the repetition penalty keeps from being drawn
    for seed in range(50):
        p = random_tokens(30, V, 3 + seed)
        a = p[0]
        p = [a] * 8 + [t for t in p if t != a][:22]
        row = plain_model.plain_forward(pcfg, weights, p)[-1]
        if row[a] < 0 and a not in ended[0].tokens:
            break
    rules = SamplingParams(0.0, repetition_penalty=10.0, presence_penalty=0.5, allowed_tokens=[a, int(row.argmin())], max_new_tokens=1)
    want = sample_reference(row, rules, p, prompt_length=len(p))
    assert want != a == sample_reference(row, rules, [], prompt_length=0)
    eng._engine.submit(p, rules, request_id="x")
    eng._engine.run_until_idle()
    assert eng._engine.requests["x"].generated == [want]


# ---- functions that fail ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bad", ["raises", "outside", "no list"])
def test_a_function_that_keeps_failing_ends_its_request_alone(ninfer, bad):
    eng, (pcfg, weights) = ninfer
    eng, asked = eng._engine, []

    def fails(generated):
        asked.append(len(generated))
        if len(generated) < 2:
            return [3, 4]
        if bad == "raises":
            raise RuntimeError("grammar")
        return [V] if bad == "outside" else 7

    kind = {"raises": RuntimeError, "outside": ValueError, "no list": TypeError}[bad]
    p = random_tokens(6, V, 2)
    rid = eng.submit(p, SamplingParams(0.0, allowed_tokens=fails, max_new_tokens=9))
    beside = eng.submit(p, SamplingParams(0.0, max_new_tokens=9))
    turn = eng.submit(p, SamplingParams(0.0, allowed_tokens=lambda g: [10 + len(g)], max_new_tokens=9))
    raised, ended = 0, []
    for _ in range(40):
        try:
            ended += eng.step()
        except kind:
            raised += 1
        if eng.scheduler.idle:
            break
    req = eng.requests[rid]
    assert raised == 1 and asked == [0, 1, 2, 2]             # the caller hears of it once, the function is asked once more
    assert req.finish_reason == "error" and isinstance(req.error, kind) and len(req.generated) == 2
    assert sorted(r.id for r in ended) == sorted([rid, beside, turn])
    assert eng.requests[beside].generated == plain_model.plain_greedy(pcfg, weights, p, 9)
    assert eng.requests[turn].generated == list(range(10, 19))
    assert not eng.cache.is_open(rid) and eng.submit(p, SamplingParams(0.0, max_new_tokens=1), request_id=rid) == rid
    eng.run_until_idle()


def test_two_functions_that_fail_and_one_that_recovers(ninfer):
    eng = ninfer[0]._engine
    count = [0]

    def recovers(generated):
        count[0] += 1
        if count[0] % 2 == 0:
            raise RuntimeError("now and then")
        return [5]

    def fails(generated):
        raise KeyError("always")

    ids = [eng.submit([1, 2], SamplingParams(0.0, allowed_tokens=f, max_new_tokens=4)) for f in (fails, recovers, fails)]
    for _ in range(40):
        try:
            eng.run_until_idle()
            break
        except (RuntimeError, KeyError):
            pass
    assert eng.scheduler.idle and [eng.requests[i].finish_reason for i in ids] == ["error", "length", "error"]
    assert eng.requests[ids[1]].generated == [5] * 4 and eng.requests[ids[1]].error is None
    # ended alone in its batch
    rid = eng.submit([1, 2], SamplingParams(0.0, allowed_tokens=fails, max_new_tokens=4))
    with pytest.raises(KeyError):
        eng.step()
    assert [r.id for r in eng.step()] == [rid] and eng.scheduler.idle


# ---- a step of the sampler that fails -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("where", ["tokens outside", "a negative token", "append", "adjust"])
def test_a_call_of_the_sampler_that_fails_loses_no_tokens(where, monkeypatch):
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    s, p = Sampler(50, "cpu"), SamplingParams(0.0, presence_penalty=100.0)
    logits = torch.arange(50.0)[None]
    draw = lambda tokens, params=p: s.sample(logits, [params], recent=[tokens], prompt_lengths=[0], keys=["a"]).tolist()
    assert draw([49]) == [48]
    with monkeypatch.context() as m:
        def broken(*a, **k):
            raise kernels.KernelError("no room")

        bad = p
        if where in ("append", "adjust"):
            m.setattr(kernels, {"append": "append_history", "adjust": "adjust_logits"}[where], broken)
        else:
            bad = SamplingParams(0.0, presence_penalty=100.0, allowed_tokens=[3, 300 if where == "tokens outside" else -1])
        with pytest.raises((kernels.KernelError, ValueError)):
            draw([49, 48, 47], bad)
    assert draw([49, 48, 47]) == [46]
    assert draw([49, 48, 47, 46]) == [45]


# ---- numbers that float32 does not hold ---------------------------------------------------------------------------------------

def test_numbers_that_are_infinite_on_the_device_are_refused(ninfer):
    from ninfer_amd_mi50_b200.sampling import check_params
    for bad in (dict(frequency_penalty=1e39), dict(presence_penalty=-1e39), dict(logit_bias={3: 1e39}), dict(logit_bias={3: -1e39}),
                dict(presence_penalty=1.0, repetition_penalty=1e-50)):
        with pytest.raises(ValueError):
            check_params(SamplingParams(0.0, **bad), 50)
    check_params(SamplingParams(0.0, frequency_penalty=3e38, presence_penalty=-3e38, logit_bias={3: 3e38, 4: -INF, 5: -3e38}), 50)
    eng, _ = ninfer
    with pytest.raises(ValueError, match="scale"):
        eng.load_adapter("a", random_adapter(CFG, 1, 9), 1e39)
    assert not eng._runner.adapters.slots


def test_a_token_that_two_biases_name_is_refused():
    from ninfer_amd_mi50_b200.sampling import check_params
    with pytest.raises(ValueError, match="twice"):
        check_params(SamplingParams(0.0, logit_bias={5: 1.0, "5": 2.0}), 50)
    p = SamplingParams(0.0, logit_bias={"5": 99.0})
    check_params(p, 50)
    assert sample_reference([0.0] * 50, p) == 5


@pytest.mark.parametrize("key,value", [("use_dora", True), ("alora_invocation_tokens", [1, 2]), ("trainable_token_indices", [3]),
                                       ("layer_replication", [[0, 2]]), ("init_lora_weights", "pissa"), ("init_lora_weights", "loftq")])
def test_a_folder_that_says_more_than_a_pair_a_tensor_is_refused(key, value, tmp_path):
    import json
    from ninfer_amd_mi50_b200.weights import SafetensorsError, read_adapter, write_safetensors
    write_safetensors(str(tmp_path / "adapter_model.safetensors"), [("m.lora_A.weight", torch.zeros(2, 4)), ("m.lora_B.weight", torch.zeros(6, 2))])
    config = {"r": 2, "lora_alpha": 4, "peft_type": "LORA", "init_lora_weights": True, "use_dora": False, "layer_replication": None}
    (tmp_path / "adapter_config.json").write_text(json.dumps(config))
    assert read_adapter(str(tmp_path))[1] == 2.0
    (tmp_path / "adapter_config.json").write_text(json.dumps(dict(config, **{key: value})))
    with pytest.raises(SafetensorsError, match=key):
        read_adapter(str(tmp_path))


def test_a_prompt_longer_than_the_tokens_is_all_of_them(monkeypatch):
    """The device reports a start beyond the log."""
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
    seen, twin = [], kernels.adjust_logits
    monkeypatch.setattr(kernels, "adjust_logits", lambda l, h, s, lengths, starts, *a, **k: (seen.append((lengths.tolist(), starts.tolist())),
                                                                                            twin(l, h, s, lengths, starts, *a, **k))[1])
    p = SamplingParams(0.0, presence_penalty=100.0)
    out = Sampler(50, "cpu").sample(torch.arange(50.0)[None], [p], recent=[[49, 48]], prompt_lengths=[5], keys=["a"])
    assert out.tolist() == [49] and seen == [([2], [2])]
