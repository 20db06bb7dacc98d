"""What requests bring of their own, where requests, sessions and functions come, go and fail: the engine's own logic on the CPU,
with the kernels replaced by their plain twins."""

import pytest
import torch

import plain_kernels
import plain_model
import plain_requests
from adapter_models import merged, random_adapter
from tiny_configs import CONFIGS, random_tokens

from ninfer_amd_mi50_b200.api import Ninfer, NinferError
from ninfer_amd_mi50_b200.weights import write_random_model

CFG, SEED = CONFIGS["B"]
V = CFG["vocab_size"]


@pytest.fixture
def ninfer(tmp_path, monkeypatch):
    d = str(tmp_path / "B")
    write_random_model(CFG, SEED, d)
    plain_kernels.install(monkeypatch)
    plain_requests.install(monkeypatch)
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
