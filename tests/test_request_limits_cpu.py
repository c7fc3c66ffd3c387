"""What a request may bring at its limits, and what becomes of an engine and its server when a step refuses something."""
import json
import urllib.error
import urllib.request

import pytest
import torch

from polyrl_b200.models import TransformerWeights, get_model_config
from polyrl_b200.models.config import ModelConfig
from polyrl_b200.rollout.engine import RolloutEngine, SamplingParams

VOCAB = 2560


def make_engine(device="cpu", dtype=torch.float32, **kw):
    cfg = ModelConfig(**{**get_model_config("tiny-llama").to_dict(), "eos_token_id": 1, "vocab_size": VOCAB})
    w = TransformerWeights(cfg, device, dtype, seed=0)
    eng = RolloutEngine(cfg, device, **{**dict(max_num_seqs=8, max_model_len=128, seed=3), **kw})
    eng.set_weights(w.embed, w.layers, w.head)
    return cfg, w, eng


def post(url, body, timeout=60):
    req = urllib.request.Request(url, json.dumps(body).encode(), {"Content-Type": "application/json"})
    try:
        with urllib.request.urlopen(req, timeout=timeout) as r:
            return r.status, json.loads(r.read())
    except urllib.error.HTTPError as e:
        return e.code, json.loads(e.read())


def run(eng):
    while eng.has_work():
        eng.step()


def check_long_bias_lists(eng):
    for n in (1024, 1025, 2046):
        bias = {t: 0.0 for t in range(2, n + 1)}
        bias[n + 1] = 1e4                                        # the last entry decides
        ruled = eng.add_request([5, 6], SamplingParams(max_new_tokens=6, temperature=0.0, logit_bias=bias))
        plain = eng.add_request([5, 6], SamplingParams(max_new_tokens=6, temperature=0.0, presence_penalty=0.5))
        run(eng)
        assert ruled.output_ids == [n + 1] * 6 and len(bias) == n
        assert plain.finished and plain.finish_reason in ("stop", "length")
    assert eng.rules.bias_ids.shape[1] == eng.rules.bias_values.shape[1] == 2046


def test_bias_lists_up_to_the_limit():
    check_long_bias_lists(make_engine()[2])


def test_stop_tokens_outside_the_vocabulary():
    """They cannot be sampled, so there is nothing to hold back; the ones inside still wait for the least length."""
    from polyrl_b200.rollout.server import EngineServer

    eng = make_engine()[2]
    odd = (2 ** 31, 2 ** 63, VOCAB, -1, float("inf"), 7.5, 9)
    r = eng.add_request([5, 6], SamplingParams(max_new_tokens=6, temperature=0.0, min_new_tokens=4, stop_token_ids=odd, logit_bias={9: 1e4, 7: 9e3, 8: 8e3}))
    run(eng)
    assert r.output_ids == [7, 7, 7, 7, 9] and r.finish_reason == "stop"
    srv = EngineServer(eng).start()
    try:
        for stops in ([2 ** 31], [2 ** 40, 9]):
            code, got = post(f"http://{srv.endpoint}/generate", {"input_ids": [5, 6], "sampling_params": {
                "max_new_tokens": 3, "temperature": 0.0, "min_new_tokens": 1, "stop_token_ids": stops, "logit_bias": {"7": 1e4}}})
            assert code == 200 and got["output_ids"] == [7, 7, 7]
        code, got = post(f"http://{srv.endpoint}/generate", {"input_ids": [5, 6], "sampling_params": {"max_new_tokens": 3, "temperature": 0.0, "ignore_eos": True}})
        assert code == 200 and len(got["output_ids"]) == 3
    finally:
        srv.stop()
