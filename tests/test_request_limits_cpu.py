"""What a request may bring at its limits, and what becomes of an engine and its server when a step refuses something."""
import json
import queue
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


def stream(srv, body, timeout=60):
    """The last payload of every index of a streamed /generate."""
    req = urllib.request.Request(f"http://{srv.endpoint}/generate", json.dumps({**body, "stream": True}).encode(), {"Content-Type": "application/json"})
    last = {}
    with urllib.request.urlopen(req, timeout=timeout) as r:
        for line in r:
            if line.startswith(b"data: {"):
                p = json.loads(line[6:])
                last[p["index"]] = p
    return last


@pytest.mark.parametrize("error", [ValueError, RuntimeError])
def test_a_step_that_fails_ends_its_requests_and_not_the_server(error):
    import threading

    from polyrl_b200.rollout.server import EngineServer

    eng = make_engine()[2]
    real, fail = eng.step, threading.Event()

    def step():
        if fail.is_set() and any(r.params.has_rules and len(r.output_ids) > 3 for r in eng.running.values()):
            fail.clear()
            raise error("no such step")
        return real()

    eng.step = step
    srv = EngineServer(eng, stream_interval=1).start()
    try:
        fail.set()
        sp = {"max_new_tokens": 60, "temperature": 0.0, "ignore_eos": True}
        out = [None, None]
        ts = [threading.Thread(target=lambda i=i, more=more: out.__setitem__(i, stream(srv, {"input_ids": [5, 6], "sampling_params": {**sp, **more}})[0]))
              for i, more in enumerate([{}, {"presence_penalty": 1.0}])]
        [t.start() for t in ts]
        [t.join(60) for t in ts]
        plain, ruled = out
        assert ruled["meta_info"]["finish_reason"]["type"] == "abort" and len(ruled["output_ids"]) > 3
        assert ("error" in ruled) == (error is ValueError) and "error" not in plain        # what is in the middle can go on elsewhere
        assert len(plain["output_ids"]) == plain["meta_info"]["completion_tokens"] == len(plain["meta_info"]["output_token_logprobs"])
        assert not eng.has_work() or not eng.running
        code, got = post(f"http://{srv.endpoint}/generate", {"input_ids": [5, 6], "sampling_params": {**sp, "presence_penalty": 1.0}})
        assert code == 200 and len(got["output_ids"]) == 60
        assert urllib.request.urlopen(f"http://{srv.endpoint}/health_generate", timeout=30).status == 200
    finally:
        srv.stop()


def test_an_engine_that_cannot_go_on_says_so():
    from polyrl_b200.rollout.server import EngineServer

    eng = make_engine()[2]

    def gone(*a, **k):
        raise RuntimeError("the device is gone")

    eng.step = eng.abort = gone
    srv = EngineServer(eng).start()
    try:
        for _ in range(2):
            code, got = post(f"http://{srv.endpoint}/generate", {"input_ids": [5, 6], "sampling_params": {"max_new_tokens": 4}})
            assert code == 200 and got["meta_info"]["finish_reason"]["type"] == "abort" and got["output_ids"] == []
        q = queue.Queue()                                       # one that was queued while the step failed
        with srv._lock:
            srv._inbox.append(("generate", ("key", [[5], [6]], SamplingParams(), q, None, None, None), None))
        assert [q.get(timeout=30)[1]["meta_info"]["finish_reason"]["type"] for _ in range(2)] == ["abort"] * 2
        with pytest.raises(urllib.error.HTTPError) as e:
            urllib.request.urlopen(f"http://{srv.endpoint}/health_generate", timeout=30)
        assert e.value.code == 503
        assert post(f"http://{srv.endpoint}/update_weights_from_agent", {"weight_version": 3})[0] == 500
    finally:
        srv.stop()


def test_steps_of_requests_without_rules_do_not_look_for_any(monkeypatch):
    asked = [0]
    has = SamplingParams.has_rules.fget

    def counted(self):
        asked[0] += 1
        return has(self)

    monkeypatch.setattr(SamplingParams, "has_rules", property(counted))
    counts = []
    for length in (4, 60):
        eng = make_engine()[2]
        asked[0] = 0
        eng.generate([[5 + i, 6] for i in range(8)], SamplingParams(max_new_tokens=length, ignore_eos=True))
        counts.append(asked[0])
    assert counts[0] == counts[1]
    r = eng.add_request([5, 6], SamplingParams(max_new_tokens=9, temperature=0.0, allowed_token_ids=(7,)))
    eng.add_request([5, 6], SamplingParams(max_new_tokens=30, ignore_eos=True))
    run(eng)
    assert r.output_ids == [7] * 9 and not eng._bringing


def test_adapters_that_the_bank_cannot_hold_are_refused():
    """Finite as they come is not enough: what the bank's type makes infinite would reach other requests, as zero times infinity."""
    from polyrl_b200.models.lora import AdapterBank

    from .test_engine_requests_cpu import make_adapter

    cfg = make_engine()[0]
    sd = make_adapter(cfg, 8, 5)
    key = "layers.1.lora.lora_o_proj_B"
    for dtype, huge in ((torch.bfloat16, torch.float32), (torch.float32, torch.float64)):
        bank = AdapterBank(cfg, 2, 16, "cpu", dtype)
        for value in (torch.finfo(huge).max, -torch.finfo(huge).max, float("nan")):
            bad = {**sd, key: torch.full_like(sd[key], value, dtype=huge)}
            with pytest.raises(ValueError, match="not finite"):
                bank.load("a", bad)
        for alpha in (float("inf"), float("nan"), 1e300):
            with pytest.raises(ValueError, match="scale"):
                bank.load("a", sd, alpha)
        with pytest.raises(ValueError, match="one rank"):
            bank.load("a", {k: v[:0] if k.endswith("_A") else v[:, :0] for k, v in sd.items()})
        assert not bank.names and not bank.scales.any() and not any(t.any() for layer in bank.layers for pair in layer.values() for t in pair)
        bank.load("a", sd, 4.0)
        assert bank.scales.tolist() == [0.5, 0.0]


def test_no_adapter_takes_the_served_models_name(tmp_path):
    from polyrl_b200.models.lora import export_peft_state_dict
    from polyrl_b200.rollout.server import EngineServer

    from .test_engine_requests_cpu import make_adapter

    cfg, _, eng = make_engine(max_adapters=2)
    sd = make_adapter(cfg, 8, 1)
    torch.save(export_peft_state_dict(sd), tmp_path / "adapter_model.bin")
    srv = EngineServer(eng, model_name="policy").start()
    try:
        code, got = post(f"http://{srv.endpoint}/load_lora_adapter", {"lora_name": "policy", "lora_path": str(tmp_path)})
        assert code == 400 and "served model" in got["message"] and not eng.adapters.names
        assert post(f"http://{srv.endpoint}/load_lora_adapter", {"lora_name": "other", "lora_path": str(tmp_path)})[0] == 200
        with urllib.request.urlopen(f"http://{srv.endpoint}/v1/models", timeout=30) as r:
            assert [d["id"] for d in json.loads(r.read())["data"]] == ["policy", "other"]
        assert srv.adapter_of("policy") is None and srv.adapter_of("other") == "other"
    finally:
        srv.stop()
    with pytest.raises(ValueError, match="served model"):
        EngineServer(eng, model_name="other")


@pytest.mark.parametrize("path,body", [("/abort_request", {"abort_all": True}), ("/release_memory_occupation", {})])
def test_an_abort_of_everything_answers_everything(path, body):
    """Nothing is left for the engine to do after it, and no step comes that would pass the last events on."""
    import threading
    import time

    from polyrl_b200.rollout.server import EngineServer

    eng = make_engine()[2]
    real = eng.step
    eng.step = lambda: (time.sleep(0.02), real())[1]
    srv = EngineServer(eng).start()
    try:
        out = [None] * 3
        req = {"input_ids": [5, 6], "sampling_params": {"max_new_tokens": 120, "temperature": 0.0, "ignore_eos": True}}
        ts = [threading.Thread(target=lambda i=i: out.__setitem__(i, post(f"http://{srv.endpoint}/generate", req))) for i in range(3)]
        [t.start() for t in ts]
        until = time.time() + 30
        while sum(len(r.output_ids) > 2 for r in list(eng.running.values())) < 3 and time.time() < until:
            time.sleep(0.01)
        assert post(f"http://{srv.endpoint}{path}", body)[0] == 200
        [t.join(30) for t in ts]
        assert all(o is not None and o[0] == 200 and o[1]["meta_info"]["finish_reason"]["type"] == "abort" and 2 < len(o[1]["output_ids"]) < 120 for o in out)
    finally:
        srv.stop()
