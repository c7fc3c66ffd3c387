"""Requests that engines refuse, through the manager: the caller hears it, the engines stay."""
import json
import time

import pytest
import torch

from polyrl_b200.manager.build import build_manager
from polyrl_b200.manager.fake_engine import FakeEngine, reference_generation
from polyrl_b200.rollout.server import EngineServer

from .test_engine_requests_cpu import make_adapter, make_engine
from .test_manager import Manager, _batch, _http, _tokens

SENDER = "127.0.0.1:18861"


def join_remote(m, ports):
    """Register engines as remote instances and bring them to the manager's weight version."""
    for port in ports:
        assert _http("POST", m.url + "/register_rollout_instance", {"host": "127.0.0.1", "port": port})[0] == 200
    v = json.loads(_http("POST", m.url + "/update_weight_version")[1])["new_weight_version"]
    eps, until = [], time.time() + 30
    while len(eps) < len(ports) and time.time() < until:             # as they pass their health checks
        got = json.loads(_http("POST", m.url + "/get_receive_instances", {"weight_sender_endpoint": SENDER, "sender_weight_version": v})[1])["instances"]
        eps += [i["instance"]["endpoint"] for i in got]
        time.sleep(0.05)
    code, body = _http("POST", m.url + "/update_weights", {"instance_endpoints": eps, "weight_version": v, "tensors_meta": [], "bootstrap": False})
    assert code == 200 and json.loads(body)["success"], body
    assert ready(m) == len(ports)


def ready(m):
    return json.loads(_http("GET", m.url + "/get_instances_status")[1])["ready_instances"]


@pytest.fixture
def manager():
    m = Manager(build_manager(), "--weight-sender-rpyc-endpoints", SENDER)
    yield m
    m.close()


def test_a_refused_request_reaches_its_caller_and_keeps_the_engines(manager):
    m = manager
    servers = [EngineServer(make_engine()[2], stream_interval=2).start() for _ in range(3)]
    try:
        join_remote(m, [s.port for s in servers])
        good = {"input_ids": [5, 6], "sampling_params": {"max_new_tokens": 4, "temperature": 0.0, "ignore_eos": True}}
        bad = [{**good, "sampling_params": {"repetition_penalty": 0.0}}, {**good, "lora_path": "nope"}, {**good, "sampling_params": {"logit_bias": [3]}},
               {"text": "no ids"}]
        for b in bad:
            code, body = _http("POST", m.url + "/generate", b)
            got = json.loads(body)
            assert code == 400 and got["error_type"] == "refused" and got["error"], (b, body)
        assert "repetition_penalty must be positive" in json.loads(_http("POST", m.url + "/generate", bad[0])[1])["error"]
        lines = _batch(m, [[1, good], [2, bad[0]], [3, good], [4, bad[1]]])
        assert lines[1]["success"] and lines[3]["success"] and len(_tokens(lines[1]["data"])) == 4
        assert not lines[2]["success"] and lines[2]["status_code"] == 400 and not lines[4]["success"]
        time.sleep(0.3)
        assert ready(m) == 3 and not any(s._stop.is_set() for s in servers)
    finally:
        for s in servers:
            s.stop()


def test_an_engine_that_fails_is_still_left_for_another(manager):
    """Statuses that say nothing of the request go on as before: the engine is evicted, another one takes the request."""
    m = manager
    bad, fine = FakeEngine(), FakeEngine()
    bad._generate = lambda h, body: h._json(500, {"error": "broken"})
    try:
        join_remote(m, [bad.port, fine.port])
        for i in range(4):
            code, body = _http("POST", m.url + "/generate", {"input_ids": [3, i], "sampling_params": {"max_new_tokens": 5}})
            assert code == 200 and _tokens(json.loads(body)) == reference_generation([3, i], 5)
        assert ready(m) == 1 and bad.shutdown_called.wait(5)
    finally:
        bad.stop(); fine.stop()


def test_a_request_refused_after_it_was_queued(manager):
    """An adapter may be unloaded between a request's check and its turn: the same answer, over every route."""
    import urllib.request

    from polyrl_b200.data.rl_dataset import ByteTokenizer

    m = manager
    servers = [EngineServer(make_engine(max_adapters=1)[2], stream_interval=2, tokenizer=ByteTokenizer(), model_name="tiny").start() for _ in range(2)]
    try:
        join_remote(m, [s.port for s in servers])
        for s in servers:
            s.check_request = lambda sp, adapter: None            # it was there when the request came in
            s.adapter_of = lambda name: name if name == "gone" else None
        req = {"input_ids": [5, 6], "lora_path": "gone", "sampling_params": {"max_new_tokens": 4, "ignore_eos": True}}
        for body in (req, {**req, "input_ids": [[5, 6]] * 2}):
            code, got = _http("POST", m.url + "/generate", body)
            assert code == 400 and json.loads(got)["error_type"] == "refused" and "gone" in json.loads(got)["error"]
            code, got = _http("POST", f"http://{servers[0].endpoint}/generate", body)
            assert code == 400 and "gone" in json.loads(got)["error"]
        for n in (1, 3):
            code, got = _http("POST", f"http://{servers[0].endpoint}/v1/completions", {"model": "gone", "prompt": "abc", "max_tokens": 4, "n": n})
            assert code == 400 and "gone" in json.loads(got)["error"]["message"]
            r = urllib.request.Request(f"http://{servers[0].endpoint}/v1/completions", json.dumps({"model": "gone", "prompt": "abc", "n": n, "stream": True}).encode(),
                                       {"Content-Type": "application/json"})
            with urllib.request.urlopen(r, timeout=60) as f:
                events = [line[6:].strip() for line in f if line.startswith(b"data: ")]
            assert "gone" in json.loads(events[0])["error"]["message"] and events[-1] == b"[DONE]"
        good = {"input_ids": [5, 6], "sampling_params": {"max_new_tokens": 4, "temperature": 0.0, "ignore_eos": True}}
        assert len(_tokens(json.loads(_http("POST", m.url + "/generate", good)[1]))) == 4
        assert ready(m) == 2 and not any(s._stop.is_set() for s in servers)
    finally:
        for s in servers:
            s.stop()
