"""A request that is cut short and continued, on another engine or after an abort, has the rules of one that was not."""
import json

import pytest

from polyrl_b200.manager.build import build_manager
from polyrl_b200.manager.fake_engine import FakeEngine, reference_generation
from polyrl_b200.rollout.engine import SamplingParams
from polyrl_b200.rollout.server import EngineServer

from .test_engine_requests_cpu import make_engine
from .test_manager import Manager, _http, _tokens
from .test_manager_refusals_cpu import SENDER, join_remote

RULES = [dict(presence_penalty=1.5, frequency_penalty=0.7), dict(repetition_penalty=1.4, frequency_penalty=0.4), dict(min_new_tokens=15, logit_bias={1: 30.0}),
         dict(min_new_tokens=12, presence_penalty=2.0, logit_bias={1: 6.0, 40: 3.0, 41: 3.0}, allowed_token_ids=[1, *range(20, 120)])]
PROMPT, LENGTH = [5, 9, 30, 31, 9], 24


def uninterrupted(eng, kw):
    return eng.generate([PROMPT], SamplingParams.from_dict({"max_new_tokens": LENGTH, "temperature": 0.0, **kw}))[0][0].output_ids


@pytest.mark.parametrize("kw", RULES)
def test_continued_on_the_engine(kw):
    eng = make_engine()[2]
    want = uninterrupted(eng, kw)
    for used in sorted({u for u in (0, 1, 7, 11, 12, 13) if u < len(want)} | {len(want) - 1}):       # a finished one is not continued
        left = {**kw, "max_new_tokens": LENGTH - used, "min_new_tokens": max(0, kw.get("min_new_tokens", 0) - used), "temperature": 0.0}
        r = eng.add_request(PROMPT + want[:used], SamplingParams.from_dict(left), continued=used)
        while eng.has_work():
            eng.step()
        assert want[:used] + r.output_ids == want, used
    with pytest.raises(ValueError, match="continued"):
        eng.add_request(PROMPT, {}, continued=6)


@pytest.fixture
def manager():
    m = Manager(build_manager(), "--weight-sender-rpyc-endpoints", SENDER)
    yield m
    m.close()


@pytest.mark.parametrize("kw", RULES)
def test_continued_by_the_manager(manager, kw):
    """Engines that abort what they have at a number of tokens, one after the other: the last one finishes."""
    m = manager
    want = uninterrupted(make_engine()[2], kw)
    servers = []

    def aborting(at):
        eng = make_engine()[2]
        real = eng.step

        def step():
            done = real()
            if any(len(r.output_ids) + r.continued >= at for r in eng.running.values()):
                done += eng.abort(abort_all=True)
            return done

        eng.step = step
        return eng

    try:
        for at in (5, 10, 10 ** 6):
            servers.append(EngineServer(aborting(at), stream_interval=3).start())
        join_remote(m, [s.port for s in servers])
        for body in ([PROMPT, PROMPT], PROMPT):
            code, got = _http("POST", m.url + "/generate", {"input_ids": body, "sampling_params": {"max_new_tokens": LENGTH, "temperature": 0.0, **kw}}, timeout=120)
            assert code == 200, got
            for one in (json.loads(got) if body != PROMPT else [json.loads(got)]):
                assert _tokens(one) == want
    finally:
        for s in servers:
            s.stop()


@pytest.mark.parametrize("ids,sp", [([[3, 4], [3, 4]], {"max_new_tokens": 20, "min_new_tokens": 8}), ([3, 4], {"max_new_tokens": 20, "min_new_tokens": 3}),
                                    ([3, 4], {"max_new_tokens": 20})])
def test_what_the_manager_sends_with_a_continuation(manager, ids, sp):
    m, bodies, n = manager, [], 5

    class Engine(FakeEngine):
        def _generate(self, h, body):
            bodies.append(body)
            super()._generate(h, body)

    engines = [Engine(die_after_tokens=n), Engine()]
    try:
        join_remote(m, [e.port for e in engines])
        for _ in range(2):                                        # one of the two calls goes to the engine that dies
            code, got = _http("POST", m.url + "/generate", {"input_ids": ids, "sampling_params": sp})
            for one in (json.loads(got) if isinstance(ids[0], list) else [json.loads(got)]):
                assert code == 200 and _tokens(one) == reference_generation([3, 4], 20)
        first, (again,) = [b for b in bodies if "continued_tokens" not in b], [b for b in bodies if "continued_tokens" in b]
        assert len(first) == 2 and all(b["sampling_params"] == sp and b["input_ids"] == ids for b in first)
        longer = [3, 4] + reference_generation([3, 4], n)
        assert again["sampling_params"] == {k: max(0, v - n) for k, v in sp.items()}
        assert (again["input_ids"], again["continued_tokens"]) == (([longer] * 2, [n] * 2) if isinstance(ids[0], list) else (longer, n))
    finally:
        for e in engines:
            e.stop()


def test_counts_that_cannot_be_are_refused():
    srv = EngineServer(make_engine()[2]).start()
    try:
        for ids, n in ((PROMPT, 6), (PROMPT, -1), (PROMPT, "x"), (PROMPT, [1]), ([PROMPT, PROMPT], [1]), ([PROMPT, PROMPT], 1)):
            code, got = _http("POST", f"http://{srv.endpoint}/generate", {"input_ids": ids, "continued_tokens": n, "sampling_params": {"max_new_tokens": 2}})
            assert code == 400 and json.loads(got)["error"], (ids, n)
    finally:
        srv.stop()


@pytest.mark.parametrize("name", ["naive", "hf"])
def test_the_rollout_without_a_cache_has_the_same_rules(name):
    """It is what the engine is compared with: greedy tokens and log-probs of all rules agree."""
    from polyrl_b200.rollout.registry import get_rollout_cls

    cfg, w, eng = make_engine()
    plain = get_rollout_cls(name)(cfg, "cpu", max_model_len=128)
    plain.set_weights(w.embed, w.layers, w.head)
    prompts = [PROMPT, [4] * 20, [7, 300]]
    for kw in RULES:
        p = SamplingParams.from_dict({"max_new_tokens": LENGTH, "temperature": 0.0, **kw})
        for a, b in zip(eng.generate(prompts, p), plain.generate(prompts, p)):
            assert a[0].output_ids == b[0].output_ids and max(abs(x - y) for x, y in zip(a[0].logprobs, b[0].logprobs)) < 1e-4, kw
    with pytest.raises(ValueError, match="repetition_penalty"):
        plain.generate(prompts, {"repetition_penalty": 0.0})


def test_least_lengths_reach_the_library_engine_up_to_the_limit(monkeypatch):
    """The native engine holds stop tokens back to the last token at most; the library refuses a least length beyond the limit."""
    import sys

    from polyrl_b200.rollout.vllm_adapter import VLLMRollout

    monkeypatch.setitem(sys.modules, "vllm", None)                    # parameters stay a dict
    roll = VLLMRollout(make_engine()[0], "cpu", llm=object())
    for least, most, want in ((5, 9, 5), (9, 9, 9), (10 ** 6, 9, 9)):
        kw = roll._sampling_params(SamplingParams(max_new_tokens=most, min_new_tokens=least))
        assert (kw["min_tokens"], kw["max_tokens"]) == (want, most)
