"""The rollout engine with what requests bring: rules on their logits, adapters; its server's routes for them."""
import json
import threading
import urllib.error
import urllib.request

import pytest
import torch

from polyrl_b200 import ops
from polyrl_b200.models import TransformerWeights, get_model_config
from polyrl_b200.models import transformer as tf
from polyrl_b200.models.config import ModelConfig
from polyrl_b200.models.lora import ALL_LINEAR, _proj_dims, export_peft_state_dict, merge_layer_
from polyrl_b200.models.transformer import PackedInput
from polyrl_b200.rollout.engine import RolloutEngine, SamplingParams

from .requests_oracle import rules64


def make_engine(device="cpu", dtype=torch.float32, seed=0, **kw):
    cfg = ModelConfig(**{**get_model_config("tiny-llama").to_dict(), "eos_token_id": 1})
    w = TransformerWeights(cfg, device, dtype, seed=seed)
    eng = RolloutEngine(cfg, device, **{**dict(max_num_seqs=8, max_model_len=128, seed=3), **kw})
    eng.set_weights(w.embed, w.layers, w.head)
    return cfg, w, eng


def make_adapter(cfg, rank, seed, modules=ALL_LINEAR, dtype=torch.float32, device="cpu", size=0.3):
    g = torch.Generator().manual_seed(seed)
    out = {}
    for i in range(cfg.num_layers):
        for p in modules:
            o, k = _proj_dims(cfg)[p]
            out[f"layers.{i}.lora.lora_{p}_A"] = (torch.randn(rank, k, generator=g) * k ** -0.5).to(dtype).to(device)
            out[f"layers.{i}.lora.lora_{p}_B"] = (torch.randn(o, rank, generator=g) * size * rank ** -0.5).to(dtype).to(device)
    return out


def merged(cfg, w, adapter, scale, device="cpu", dtype=torch.float32):
    m = TransformerWeights(cfg, device, dtype, init=False)
    m.load_state_dict({n: t.clone() for n, t in w.named_tensors()})
    for i in range(cfg.num_layers):
        merge_layer_(cfg, m.layers[i], {k.split(".lora.")[1]: v for k, v in adapter.items() if k.startswith(f"layers.{i}.")}, scale)
    return m


def full_logits(cfg, w, ids):
    """[n, V] logits of a sequence without any cache."""
    dev = w.embed["embed"].device
    t = torch.tensor(ids, device=dev)
    inp = PackedInput(t, torch.arange(len(ids), device=dev), torch.tensor([0, len(ids)], dtype=torch.int32, device=dev), len(ids))
    with torch.no_grad():
        return tf.logits_forward(cfg, w.head, w.embed, tf.final_norm(cfg, w.head, tf.forward_hidden(cfg, w, inp))).float()


def rules_of(p, prompt, out, stops):
    """Oracle's rules for the next token of one request."""
    t = lambda v, d=torch.int32: torch.tensor([v], dtype=d)  # noqa: E731
    kw = dict(tokens=t(prompt + out), lens=t(len(prompt) + len(out)), prompt_lens=t(len(prompt)), repetition=t(p.repetition_penalty, torch.float32),
              presence=t(p.presence_penalty, torch.float32), frequency=t(p.frequency_penalty, torch.float32))
    if p.logit_bias:
        kw |= dict(bias_ids=t(list(p.logit_bias)), bias_values=t(list(p.logit_bias.values()), torch.float32))
    if p.min_new_tokens and stops:
        kw |= dict(stop_ids=t(sorted(stops)), min_lens=t(len(prompt) + p.min_new_tokens))
    if p.allowed_token_ids is not None:
        kw |= dict(masks=ops.token_mask(p.allowed_token_ids, 512).unsqueeze(0))
    return kw


def check_ruled(cfg, w, reqs, eng, slack):
    """Every token is the best of the oracle's adjusted logits (within `slack`), and its log-prob theirs."""
    for r in reqs:
        z = full_logits(cfg, w, r.prompt_ids + r.output_ids).cpu()
        for j, tok in enumerate(r.output_ids):
            adj, _ = rules64(z[len(r.prompt_ids) + j - 1:len(r.prompt_ids) + j], **rules_of(r.params, r.prompt_ids, r.output_ids[:j], eng._stop_ids(r.params)))
            assert adj[0, tok] >= adj[0].max() - slack, (r.params, j)


RULED = [dict(repetition_penalty=1.3), dict(presence_penalty=2.0, frequency_penalty=0.5), dict(logit_bias={3: 50.0, 4: 49.0}, presence_penalty=1.5), {},
         dict(allowed_token_ids=(1, 7, 9, 11, 300, 511), frequency_penalty=1.0), dict(min_new_tokens=9, allowed_token_ids=(1, 5, 6)),
         dict(min_new_tokens=4, logit_bias={1: 1e4}), dict(logit_bias={**{t: -float("inf") for t in range(2, 500)}})]


def run_ruled(eng, extra=()):
    torch.manual_seed(0)
    reqs = [eng.add_request(torch.randint(2, 512, (5 + 3 * i,)).tolist(), SamplingParams(max_new_tokens=12 + i, temperature=0.0, **kw)) for i, kw in enumerate([*RULED, *extra])]
    while eng.has_work():
        eng.step()
    return reqs


def test_rules_in_the_engine():
    cfg, w, eng = make_engine()
    reqs = run_ruled(eng, extra=RULED[:3])                                # more requests than slots
    check_ruled(cfg, w, reqs, eng, 1e-3)
    for r, kw in zip(reqs, [*RULED, *RULED[:3]]):
        assert 1 not in r.output_ids[:kw.get("min_new_tokens", 0)]
        if "allowed_token_ids" in kw:
            assert set(r.output_ids) <= set(kw["allowed_token_ids"])
    assert reqs[6].output_ids[4] == 1 and reqs[6].finish_reason == "stop" and len(reqs[6].output_ids) == 5
    # a batch without rules is what it is in an engine that has never seen any
    plain = make_engine()[2]
    prompts = [[5, 6, 7], [9] * 20]
    a, b = (e.generate(prompts, SamplingParams(max_new_tokens=9, temperature=0.0)) for e in (eng, plain))
    assert [r.output_ids for g in a for r in g] == [r.output_ids for g in b for r in g]
    assert not (eng.rules.mask_rows >= 0).any() and (eng.rules.repetition == 1).all()


def test_rules_of_samples_of_one_prompt_and_of_moved_slots():
    cfg, w, eng = make_engine()
    long = eng.generate([[4, 5, 6, 7]], SamplingParams(max_new_tokens=20, temperature=0.0, n=6, frequency_penalty=0.7))[0]
    check_ruled(cfg, w, long, eng, 1e-3)
    assert all(r.output_ids == long[0].output_ids for r in long)
    eng = make_engine(max_num_seqs=16)[2]
    reqs = [eng.add_request([7 + i], SamplingParams(max_new_tokens=3 if i < 12 else 25, temperature=0.0, frequency_penalty=0.6 + 0.1 * i,
                                                    logit_bias={20 + i: 3.0}, allowed_token_ids=tuple(range(2 + i, 300)))) for i in range(16)]
    while eng.has_work():
        eng.step()
    check_ruled(cfg, w, reqs, eng, 1e-3)


def test_rules_of_a_request_whose_prompt_is_not_in_yet():
    cfg, w, eng = make_engine(max_prefill_tokens=16)
    prompt, late = [5, 6, 7], list(range(9, 90))
    first = eng.add_request(prompt, SamplingParams(max_new_tokens=30, temperature=0.0))
    while not first.output_ids:
        eng.step()
    second = eng.add_request(late, SamplingParams(max_new_tokens=12, temperature=0.0, presence_penalty=2.0, frequency_penalty=0.5))
    while eng.has_work():
        eng.step()
    check_ruled(cfg, w, [first, second], eng, 1e-3)
    assert len(second.output_ids) > 1


def test_stop_tokens_of_a_slots_last_request_are_forgotten():
    cfg, w, eng = make_engine(max_num_seqs=1)
    many = tuple(range(40, 52))
    eng.generate([[5, 6]], SamplingParams(max_new_tokens=4, temperature=0.0, min_new_tokens=3, stop_token_ids=many))
    r = eng.generate([[5, 6]], SamplingParams(max_new_tokens=6, temperature=0.0, min_new_tokens=5, logit_bias={45: 1e4}))[0][0]
    assert r.output_ids == [45] * 6
    check_ruled(cfg, w, [r], eng, 1e-3)


def test_rules_refused():
    cfg, w, eng = make_engine()
    for kw in [dict(repetition_penalty=0.0), dict(repetition_penalty=float("nan")), dict(presence_penalty=float("inf")), dict(min_new_tokens=-1),
               dict(logit_bias={512: 1.0}), dict(logit_bias={3: float("nan")}), dict(allowed_token_ids=()), dict(allowed_token_ids=(512,)),
               dict(allowed_token_ids=(1,), min_new_tokens=2), dict(logit_bias={t: 0.0 for t in range(2047)})]:
        with pytest.raises(ValueError):
            eng.add_request([5], SamplingParams(**kw))
    p = SamplingParams.from_dict({"logit_bias": {"7": 1}, "presence_penalty": 1, "allowed_token_ids": [3, 4], "min_new_tokens": 2, "repetition_penalty": None})
    assert p.logit_bias == {7: 1.0} and p.presence_penalty == 1.0 and p.allowed_token_ids == (3, 4) and p.min_new_tokens == 2 and p.repetition_penalty == 1.0
    assert not eng.has_work()


def test_no_rules_leave_nothing_to_sample():
    """Numbers that could take every allowed logit to -inf, and lists that ban every token, are refused; what is let in keeps a finite one."""
    cfg, w, eng = make_engine()
    ban = {t: -float("inf") for t in range(512)}
    for kw in [dict(repetition_penalty=1e-30), dict(repetition_penalty=1e30), dict(presence_penalty=1e30), dict(frequency_penalty=-1e30), dict(logit_bias={3: -1e30}),
               dict(logit_bias=ban), dict(logit_bias={t: v for t, v in ban.items() if t != 1}, min_new_tokens=1)]:
        with pytest.raises(ValueError):
            eng.add_request([5], SamplingParams(**kw))
    reqs = [eng.add_request([5, 6], SamplingParams(max_new_tokens=8, temperature=t, **kw)) for t in (0.0, 1.0, 1e-6)
            for kw in [dict(allowed_token_ids=(5,), frequency_penalty=1e20, presence_penalty=1e20, repetition_penalty=1e20), dict(allowed_token_ids=(5,), logit_bias={5: -1e20})]]
    late = eng.add_request([5, 6], SamplingParams(max_new_tokens=8, min_new_tokens=2 ** 40, logit_bias={1: 1e4}))
    while eng.has_work():
        eng.step()
    assert all(r.output_ids == [5] * 8 for r in reqs) and len(late.output_ids) == 8 and 1 not in late.output_ids
    with pytest.raises(ValueError, match="history"):
        RolloutEngine.check_request(type("E", (), dict(cfg=cfg, max_model_len=1 << 20, _stop_ids=lambda self, p: set()))(), SamplingParams(presence_penalty=1.0))


def check_adapted(cfg, reqs, weights, slack):
    """Greedy tokens of every request are those of its adapter's merged model, up to near-ties."""
    for r, m in zip(reqs, weights):
        z = full_logits(cfg, m, r.prompt_ids + r.output_ids)
        for j, tok in enumerate(r.output_ids):
            row = z[len(r.prompt_ids) + j - 1]
            assert row[tok] >= row.max() - slack, (r.adapter, j)


def adapted_run(eng, names):
    torch.manual_seed(1)
    reqs = [eng.add_request(torch.randint(2, 512, (3 + 7 * i,)).tolist(), SamplingParams(max_new_tokens=6 + i, temperature=0.0, ignore_eos=True), adapter=n)
            for i, n in enumerate(names)]
    while eng.has_work():
        eng.step()
    return reqs


def test_adapters_in_the_engine():
    cfg, w, eng = make_engine(max_adapters=3, max_adapter_rank=16, max_prefill_tokens=24)       # long prompts come in pieces
    sets = {"all": make_adapter(cfg, 8, 1), "qv": make_adapter(cfg, 16, 2, ("q_proj", "v_proj"), size=1.0), "mlp": make_adapter(cfg, 5, 3, ("up_proj", "down_proj"), size=1.0)}
    alpha = {"all": 16.0, "qv": None, "mlp": 2.5}
    for n, sd in sets.items():
        eng.load_adapter(n, sd, alpha[n])
    scale = {"all": 2.0, "qv": 1.0, "mlp": 0.5}
    models = {None: w, **{n: merged(cfg, w, sd, scale[n]) for n, sd in sets.items()}}
    names = ["all", None, "qv", "mlp", "all", None, "mlp", "qv", "all", None]
    reqs = adapted_run(eng, names)
    check_adapted(cfg, reqs, [models[n] for n in names], 2e-3)
    plain = make_engine()[2]
    base = adapted_run(plain, [None] * len(names))
    assert any(a.output_ids != b.output_ids for a, b, n in zip(reqs, base, names) if n)
    assert all(a.output_ids == b.output_ids for a, b, n in zip(reqs, base, names) if n is None)
    with pytest.raises(ValueError, match="taken"):
        eng.load_adapter("more", sets["qv"])
    eng.unload_adapter("qv")
    eng.load_adapter("again", sets["mlp"], 2.5)                                    # takes the free place; nothing of the old one is left
    check_adapted(cfg, adapted_run(eng, ["again", "all"]), [models["mlp"], models["all"]], 2e-3)


@pytest.mark.parametrize("native", ["0", "1"])
def test_adapters_do_not_share_keys(native, monkeypatch):
    """Prompts that are alike share pages within an adapter, and never across."""
    monkeypatch.setenv("POLYRL_NATIVE_KV", native)
    monkeypatch.setenv("POLYRL_NATIVE_SCHED", native)
    cfg, w, eng = make_engine(max_adapters=2, enable_prefix_cache=True)
    sd = make_adapter(cfg, 8, 4)
    eng.load_adapter("a", sd)
    m = merged(cfg, w, sd, 1.0)
    prompt, tag = list(range(30, 70)), object()
    p = SamplingParams(max_new_tokens=5, temperature=0.0, ignore_eos=True)
    reqs = [eng.add_request(prompt, p, group=tag, adapter=n) for n in (None, "a", None, "a")]
    while eng.has_work():
        eng.step()
    check_adapted(cfg, reqs, [w, m, w, m], 2e-3)
    assert reqs[0].output_ids == reqs[2].output_ids and reqs[1].output_ids == reqs[3].output_ids
    for n, want in (("a", m), (None, w), ("a", m)):
        r = eng.generate([prompt], p, adapter=n)[0][0]
        check_adapted(cfg, [r], [want], 2e-3)
        assert (r.cached_tokens > 0) == (n is None)


def test_adapters_refused(tmp_path):
    cfg, w, eng = make_engine(max_adapters=2)
    sd = make_adapter(cfg, 8, 5)
    eng.load_adapter("a", sd)
    for match, fn in [("no adapter", lambda: eng.add_request([3], {}, adapter="b")), ("loaded already", lambda: eng.load_adapter("a", sd)),
                      ("up to 16", lambda: eng.load_adapter("b", make_adapter(cfg, 17, 0))), ("one rank", lambda: eng.load_adapter("b", {})),
                      ("partner", lambda: eng.load_adapter("b", {k: v for k, v in sd.items() if not k.endswith("layers.1.lora.lora_o_proj_B")})),
                      ("no module", lambda: eng.load_adapter("b", {k.replace("layers.1", "layers.7"): v for k, v in sd.items()})),
                      ("belong to no module", lambda: eng.load_adapter("b", {**export_peft_state_dict(sd), "lm_head.lora_A.weight": torch.zeros(8, 256)})),
                      ("not finite", lambda: eng.load_adapter("b", {k: torch.full_like(v, float("inf")) if k.endswith("1.lora.lora_o_proj_B") else v for k, v in sd.items()})),
                      ("no adapter", lambda: eng.unload_adapter("b"))]:
        with pytest.raises(ValueError, match=match):
            fn()
    r = eng.add_request([3, 4], SamplingParams(max_new_tokens=2), adapter="a")
    with pytest.raises(ValueError, match="in use"):
        eng.unload_adapter("a")
    while eng.has_work():
        eng.step()
    assert r.finished
    with pytest.raises(ValueError, match="serves no adapters"):
        make_engine()[2].add_request([3], {}, adapter="a")
    d = tmp_path / "p"
    d.mkdir()
    torch.save(export_peft_state_dict(sd), d / "adapter_model.bin")
    (d / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 4, "use_dora": True}))
    with pytest.raises(NotImplementedError, match="use_dora"):
        eng.load_adapter("b", str(d))
    (d / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 4}))
    eng.load_adapter("b", str(d))
    assert eng.adapters.scales[eng.adapters.place("b")] == 0.5
    with pytest.raises(NotImplementedError):
        RolloutEngine(get_model_config("gpt2-small"), "cpu", max_adapters=1)


def test_server_routes(tmp_path):
    from polyrl_b200.rollout.server import EngineServer

    cfg, w, eng = make_engine(max_adapters=1)
    sd = make_adapter(cfg, 8, 6)
    torch.save(export_peft_state_dict(sd), tmp_path / "adapter_model.bin")
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 8, "lora_alpha": 8}))
    srv = EngineServer(eng).start()

    def post(path, body):
        req = urllib.request.Request(f"http://{srv.endpoint}{path}", json.dumps(body).encode(), {"Content-Type": "application/json"})
        try:
            with urllib.request.urlopen(req, timeout=120) as r:
                return r.status, json.loads(r.read())
        except urllib.error.HTTPError as e:
            return e.code, json.loads(e.read())

    try:
        prompt, sp = [5, 9, 30, 31], {"max_new_tokens": 5, "temperature": 0.0, "ignore_eos": True}
        assert post("/generate", {"input_ids": prompt, "sampling_params": sp, "lora_path": "mine"})[0] == 400
        assert post("/load_lora_adapter", {"lora_name": "mine"})[0] == 400
        assert post("/load_lora_adapter", {"lora_name": "mine", "lora_path": str(tmp_path / "none")})[0] == 400
        assert post("/load_lora_adapter", {"lora_name": "mine", "lora_path": str(tmp_path)})[0] == 200
        out = [None, None]
        ts = [threading.Thread(target=lambda i=i, b=b: out.__setitem__(i, post("/generate", b)))
              for i, b in enumerate([{"input_ids": prompt, "sampling_params": sp, "lora_path": "mine"}, {"input_ids": prompt, "sampling_params": sp}])]
        [t.start() for t in ts]
        [t.join() for t in ts]
        for (code, got), m in zip(out, (merged(cfg, w, sd, 1.0), w)):
            z, ids = full_logits(cfg, m, prompt + got["output_ids"]), got["output_ids"]
            assert code == 200 and all(z[len(prompt) + j - 1, t] >= z[len(prompt) + j - 1].max() - 2e-3 for j, t in enumerate(ids))
        with urllib.request.urlopen(f"http://{srv.endpoint}/v1/models", timeout=30) as r:
            assert "mine" in [d["id"] for d in json.loads(r.read())["data"]]
        code, got = post("/generate", {"input_ids": prompt, "sampling_params": {**sp, "allowed_token_ids": [8, 9]}})
        assert code == 200 and set(got["output_ids"]) <= {8, 9}
        assert post("/generate", {"input_ids": prompt, "sampling_params": {**sp, "repetition_penalty": -1}})[0] == 400
        assert post("/unload_lora_adapter", {"lora_name": "mine"})[0] == 200 and post("/unload_lora_adapter", {"lora_name": "mine"})[0] == 400
    finally:
        srv.stop()


def test_server_refuses_what_is_no_number():
    from polyrl_b200.rollout.server import EngineServer

    srv = EngineServer(make_engine()[2]).start()
    try:
        for sp in ({"min_new_tokens": float("inf")}, {"allowed_token_ids": [float("inf")]}, {"logit_bias": {"x": 1}}, {"logit_bias": [3]}, {"presence_penalty": "high"}):
            req = urllib.request.Request(f"http://{srv.endpoint}/generate", json.dumps({"input_ids": [5, 6], "sampling_params": sp}).encode(), {"Content-Type": "application/json"})
            with pytest.raises(urllib.error.HTTPError) as e:
                urllib.request.urlopen(req, timeout=60)
            assert e.value.code == 400
    finally:
        srv.stop()
