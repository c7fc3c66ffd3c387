"""The rollout engine on the GPU with what requests bring (captured steps), and a decoder block whose adapters are trained.

Logits of bf16 steps and of a bf16 forward over the whole sequence differ by their roundings: some 16 of them on the way, each 2^-9 of the value in
the mean, so 4 * 2^-9 of a row's root mean square; a token may be the best of one and not of the other within six times that on both sides."""
import pytest
import torch

from polyrl_b200.models import TransformerWeights, get_model_config
from polyrl_b200.models import transformer as tf
from polyrl_b200.models.transformer import PackedInput
from polyrl_b200.rollout.engine import SamplingParams

from .requests_oracle import rules64
from .test_engine_requests_cpu import RULED, adapted_run, full_logits, make_adapter, make_engine, merged, rules_of, run_ruled

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SLACK = 2 * 6 * 4 * 2.0 ** -9


def engine(**kw):
    return make_engine("cuda", BF, **kw)


def check_steps(cfg, reqs, models, eng):
    for r, m in zip(reqs, models):
        z = full_logits(cfg, m, r.prompt_ids + r.output_ids).cpu()
        slack = SLACK * z.pow(2).mean().sqrt().item()
        for j, tok in enumerate(r.output_ids):
            row = z[len(r.prompt_ids) + j - 1:len(r.prompt_ids) + j]
            if r.params.has_rules:
                adj, _ = rules64(row, **rules_of(r.params, r.prompt_ids, r.output_ids[:j], eng._stop_ids(r.params)))
                far = slack * max(1.0, r.params.repetition_penalty)
            else:
                adj, far = row.double(), slack
            assert adj[0, tok] >= adj[0].max() - far, (r.params, r.adapter, j)


@pytest.mark.parametrize("sync", [1, 4])
def test_rules_in_captured_steps(sync):
    cfg, w, eng = engine(steps_per_sync=sync)
    reqs = run_ruled(eng, extra=RULED[:4])
    check_steps(cfg, reqs, [w] * len(reqs), eng)
    assert any("rules" in k for k in eng._graphs)
    eager = engine(use_cuda_graph=False, steps_per_sync=sync)[2]
    assert [r.output_ids for r in run_ruled(eager, extra=RULED[:4])] == [r.output_ids for r in reqs]
    # again, over graphs that are there
    assert [r.output_ids for r in run_ruled(eng, extra=RULED[:4])] == [r.output_ids for r in reqs]


def test_sampled_tokens_follow_the_rules():
    cfg, w, eng = engine()
    groups = eng.generate([[5, 6, 7]] * 4, SamplingParams(max_new_tokens=40, temperature=1.0, allowed_token_ids=(1, 2, 3, 4, 10), min_new_tokens=30, logit_bias={4: 3.0},
                                                          frequency_penalty=0.3, n=2))
    for r in (r for g in groups for r in g):
        assert set(r.output_ids) <= {1, 2, 3, 4, 10} and 1 not in r.output_ids[:30] and all(lp <= 0 for lp in r.logprobs)


def adapters_for(cfg, eng, w):
    sets = {"all": make_adapter(cfg, 8, 1, dtype=BF, device="cuda"), "qv": make_adapter(cfg, 16, 2, ("q_proj", "v_proj"), BF, "cuda", 1.0),
            "mlp": make_adapter(cfg, 5, 3, ("up_proj", "down_proj"), BF, "cuda", 1.0)}
    models = {None: w}
    for n, sd in sets.items():
        eng.load_adapter(n, sd, 2.0 * next(t.shape[0] for k, t in sd.items() if k.endswith("_A")))
        models[n] = merged(cfg, w, sd, 2.0, "cuda", BF)
    return models


def test_adapters_in_captured_steps():
    names = ["all", None, "qv", "mlp", "all", None, "mlp", "qv", "all", None]
    cfg, w, eng = engine(max_adapters=5, max_prefill_tokens=40)
    models = adapters_for(cfg, eng, w)
    reqs = adapted_run(eng, names)
    check_steps(cfg, reqs, [models[n] for n in names], eng)
    assert any("adapters" in k for k in eng._graphs)
    cfg, w, eager = engine(max_adapters=5, max_prefill_tokens=40, use_cuda_graph=False)
    adapters_for(cfg, eager, w)
    assert [r.output_ids for r in adapted_run(eager, names)] == [r.output_ids for r in reqs]
    # another adapter in the place of one: captured steps see it
    eng.unload_adapter("qv")
    sd = make_adapter(cfg, 8, 9, dtype=BF, device="cuda", size=1.0)
    eng.load_adapter("new", sd)
    m = merged(cfg, w, sd, 1.0, "cuda", BF)
    check_steps(cfg, adapted_run(eng, ["new", "all"]), [m, models["all"]], eng)


def test_adapters_and_rules_together_over_fp8_weights():
    for kw in (dict(), dict(weight_dtype="fp8")):
        cfg, w, eng = engine(max_adapters=3, **kw)
        models = adapters_for(cfg, eng, w)
        names = ["all", None, "mlp", "qv", None]
        torch.manual_seed(2)
        reqs = [eng.add_request(torch.randint(2, 512, (9 + i,)).tolist(), SamplingParams(max_new_tokens=14, temperature=0.0, **RULED[i]), adapter=n) for i, n in enumerate(names)]
        while eng.has_work():
            eng.step()
        assert all(r.finished and r.output_ids for r in reqs)
        if not kw:
            check_steps(cfg, reqs, [models[n] for n in names], eng)


@pytest.mark.parametrize("modules", [("q_proj", "v_proj"), ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"), ("up_proj", "o_proj")])
def test_block_with_trained_adapters(modules):
    """Forward and gradients of a block in bf16 kernels against the same block in fp32 on the CPU: the 2-norm of the difference, some twenty
    roundings of 2^-9 in the mean, within twice that."""
    cfg = get_model_config("tiny-llama")
    w = TransformerWeights(cfg, "cpu", torch.float32, seed=1).layers[0]
    w = {k: v.to(BF).float() for k, v in w.items()}
    sd = {k.split(".lora.")[1]: v.to(BF).float() for k, v in make_adapter(cfg, 8, 4, modules).items() if k.startswith("layers.0.")}
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(300, 256, generator=g).to(BF).float() for _ in range(2))
    res = {}
    for dev, dt in (("cpu", torch.float32), ("cuda", BF)):
        leaves = {"x": x.to(dev, dt).requires_grad_(), **{k: v.to(dev, dt).requires_grad_() for k, v in sd.items()}}
        wd = {**{k: v.to(dev, dt) for k, v in w.items()}, **{k: v for k, v in leaves.items() if k != "x"}, "_lora_scale": 2.0}
        cu = torch.tensor([0, 130, 300], dtype=torch.int32, device=dev)
        inp = PackedInput(torch.zeros(300, dtype=torch.long, device=dev), torch.cat([torch.arange(130), torch.arange(170)]).to(dev), cu, 170)
        y = tf.layer_forward(cfg, wd, leaves["x"], inp)
        grads = torch.autograd.grad(y, list(leaves.values()), dy.to(dev, dt))
        res[dev] = dict(zip(["y", *leaves], [t.detach().float().cpu() for t in (y, *grads)]))
    for n, want in res["cpu"].items():
        off = (res["cuda"][n] - want).norm() / want.norm()
        assert off < 2 * 20 ** 0.5 * 2.0 ** -9, (n, off.item())
