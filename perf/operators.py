"""Performance cases of the operators that adapters and per-request sampling rules need.

  lora      a projection of a frozen weight with a trained low-rank adapter beside it, forward and backward (policy update with adapters)
  adapters  a projection whose rows belong to requests with different adapters, or none (rollout and serving: decode steps and prompts)
  rules     a step's logits under each request's penalties, biases, least length and token mask (what is sampled from)

Sizes are the projections and vocabularies of the model presets.  Where ``own`` is false the operators are computed in their plain form.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

# (hidden, query width, key / value width, MLP width) of the presets
DIMS = {"qwen2.5-0.5b": (896, 896, 128, 4864), "qwen3-1.7b": (2048, 2048, 1024, 6144), "qwen2-7b": (3584, 3584, 512, 18944),
        "llama3-8b": (4096, 4096, 1024, 14336)}
VOCABS = (32768, 50257, 128256, 151936)
PROJ = ("qkv", "o", "gate_up", "down")


def listed():
    return [
        # update of a small policy on a few short sequences: launches count; fused query / key / value projection with its bias
        dict(name="lora 0.5b qkv short", kind="lora", model="qwen2.5-0.5b", proj="qkv", tokens=387, rank=8, bias=True),
        # ordinary micro-batch, adapters of a large rank on the output of the MLP
        dict(name="lora 1.7b down", kind="lora", model="qwen3-1.7b", proj="down", tokens=4099, rank=64, bias=False),
        # micro-batch of an 8B policy, usual rank
        dict(name="lora 8b qkv", kind="lora", model="llama3-8b", proj="qkv", tokens=8191, rank=16, bias=False),
        # the largest projection of the same policy: adapters act before the activation
        dict(name="lora 8b gate_up", kind="lora", model="llama3-8b", proj="gate_up", tokens=6001, rank=32, bias=False),
        # a single request's token
        dict(name="adapters one token", kind="adapters", model="qwen2.5-0.5b", proj="qkv", rows=1, runs=1, adapters=1, rank=16, bias=True),
        # decode step of a full batch, many adapters, rows in any order
        dict(name="adapters 8b decode", kind="adapters", model="llama3-8b", proj="qkv", rows=128, runs=128, adapters=24, rank=16, bias=False),
        # gate / up of a partly drained batch
        dict(name="adapters 7b decode gate_up", kind="adapters", model="qwen2-7b", proj="gate_up", rows=45, runs=45, adapters=9, rank=32, bias=False),
        # packed prompts of a few requests, output projection of the attention
        dict(name="adapters 1.7b prompts", kind="adapters", model="qwen3-1.7b", proj="o", rows=5003, runs=11, adapters=5, rank=64, bias=False),
        # one request's next token
        dict(name="rules one row", kind="rules", rows=1, vocab=151936, tokens=300, dtype="bf16"),
        # decode step of a full batch, responses of ordinary length
        dict(name="rules batch", kind="rules", rows=256, vocab=128256, tokens=1100, dtype="bf16"),
        # fp32 logits of an odd vocabulary
        dict(name="rules fp32 odd", kind="rules", rows=37, vocab=50257, tokens=700, dtype="fp32"),
        # long responses
        dict(name="rules long", kind="rules", rows=24, vocab=151936, tokens=30011, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("lora", "adapters", "rules"))
    if kind == "rules":
        rows = _log(rng, 1, 256)
        return dict(kind=kind, rows=rows, vocab=rng.choice(VOCABS), tokens=_log(rng, 8, min(32000, 600000 // rows)), dtype=rng.choice(("bf16", "bf16", "fp32")))
    model, proj = rng.choice(tuple(DIMS)), rng.choice(PROJ)
    _, k, n = _shape(model, proj)
    case = dict(kind=kind, model=model, proj=proj, rank=rng.choice((8, 16, 32, 64) if kind == "lora" else (16, 32, 64)), bias=proj == "qkv" and rng.random() < 0.5)
    if kind == "lora":
        return dict(case, tokens=_log(rng, 64, min(8192, 3.8e11 / (k * n))))
    rows, adapters = (_log(rng, 1, 256), rng.randint(1, 32)) if rng.random() < 0.6 else (_log(rng, 257, min(8192, 4e11 / (k * n))), rng.randint(1, 8))
    return dict(case, rows=rows, runs=rows if rows <= 256 else rng.randint(1, 24), adapters=adapters)


def _shape(model, proj):
    """(widths of the projection's slices, reduction length, columns)."""
    h, q, kv, f = DIMS[model]
    widths, k = {"qkv": ((q, kv, kv), h), "o": ((h,), q), "gate_up": ((f, f), h), "down": ((h,), f)}[proj]
    return widths, k, sum(widths)


def _interleave(gate, up, dim=0):
    """Gate and up as the fused weight holds them: blocks of 128 rows of each in turn."""
    f = gate.shape[dim]
    shape = gate.shape[:dim] + (f // 128, 128) + gate.shape[dim + 1:]
    return torch.cat([gate.reshape(shape), up.reshape(shape)], dim=dim + 1).reshape(gate.shape[:dim] + (2 * f,) + gate.shape[dim + 1:])


def _deinterleave(t):
    """Columns [.., 2f] of the fused projection -> gate, up."""
    v = t.unflatten(-1, (-1, 2, 128))
    return v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2)


# ------------------------------------------------------------------------------------------------------------------ inputs
def _normal(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    if case["kind"] == "rules":
        return dict(case=case, **_rules_inputs(case, g))
    widths, k, n = _shape(case["model"], case["proj"])
    r, t = case["rank"], case.get("tokens") or case["rows"]
    st = dict(case=case, widths=widths, x=_normal(g, t, k), w=_normal(g, n, k, scale=0.02), bias=_normal(g, n, scale=0.1) if case["bias"] else None)
    # the residual stream goes into the products that end a half of a block
    st["residual"] = _normal(g, t, n) if case["proj"] in ("o", "down") else None
    if case["kind"] == "lora":
        # A as initialised, B after some training; alpha twice the rank
        st["scale"] = 2.0
        st["parts"] = [(((_rand(g, r, k) * 2 - 1) * k ** -0.5).bfloat16(), _normal(g, m, r, scale=0.02)) for m in widths]
        st["dy"] = _normal(g, t, n // 2 if case["proj"] == "gate_up" else n, scale=0.01)
        return st
    num = case["adapters"]
    st["a"] = ((_rand(g, num, len(widths) * r, k) * 2 - 1) * k ** -0.5).bfloat16()
    b = [_normal(g, num, m, r, scale=0.02) for m in widths]
    st["b"] = _interleave(b[0], b[1], 1) if case["proj"] == "gate_up" else torch.cat(b, dim=1)
    st["scales"] = 0.5 + 1.5 * _rand(g, num)
    # requests: adapters at random, one in eight without one; a prompt's rows belong to one request
    of_run = torch.randint(0, num, (case["runs"],), generator=g, device="cuda").masked_fill(_rand(g, case["runs"]) < 0.125, -1)
    rng = random.Random(int(seed) * 31 + t)
    cuts = sorted(rng.sample(range(1, t), case["runs"] - 1)) if case["runs"] < t else list(range(1, t))
    lens = torch.tensor([hi - lo for lo, hi in zip([0] + cuts, cuts + [t])], device="cuda")
    st["ids"] = of_run.repeat_interleave(lens).to(torch.int32)
    return st


def _rules_inputs(case, g):
    """Requests as a server sees them: every row has a history; penalties, biases, a least length and a mask only some of them."""
    rows, v, n = case["rows"], case["vocab"], case["tokens"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    logits = _normal(g, rows, v, scale=2.0, dtype=torch.float32)
    logits += 12.0 * (_rand(g, rows, v) < 40.0 / v)                               # a few dozen likely tokens over a broad background
    lens = (n * (0.2 + 0.8 * _rand(g, rows))).int()
    lens[0] = n
    prompt = (lens * (0.1 + 0.5 * _rand(g, rows))).int()
    tokens = (v * _rand(g, rows, n) ** 4).int().clamp_(max=v - 1)                 # frequent tokens are frequent
    pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]  # noqa: E731
    m = 24
    ids = (torch.argsort(_rand(g, rows, 64), dim=1)[:, :m] * (v // 64) + torch.randint(0, v // 64, (rows, m), generator=g, device="cuda")).int()
    ids.masked_fill_(torch.arange(m, device="cuda") >= torch.randint(0, m + 1, (rows, 1), generator=g, device="cuda"), -1)     # lists of uneven length
    words, tables = (v + 31) // 32, max(1, rows // 8)
    bits = torch.randint(-2 ** 31, 2 ** 31, (6, tables, words), generator=g, device="cuda", dtype=torch.int64).int()
    masks = bits[0] & bits[1] & bits[2] & bits[3] & bits[4]                       # a grammar leaves a few of a hundred tokens
    masks[::2] |= bits[5][::2]                                                       # or half of them
    mask_rows = torch.randint(0, tables, (rows,), generator=g, device="cuda").masked_fill(_rand(g, rows) < 0.6, -1).int()
    return dict(logits=logits.to(dt), tokens=tokens, lens=lens, prompt_lens=prompt, repetition=pick([1.0, 1.0, 1.05, 1.2, 0.9]),
                presence=pick([0.0, 0.0, 0.5, 1.5]), frequency=pick([0.0, 0.0, 0.1, 0.7]), bias_ids=ids, bias_values=_normal(g, rows, m, scale=4.0, dtype=torch.float32),
                stop_ids=torch.randint(0, v, (rows, 2), generator=g, device="cuda").int(), min_lens=(lens + pick([-4, -4, 5])).int(), masks=masks, mask_rows=mask_rows)


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"lora": _run_lora, "adapters": _run_adapters, "rules": _run_rules}[state["case"]["kind"]](state)


def _run_lora(st):
    gate_up = st["case"]["proj"] == "gate_up"
    if own:
        from polyrl_b200 import ops

        x = st["x"].detach().requires_grad_()
        parts = [(a.detach().requires_grad_(), b.detach().requires_grad_()) for a, b in st["parts"]]
        if gate_up:
            y = ops.lora_linear_swiglu(x, st["w"], parts[0], parts[1], st["scale"])
        else:
            y = ops.lora_linear(x, st["w"], parts, st["scale"], bias=st["bias"], residual=st["residual"])
        leaves = [x] + [p for ab in parts for p in ab]
        grads = torch.autograd.grad(y, leaves, st["dy"])
        return [y.detach(), *grads]
    s, x, w = st["scale"], st["x"].float(), st["w"].float()
    ab = [(a.float(), b.float()) for a, b in st["parts"]]
    low = [x @ a.t() for a, _ in ab]
    deltas = [s * (t @ b.t()) for t, (_, b) in zip(low, ab)]
    y = x @ w.t() + (_interleave(deltas[0], deltas[1], 1) if gate_up else torch.cat(deltas, 1))
    dy = st["dy"].float()
    if gate_up:
        gate, up = _deinterleave(y)
        sg = torch.sigmoid(gate)
        y = gate * sg * up
        slices = [dy * up * sg * (1 + gate * (1 - sg)), dy * gate * sg]
        dy = _interleave(slices[0], slices[1], 1)
    else:
        if st["bias"] is not None:
            y = y + st["bias"].float()
        if st["residual"] is not None:
            y = y + st["residual"].float()
        slices = dy.split(st["widths"], 1)
    dx = dy @ w
    out = []
    for d, t, (a, b) in zip(slices, low, ab):
        dt = s * (d @ b)
        dx = dx + dt @ a
        out += [dt.t() @ x, s * (d.t() @ t)]
    return [v.bfloat16() for v in [y, dx, *out]]


def _run_adapters(st):
    gate_up = st["case"]["proj"] == "gate_up"
    if own:
        from polyrl_b200 import ops

        plan = ops.adapter_plan(st["ids"], st["a"].shape[0])
        if gate_up:
            return ops.adapter_linear_swiglu(st["x"], st["w"], st["a"], st["b"], st["scales"], plan)
        return ops.adapter_linear(st["x"], st["w"], st["a"], st["b"], st["scales"], plan, widths=st["widths"], bias=st["bias"], residual=st["residual"])
    x, r = st["x"].float(), st["case"]["rank"]
    num, t = st["a"].shape[0], x.shape[0]
    y = x @ st["w"].float().t()
    # every row's low-rank values under every adapter, all but its own set to zero: then one product with all of them side by side
    weight = (st["ids"].unsqueeze(1) == torch.arange(num, device="cuda")).float() * st["scales"]
    low = (x @ st["a"].float().flatten(0, 1).t()).view(t, num, len(st["widths"]), r) * weight[:, :, None, None]
    b = st["b"].float()
    if gate_up:
        halves = [h.transpose(1, 2) for h in _deinterleave(b.transpose(1, 2))]
        gate, up = _deinterleave(y)
        gate = gate + low[:, :, 0].reshape(t, -1) @ halves[0].transpose(1, 2).reshape(num * r, -1)
        up = up + low[:, :, 1].reshape(t, -1) @ halves[1].transpose(1, 2).reshape(num * r, -1)
        return (gate * torch.sigmoid(gate) * up).bfloat16()
    y = y + torch.cat([low[:, :, i].reshape(t, -1) @ h.transpose(1, 2).reshape(num * r, -1) for i, h in enumerate(b.split(st["widths"], 1))], 1)
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.bfloat16()


RULES = ("tokens", "lens", "prompt_lens", "repetition", "presence", "frequency", "bias_ids", "bias_values", "stop_ids", "min_lens", "masks", "mask_rows")


def _run_rules(st):
    if own:
        from polyrl_b200 import ops

        return ops.adjust_logits(st["logits"], ops.LogitRules(**{k: st[k] for k in RULES}))
    z = st["logits"].float()
    rows, v = z.shape
    tokens, at = st["tokens"].long(), torch.arange(st["tokens"].shape[1], device="cuda")
    prompt = (at < st["prompt_lens"][:, None]).float()
    output = (at < st["lens"][:, None]).float() - prompt
    count = torch.zeros_like(z).scatter_add_(1, tokens, output)
    seen = count + torch.zeros_like(z).scatter_add_(1, tokens, prompt) > 0
    rep = st["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0).float()
    listed_ = (st["bias_ids"] >= 0).float()
    z = z.scatter_add(1, st["bias_ids"].clamp(min=0).long(), st["bias_values"] * listed_)
    short = (st["lens"] < st["min_lens"])[:, None].float()
    banned = torch.zeros_like(z).scatter_add_(1, st["stop_ids"].long(), short.expand(-1, st["stop_ids"].shape[1])) > 0
    bit = (st["masks"].unsqueeze(2) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    refused = (bit.flatten(1)[:, :v] == 0)[st["mask_rows"].clamp(min=0).long()] & (st["mask_rows"] >= 0)[:, None]
    return z.masked_fill(banned | refused, float("-inf")).to(st["logits"].dtype)


# ------------------------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "rules":
        e = 2 if case["dtype"] == "bf16" else 4
        rows, v, n = case["rows"], case["vocab"], case["tokens"]
        return {"bytes": 2 * e * rows * v + 4 * rows * (n + 24 * 2 + 2 + 8) + 4 * max(1, rows // 8) * ((v + 31) // 32), "flops": rows * (v + 6 * n)}
    widths, k, n = _shape(case["model"], case["proj"])
    r, out = case["rank"], n // 2 if case["proj"] == "gate_up" else n
    low = len(widths) * r * k + n * r                                  # numbers of one adapter
    res = case["proj"] in ("o", "down")
    if case["kind"] == "lora":
        t = case["tokens"]
        return {"bytes": 2 * (2 * t * k + n * k + 2 * low + 2 * t * out + (t * n if res else 0)), "flops": 4 * t * k * n + 6 * t * low}
    t = case["rows"]
    used = min(case["adapters"], case["runs"])
    return {"bytes": 2 * (t * k + n * k + used * low + t * out + (t * n if res else 0)), "flops": 2 * t * k * n + 2 * t * low}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rules":
        return _exact_rules(st)
    x, w, widths, r = st["x"].double(), st["w"].double(), st["widths"], case["rank"]
    gate_up = case["proj"] == "gate_up"
    # columns of the fused projection that belong to each slice
    if gate_up:
        block = torch.arange(sum(widths), device="cuda") // 128
        cols = [torch.nonzero(block % 2 == i).flatten() for i in range(2)]
    else:
        cols = list(torch.arange(sum(widths), device="cuda").split(widths))
    extra = torch.zeros(sum(widths), dtype=torch.float64, device="cuda")
    if st["bias"] is not None:
        extra += st["bias"].double()
    if case["kind"] == "lora":
        eff = w.clone()                                                # the merged weight
        for c, (a, b) in zip(cols, st["parts"]):
            eff[c] += st["scale"] * (b.double() @ a.double())
        z = x @ eff.t() + extra
        dz = st["dy"].double()
        if gate_up:
            gate, up = z[:, cols[0]], z[:, cols[1]]
            e = 1 / (1 + torch.exp(-gate))
            y, dh = gate * e * up, dz
            dz = torch.empty_like(z)
            dz[:, cols[0]] = dh * up * (e + gate * e * (1 - e))
            dz[:, cols[1]] = dh * gate * e
        else:
            y = z if st["residual"] is None else z + st["residual"].double()
        out = [y, dz @ eff]
        for c, (a, b) in zip(cols, st["parts"]):
            dw = dz[:, c].t() @ x                                      # gradient of the merged weight's rows
            out += [st["scale"] * (b.double().t() @ dw), st["scale"] * (dw @ a.double().t())]
        return out
    z = torch.empty(x.shape[0], sum(widths), dtype=torch.float64, device="cuda")
    for i in range(-1, case["adapters"]):
        rows = torch.nonzero(st["ids"] == i).flatten()
        if rows.numel() == 0:
            continue
        z[rows] = x[rows] @ w.t() + extra
        if i >= 0:
            for s, c in enumerate(cols):
                low = x[rows] @ st["a"][i, s * r:(s + 1) * r].double().t()
                z[rows[:, None], c] += st["scales"][i].double() * (low @ st["b"][i, c].double().t())
    if gate_up:
        gate = z[:, cols[0]]
        return gate / (1 + torch.exp(-gate)) * z[:, cols[1]]
    return z if st["residual"] is None else z + st["residual"].double()


def _exact_rules(st):
    z = st["logits"].double()
    v = z.shape[1]
    for i in range(z.shape[0]):
        n, p = int(st["lens"][i]), int(st["prompt_lens"][i])
        used, times = torch.unique(st["tokens"][i, p:n].long(), return_counts=True)
        seen = torch.unique(st["tokens"][i, :n].long())
        rep = st["repetition"][i].double()
        old = z[i, seen]
        z[i, seen] = torch.where(old > 0, old / rep, old * rep)
        z[i, used] -= st["frequency"][i].double() * times + st["presence"][i].double()
        keep = st["bias_ids"][i] >= 0
        z[i, st["bias_ids"][i][keep].long()] += st["bias_values"][i][keep].double()
        if n < int(st["min_lens"][i]):
            z[i, st["stop_ids"][i].long()] = float("-inf")
        if int(st["mask_rows"][i]) >= 0:
            words = st["masks"][int(st["mask_rows"][i])].cpu().numpy().astype("<i4").view("uint8")
            allowed = np.unpackbits(words, bitorder="little")[:v]
            z[i, torch.from_numpy(allowed).cuda() == 0] = float("-inf")
    return z
