"""LoRA adapters for the fused-projection transformer blocks.

The reference trains LoRA through peft on top of FSDP (``lora_rank`` / ``lora_alpha`` / ``target_modules``,
3rdparty/verl/verl/workers/fsdp_workers.py:269-577) and merges the adapters layer by layer before handing weights
to the rollout engine (verl/utils/fsdp_utils.py:569-694 "layered summon").  Here an adapter is an extra, trainable
ZeRO unit per decoder block next to a FROZEN base unit (no fp32 master / moments / gradient storage for the base:
12 bytes per base parameter saved), the low-rank path is added to the fused qkv / o / gate-up / down projections,
and ``merge_layer_`` folds ``scale * B @ A`` into a weight replica for the rollout engine.

Adapters are kept per HF projection (q/k/v/o/gate/up/down) so they export 1:1 to peft names.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import ops
from ..ops import reference as ref
from .config import ModelConfig

ALL_LINEAR = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")
_PEFT_MODULE_NAMES = {"q_proj": "self_attn.q_proj", "k_proj": "self_attn.k_proj", "v_proj": "self_attn.v_proj", "o_proj": "self_attn.o_proj",
                      "gate_proj": "mlp.gate_proj", "up_proj": "mlp.up_proj", "down_proj": "mlp.down_proj"}


@dataclass
class LoraConfig:
    rank: int = 8
    alpha: float = 16.0
    target_modules: tuple = ALL_LINEAR

    @property
    def scale(self) -> float:
        return self.alpha / self.rank

    @classmethod
    def from_model_cfg(cls, rank: int, alpha: float, target_modules, exclude_modules: str | None = None) -> "LoraConfig | None":
        """``exclude_modules``: regex over HF-style module names (``model.layers.0.self_attn.q_proj``, ``visual...``); a target whose
        name matches gets no adapter (verl model.exclude_modules, e.g. ".*visual.*" — the vision tower never carries adapters here)."""
        if not rank or rank <= 0:
            return None
        if target_modules in (None, "all-linear", "all_linear"):
            tm = ALL_LINEAR
        elif isinstance(target_modules, str):
            tm = tuple(t.strip() for t in target_modules.strip("[]").split(",") if t.strip())
        else:
            tm = tuple(target_modules)
        bad = [t for t in tm if t not in ALL_LINEAR]
        if bad:
            raise ValueError(f"unsupported LoRA target module(s) {bad}; supported: {ALL_LINEAR}")
        if exclude_modules:
            import re

            pat = re.compile(exclude_modules)
            tm = tuple(t for t in tm if not pat.fullmatch(f"model.layers.0.{_PEFT_MODULE_NAMES[t]}") and not pat.fullmatch(t))
            if not tm:
                raise ValueError(f"exclude_modules={exclude_modules!r} removes every LoRA target")
        return cls(rank=int(rank), alpha=float(alpha), target_modules=tm)


def _proj_dims(cfg: ModelConfig) -> dict[str, tuple[int, int]]:
    """projection -> (out_features, in_features)"""
    h, f, d = cfg.hidden_size, cfg.intermediate_size, cfg.head_dim
    return {"q_proj": (cfg.num_heads * d, h), "k_proj": (cfg.num_kv_heads * d, h), "v_proj": (cfg.num_kv_heads * d, h),
            "o_proj": (h, cfg.num_heads * d), "gate_proj": (f, h), "up_proj": (f, h), "down_proj": (h, f)}


def lora_param_specs(cfg: ModelConfig, lcfg: LoraConfig) -> list[tuple[str, tuple[int, ...]]]:
    if cfg.family != "llama":
        raise NotImplementedError("LoRA is implemented for the llama/qwen block family")
    dims = _proj_dims(cfg)
    specs = []
    for p in ALL_LINEAR:
        if p in lcfg.target_modules:
            out_f, in_f = dims[p]
            specs.append((f"lora_{p}_A", (lcfg.rank, in_f)))
            specs.append((f"lora_{p}_B", (out_f, lcfg.rank)))
    return specs


def _part(w: dict, proj: str):
    """The adapter of one projection, or None."""
    a = w.get(f"lora_{proj}_A")
    return None if a is None else (a, w[f"lora_{proj}_B"])


def has_lora(w: dict, *projs: str) -> bool:
    return any(f"lora_{p}_A" in w for p in projs)


def qkv_linear(cfg: ModelConfig, w: dict, h: torch.Tensor) -> torch.Tensor:
    """The fused [q | k | v] projection with the adapters of its parts."""
    if not has_lora(w, "q_proj", "k_proj", "v_proj"):
        return ops.linear(h, w["wqkv"], bias=w.get("bqkv"))
    dims = _proj_dims(cfg)
    return ops.lora_linear(h, w["wqkv"], [_part(w, p) or dims[p][0] for p in ("q_proj", "k_proj", "v_proj")], w["_lora_scale"], bias=w.get("bqkv"))


def single_linear(w: dict, x: torch.Tensor, name: str, proj: str, residual: torch.Tensor | None = None) -> torch.Tensor:
    """Projection ``w[name]`` with the adapter of ``proj``, where it has one (+ residual)."""
    if not has_lora(w, proj):
        return ops.linear(x, w[name], residual=residual)
    return ops.lora_linear(x, w[name], [_part(w, proj)], w["_lora_scale"], residual=residual)


def gate_up_swiglu(w: dict, h: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up of the block-interleaved [128 gate | 128 up] projection; adapters act before the activation."""
    if not has_lora(w, "gate_proj", "up_proj"):
        return ops.linear_swiglu(h, w["wgu"])
    return ops.lora_linear_swiglu(h, w["wgu"], _part(w, "gate_proj"), _part(w, "up_proj"), w["_lora_scale"])


@torch.no_grad()
def merge_layer_(cfg: ModelConfig, base: dict, lora: dict, scale: float) -> None:
    """In place: fold the adapters of one block into (a copy of) its fused base weights."""
    nq, nkv, d = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim

    def ba(p):
        a = lora.get(f"lora_{p}_A")
        return None if a is None else (lora[f"lora_{p}_B"].float() @ a.float()) * scale

    row = 0
    for p, rows in (("q_proj", nq * d), ("k_proj", nkv * d), ("v_proj", nkv * d)):
        m = ba(p)
        if m is not None:
            base["wqkv"][row:row + rows] += m.to(base["wqkv"].dtype)
        row += rows
    m = ba("o_proj")
    if m is not None:
        base["wo"] += m.to(base["wo"].dtype)
    g, u = ba("gate_proj"), ba("up_proj")
    if g is not None or u is not None:
        f, h = cfg.intermediate_size, cfg.hidden_size
        z = torch.zeros(f, h, device=base["wgu"].device)
        base["wgu"] += ref.interleave_gate_up(g if g is not None else z, u if u is not None else z).to(base["wgu"].dtype)
    m = ba("down_proj")
    if m is not None:
        base["wd"] += m.to(base["wd"].dtype)


_PEFT_MODULE = {"q_proj": "self_attn.q_proj", "k_proj": "self_attn.k_proj", "v_proj": "self_attn.v_proj",
                "o_proj": "self_attn.o_proj", "gate_proj": "mlp.gate_proj", "up_proj": "mlp.up_proj", "down_proj": "mlp.down_proj"}


def export_peft_state_dict(named: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
    """``layers.{i}.lora.lora_{proj}_{A|B}`` -> peft ``base_model.model.model.layers.{i}.<module>.lora_{A|B}.weight``"""
    out = {}
    for k, v in named.items():
        if ".lora.lora_" not in k:
            continue
        layer = k.split(".")[1]
        tail = k.split(".lora.lora_")[1]
        proj, ab = tail.rsplit("_", 1)
        out[f"base_model.model.model.layers.{layer}.{_PEFT_MODULE[proj]}.lora_{ab}.weight"] = v
    return out


def peft_adapter_config(cfg: ModelConfig, lcfg: LoraConfig) -> dict:
    return {"peft_type": "LORA", "r": lcfg.rank, "lora_alpha": lcfg.alpha, "target_modules": list(lcfg.target_modules),
            "bias": "none", "task_type": "CAUSAL_LM", "lora_dropout": 0.0}


def import_peft_state_dict(peft_sd: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
    """Inverse of ``export_peft_state_dict``: peft adapter tensors (any prefix up to ``layers.{i}.``, optional ``.default``
    adapter name) -> ``layers.{i}.lora.lora_{proj}_{A|B}``.  Tensors of modules this framework does not adapt are ignored."""
    import re

    inv = {v: k for k, v in _PEFT_MODULE.items()}
    out = {}
    for k, v in peft_sd.items():
        m = re.search(r"layers\.(\d+)\.((?:self_attn|mlp)\.\w+)\.lora_([AB])(?:\.\w+)?\.weight$", k)
        if m and m.group(2) in inv:
            out[f"layers.{m.group(1)}.lora.lora_{inv[m.group(2)]}_{m.group(3)}"] = v
    return out


def load_peft_adapter(engine, path: str) -> int:
    """Start the ZeRO engine's adapter units from a peft adapter directory (``adapter_model.safetensors`` / ``.bin`` next to
    ``adapter_config.json``); reference: model.lora_adapter_path, verl/workers/fsdp_workers.py (PeftModel.from_pretrained).  Rank and
    target modules must match the engine's LoRA config.  Returns the number of tensors loaded."""
    import json
    from pathlib import Path

    from .transformer import rope_feature_perm

    if rope_feature_perm(engine.cfg) is not None:
        raise NotImplementedError("peft adapters for checkpoints whose rotary layout is permuted at load time (GLM family): "
                                  "the q / k adapter rows would need the same permutation")
    p = Path(path)
    cfg_file = p / "adapter_config.json"
    if cfg_file.exists():
        ac = json.loads(cfg_file.read_text())
        if engine.lora is not None and int(ac.get("r", engine.lora.rank)) != engine.lora.rank:
            raise ValueError(f"adapter rank {ac.get('r')} != model.lora_rank {engine.lora.rank}")
    ours = import_peft_state_dict(read_peft_adapter(path)[0])
    n = 0
    for i, unit in enumerate(engine.lora_layers):
        pre = f"layers.{i}.lora."
        named = {k[len(pre):]: v for k, v in ours.items() if k.startswith(pre)}
        if named:
            missing = [name for name, _ in unit.specs if name not in named]
            if missing:
                raise KeyError(f"adapter at {path!r} lacks {missing[:3]} for layer {i} (target modules differ?)")
            unit.load_full_state(named)
            n += len(named)
    return n


# --------------------------------------------------------------------------------------------
# adapters of requests: many beside one model (rollout engine)
# --------------------------------------------------------------------------------------------
def read_peft_adapter(path: str) -> tuple[dict[str, torch.Tensor], dict]:
    """(peft tensors, adapter_config.json or {}) of a peft adapter directory."""
    import json
    from pathlib import Path

    p = Path(path)
    if (p / "adapter_model.safetensors").exists():
        from safetensors.torch import load_file

        sd = load_file(str(p / "adapter_model.safetensors"))
    elif (p / "adapter_model.bin").exists():
        sd = torch.load(p / "adapter_model.bin", map_location="cpu", weights_only=True)
    else:
        raise FileNotFoundError(f"no adapter_model.safetensors / adapter_model.bin in {path!r}")
    return sd, json.loads((p / "adapter_config.json").read_text()) if (p / "adapter_config.json").exists() else {}


class LayerAdapters:
    """The bank's adapters of one block beside its weights, for the rows of one step."""

    def __init__(self, bank: "AdapterBank", layer: int, plan):
        self.bank, self.stacks, self.plan = bank, bank.layers[layer], plan

    def linear(self, name: str, x: torch.Tensor, w, bias=None, residual=None) -> torch.Tensor:
        a, b = self.stacks[name]
        return ops.adapter_linear(x, w, a, b, self.bank.scales, self.plan, self.bank.widths[name], bias, residual)

    def swiglu(self, x: torch.Tensor, wgu) -> torch.Tensor:
        a, b = self.stacks["gate_up"]
        return ops.adapter_linear_swiglu(x, wgu, a, b, self.bank.scales, self.plan)


class AdapterBank:
    """Up to ``capacity`` adapters of a rank up to ``max_rank`` for the blocks of one model, stacked as ``ops.adapter_linear`` reads them:
    a [capacity, parts * rank, in], b [capacity, out, rank] for every fused projection.  An adapter's place is its row in the stacks; what it
    does not adapt, and the columns that its rank does not fill, are zeros.  Addresses are fixed, so captured steps see what is loaded."""

    PARTS = {"qkv": ("q_proj", "k_proj", "v_proj"), "o": ("o_proj",), "gate_up": ("gate_proj", "up_proj"), "down": ("down_proj",)}

    def __init__(self, cfg: ModelConfig, capacity: int, max_rank: int, device, dtype):
        from .transformer import rope_feature_perm

        if cfg.family != "llama" or cfg.attn_type != "mha" or cfg.num_experts or cfg.mlp_act != "swiglu":
            raise NotImplementedError("adapters of requests are implemented for dense llama / qwen blocks")
        if rope_feature_perm(cfg) is not None:
            raise NotImplementedError("adapters of requests for checkpoints whose rotary layout is permuted at load time")
        if not 1 <= capacity <= 1024 or not 1 <= max_rank <= 128:
            raise ValueError("1 to 1024 adapters of rank 1 to 128")
        self.dtype = dtype
        self.cfg, self.capacity, self.rank = cfg, capacity, -(-max_rank // 16) * 16
        self.dims = _proj_dims(cfg)
        self.widths = {n: tuple(self.dims[p][0] for p in parts) for n, parts in self.PARTS.items()}
        if any(m % 32 for ws in self.widths.values() for m in ws) or any(k % 32 for _, k in self.dims.values()):
            raise NotImplementedError("adapters of requests need widths that are multiples of 32")
        self.scales = torch.zeros(capacity, dtype=torch.float32, device=device)
        zeros = lambda *s: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
        self.layers = [{n: (zeros(capacity, len(parts) * self.rank, self.dims[parts[0]][1]), zeros(capacity, sum(self.widths[n]), self.rank))
                        for n, parts in self.PARTS.items()} for _ in range(cfg.num_layers)]
        self.names: dict[str, int] = {}

    def place(self, name: str) -> int:
        if name not in self.names:
            raise ValueError(f"no adapter {name!r} is loaded")
        return self.names[name]

    def load(self, name: str, source, alpha: float | None = None) -> int:
        """``source``: a peft adapter directory, or tensors by name (with ``alpha``, default the rank).  Returns the adapter's place."""
        if name in self.names:
            raise ValueError(f"adapter {name!r} is loaded already")
        free = sorted(set(range(self.capacity)) - set(self.names.values()))
        if not free:
            raise ValueError(f"all {self.capacity} places for adapters are taken")
        root = False
        if not isinstance(source, dict):
            source, ac = read_peft_adapter(source)
            odd = [k for k in ("use_dora", "alpha_pattern", "rank_pattern", "modules_to_save") if ac.get(k)]
            if odd or ac.get("bias", "none") != "none":
                raise NotImplementedError(f"adapter {name!r}: {', '.join(odd) or 'trained biases'} (adapter_config.json)")
            root = bool(ac.get("use_rslora"))
            alpha = float(ac["lora_alpha"]) if alpha is None and "lora_alpha" in ac else alpha
        ours = {k for k in source if ".lora.lora_" in k}
        sd = {k: source[k] for k in ours} if ours else import_peft_state_dict(source)
        if len(sd) != len(source):
            raise ValueError(f"adapter {name!r}: {len(source) - len(sd)} of its {len(source)} tensors belong to no module that is adapted here")
        ranks = {t.shape[0] for n, t in sd.items() if n.endswith("_A")}
        if len(ranks) != 1 or 0 in ranks:
            raise ValueError(f"adapter {name!r}: one rank for all of its modules expected, not {sorted(ranks)}")
        (rank,) = ranks
        if rank > self.rank:
            raise ValueError(f"adapter {name!r} has rank {rank}, the bank holds up to {self.rank}")
        known = {f"layers.{i}.lora.lora_{p}_{m}": (p, m) for i in range(self.cfg.num_layers) for p in self.dims for m in "AB"}
        for n, t in sd.items():
            if n not in known:
                raise ValueError(f"adapter {name!r}: {n} is no module of {self.cfg.name}")
            p, m = known[n]
            want = (rank, self.dims[p][1]) if m == "A" else (self.dims[p][0], rank)
            if tuple(t.shape) != want or n[:-1] + "AB"[m == "A"] not in sd:
                raise ValueError(f"adapter {name!r}: {n} is {tuple(t.shape)}, {want} and its partner expected")
            if not torch.isfinite(t.to(self.dtype)).all():      # (as the stacks hold it: zeros of other requests' rows are multiplied by it)
                raise ValueError(f"adapter {name!r}: {n} is not finite in {self.dtype}")
        scale = (rank if alpha is None else float(alpha)) / (rank ** 0.5 if root else rank)
        if not abs(scale) <= torch.finfo(torch.float32).max:
            raise ValueError(f"adapter {name!r}: a scale of {scale}")
        at = free[0]
        self._write(at, sd, rank)
        self.scales[at] = scale
        self.names[name] = at
        return at

    @torch.no_grad()
    def _write(self, at: int, sd: dict, rank: int) -> None:
        for i, stacks in enumerate(self.layers):
            for n, parts in self.PARTS.items():
                a, b = stacks[n]
                a[at].zero_()
                b[at].zero_()
                for k, (p, m) in enumerate(zip(parts, self.widths[n])):
                    ta, tb = (sd.get(f"layers.{i}.lora.lora_{p}_{x}") for x in "AB")
                    if ta is None:
                        continue
                    a[at, k * self.rank:k * self.rank + rank].copy_(ta)
                    if n == "gate_up":          # rows in blocks of 128 of gate and up, as the fused weight has them
                        b[at].view(m // 128, 2, 128, self.rank)[:, k, :, :rank].copy_(tb.view(m // 128, 128, rank))
                    else:
                        lo = sum(self.widths[n][:k])
                        b[at, lo:lo + m, :rank].copy_(tb)

    def unload(self, name: str) -> None:
        self.scales[self.place(name)] = 0.0
        del self.names[name]

    def beside(self, layers: list[dict], plan) -> list[dict]:
        """The blocks' weights with the bank's adapters beside them, for rows whose adapters the plan holds."""
        return [{**w, "_adapters": LayerAdapters(self, i, plan)} for i, w in enumerate(layers)]
