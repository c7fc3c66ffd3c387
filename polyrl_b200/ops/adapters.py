"""Low-rank adapters beside a shared projection.

``lora_linear`` / ``lora_linear_swiglu``: a (frozen) projection with one adapter, with gradients: the trainer's LoRA path (csrc/lora.cu,
gemm2_sm100.cuh).  Reference capability: peft LoRA layers through FSDP (3rdparty/verl/verl/workers/fsdp_workers.py:269-577).

``adapter_plan`` / ``adapter_linear`` / ``adapter_linear_swiglu``: inference over rows that belong to requests with different adapters, or none
(csrc/adapters.cu; plain PyTorch on CPU tensors).  Reference capability: the adapters that the SGLang server of a rollout worker serves by
name; the reference's trainer merges its one adapter before rollout (3rdparty/verl/verl/utils/fsdp_utils.py:569-694)."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import functional as fn
from . import reference as ref


def _C():
    from . import ext

    return ext()


# --------------------------------------------------------------------------------------------
# many adapters at once (inference)
# --------------------------------------------------------------------------------------------
@dataclass
class AdapterPlan:
    """Rows sorted by adapter and cut into tiles: made once a step by ``adapter_plan``, used by every projection of the step."""

    ids: torch.Tensor            # [T] int32; outside [0, num_adapters): the row has none
    num_adapters: int
    tile_rows: int = 0
    max_tiles: int = 0
    buf: torch.Tensor | None = None


def adapter_plan(ids: torch.Tensor, num_adapters: int) -> AdapterPlan:
    """Plan of a batch whose row i belongs to adapter ``ids[i]`` (int32; a negative id, or one that is not below ``num_adapters``, means no
    adapter).  One kernel, no host synchronisation: a captured step makes its plan anew at every replay."""
    if ids.dim() != 1 or ids.dtype != torch.int32:
        raise ValueError(f"adapter_plan: one int32 id a row, not {ids.dtype} {tuple(ids.shape)}")
    if not 1 <= num_adapters <= 1024:
        raise ValueError("adapter_plan: 1 to 1024 adapters")
    t = ids.shape[0]
    if not ids.is_cuda:
        return AdapterPlan(ids, num_adapters)
    tile = 16 if t <= 256 else 32
    groups = min(num_adapters + 1, t)
    most = (t - groups) // tile + groups           # tiles: the groups' rows, each rounded up
    return AdapterPlan(ids, num_adapters, tile, most, _C().adapter_plan(ids, num_adapters, tile, most))


def _check_adapters(name: str, x, w, a, b, scales, plan: AdapterPlan, widths, bias=None, residual=None) -> None:
    n, k = w.shape
    if x.dim() != 2 or x.shape[1] != k or not x.is_floating_point():
        raise ValueError(f"{name}: rows [T, {k}] expected, not {tuple(x.shape)}")
    if plan.ids.shape[0] != x.shape[0] or plan.ids.device != x.device:
        raise ValueError(f"{name}: the plan is of {plan.ids.shape[0]} rows on {plan.ids.device}, x has {x.shape[0]} on {x.device}")
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[0] != plan.num_adapters:
        raise ValueError(f"{name}: a [{plan.num_adapters}, parts * rank, K] and b [{plan.num_adapters}, N, rank] expected, not {tuple(a.shape)} and {tuple(b.shape)}")
    if a.shape[2] != k or b.shape[1] != n or a.shape[1] != len(widths) * b.shape[2] or sum(widths) != n:
        raise ValueError(f"{name}: stacked adapters {tuple(a.shape)}, {tuple(b.shape)} do not fit a projection {tuple(w.shape)} in parts {tuple(widths)}")
    if not 1 <= len(widths) <= 3 or any(m <= 0 or m % 32 for m in widths) or k % 32 or b.shape[2] % 16 or not 16 <= b.shape[2] or len(widths) * b.shape[2] > 384:
        raise ValueError(f"{name}: one to three parts of a multiple of 32 columns, K a multiple of 32, a rank that is a multiple of 16, parts * rank at most 384")
    if scales.shape != (plan.num_adapters,) or scales.dtype != torch.float32:
        raise ValueError(f"{name}: one fp32 scale an adapter")
    if any(t.dtype != x.dtype or t.device != x.device for t in (a, b) + tuple(t for t in (bias, residual) if t is not None)):
        raise ValueError(f"{name}: adapters, bias and residual of the rows' type and device")
    if bias is not None and bias.shape != (n,) or residual is not None and residual.shape != (x.shape[0], n):
        raise ValueError(f"{name}: bias [N], residual [T, N]")


def _of_plan(name: str, a: torch.Tensor, plan: AdapterPlan) -> None:
    """The plan holds places in the stacks: of other stacks it could point behind these."""
    if a.shape[0] != plan.num_adapters:
        raise ValueError(f"{name}: a plan for {plan.num_adapters} adapters, the stacks hold {a.shape[0]}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows as the kernels read them: unit inner stride, pitch and base on 16 bytes."""
    if t.stride(-1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    t = fn._aligned(t)
    return t if t.shape[0] != 1 else t.as_strided(t.shape, (t.shape[1], 1))      # a single row counts as contiguous whatever its pitch is


def _delta(x, a, b, scales, plan, widths, interleaved, bias=None, residual=None, onto=None):
    return _C().adapter_delta(_rows(x), a, b, scales, plan.buf, plan.tile_rows, plan.max_tiles, list(widths), interleaved,
                              None if bias is None else fn._aligned(bias), None if residual is None else _rows(residual), onto)


def _together(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Many rows: whether the adapters' part goes through the large product as further k-blocks, the low-rank values of all adapters side by
    side with a row's own kept (lora.cu).  That is LR (K + N) products a row for LR = adapters * parts * rank, whichever adapters the rows have;
    a pass of its own is bound by the array of N values a row that it leaves.  The line, 2000 LR values' worth of products for one of the array's, was
    drawn before the pass of its own got faster; it is right to about a tenth but for the last size below.  The call on the device with its plan made
    before (packing of ``b`` and the shared product are part of it), apart and together, rows, K, N, LR, us: 5003, 2048, 2048, 320: 68 and 59, with 768
    69 and 76; 2900, 3584, 37888 (gate and up), 1024: 1020 and 938; 3000, 896, 9728 (gate and up), 512: 284 and 225; 700, 4096, 6144, 384: 53 and 41,
    8000 rows 353 and 370; 4000, 14336, 4096, 512, which the line puts apart: 485 and 422."""
    return a.shape[0] * a.shape[1] * (a.shape[2] + b.shape[1]) <= 2000 * b.shape[1]


def _delta_reference(x, a, b, scales, ids, widths, interleaved):
    out = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float32, device=x.device)
    n, r = b.shape[1], b.shape[2]
    part = (torch.arange(n) // 128) % 2 if interleaved else torch.repeat_interleave(torch.arange(len(widths)), torch.tensor(widths))
    part = part.to(x.device)
    for l in range(a.shape[0]):
        rows = torch.nonzero(ids == l).flatten()
        if rows.numel():
            low = (x[rows].float() @ a[l].float().t()).view(rows.numel(), len(widths), r) * scales[l]
            for i in range(len(widths)):
                cols = torch.nonzero(part == i).flatten()
                out[rows[:, None], cols] = low[:, i] @ b[l, cols].float().t()
    return out


def adapter_linear(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, plan: AdapterPlan, widths=None,
                   bias: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """Rows of ``x`` [T, K] through the shared projection ``w`` [N, K] (or an ``Fp8Weight``) and each through its own adapter l:

        y_i = w x_i + scales[l] * b[l] (a[l] x_i)  (+ bias) (+ residual_i)

    ``widths``: the columns of a fused projection's parts (query, key, value), each with ``rank`` rows of ``a`` [adapters, parts * rank, K] and
    its rows of ``b`` [adapters, N, rank]; an adapter that leaves a part alone has zeros there.  Ranks are multiples of 16 (smaller ones are
    padded with zeros).  Up to 256 rows the adapters add to what ``linear`` gives, so that a row without one is ``linear``'s bit for bit (without
    a residual).  With more rows ``b`` must be finite: rows of other adapters may be multiplied by it and zero.  Inference only."""
    widths = (w.shape[0],) if widths is None else tuple(widths)
    if plan.buf is not None and x.shape[0] <= fn._SKINNY_MAX_ROWS and fn._plain_decode(x, w):          # one call: a step of few rows is bound by the host
        return _C().adapter_linear(x, w, a, b, scales, plan.buf, plan.num_adapters, plan.tile_rows, plan.max_tiles, widths, bias, residual)
    return _adapter_linear(x, w, a, b, scales, plan, widths, bias, residual)


@torch.no_grad()
def _adapter_linear(x, w, a, b, scales, plan, widths, bias, residual):
    if not fn._is_kernel_tensor(x) or plan.buf is None:          # (the kernels' bindings check as much, but for what the plan was made for)
        _check_adapters("adapter_linear", x, w, a, b, scales, plan, widths, bias, residual)
        y = fn.linear(x, w, bias, residual)
        return (y.float() + _delta_reference(x, a, b, scales, plan.ids, widths, False)).to(x.dtype)
    _of_plan("adapter_linear", a, plan)
    if x.shape[0] <= fn._SKINNY_MAX_ROWS or isinstance(w, fn.Fp8Weight) or fn._cublas():
        return _delta(x, a, b, scales, plan, widths, False, None, residual, fn.linear(x, w, bias).contiguous())
    w = fn._g2_operand(w.to(x.dtype))
    if _together(a, b):
        return _C().adapter_gemm(_rows(x), w, a, b, scales, plan.ids, widths, False, bias if bias is None else fn._aligned(bias),
                                 residual if residual is None else fn._aligned(residual))
    d = _delta(x, a, b, scales, plan, widths, False, bias, residual)
    return _C().gemm_bf16(_rows(x), w, d)


def adapter_linear_swiglu(x: torch.Tensor, wgu: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, plan: AdapterPlan) -> torch.Tensor:
    """``linear_swiglu`` with an adapter for every row: ``a`` [adapters, 2 * rank, K] (gate, up), ``b`` [adapters, 2 F, rank] with its rows in the
    order of ``wgu``'s (blocks of 128 gate and 128 up rows); the adapters act before the activation.  Inference only."""
    n = wgu.shape[0]
    if n % 256:
        raise ValueError("adapter_linear_swiglu: gate and up in blocks of 128 rows each")
    widths = (n // 2, n // 2)
    if not isinstance(wgu, fn.Fp8Weight) and wgu.dtype != x.dtype:
        wgu = wgu.to(x.dtype)
    if not fn._is_kernel_tensor(x) or plan.buf is None or isinstance(wgu, fn.Fp8Weight) or fn._cublas():
        return _adapter_linear_swiglu(x, wgu, a, b, scales, plan, widths)
    _of_plan("adapter_linear_swiglu", a, plan)
    if x.shape[0] > fn._SKINNY_MAX_ROWS and _together(a, b):
        return _C().adapter_gemm(_rows(x), fn._g2_operand(wgu), a, b, scales, plan.ids, widths, True, None, None)
    x = _rows(x)
    d = _delta(x, a, b, scales, plan, widths, True)
    if fn._stream_swiglu(x, wgu):
        return _C().stream_gemm(x, wgu, d, None, None, None, 2, 0, None, -1)
    return _C().gemm_swiglu_add(x, wgu, d)


@torch.no_grad()
def _adapter_linear_swiglu(x, wgu, a, b, scales, plan, widths):
    if not fn._is_kernel_tensor(x) or plan.buf is None:
        _check_adapters("adapter_linear_swiglu", x, wgu, a, b, scales, plan, widths)
        gu = fn.linear(x, wgu).float() + _delta_reference(x, a, b, scales, plan.ids, widths, True)
        return ref.swiglu(gu).to(x.dtype)
    _of_plan("adapter_linear_swiglu", a, plan)
    x = _rows(x)
    d = _delta(x, a, b, scales, plan, widths, True)
    if isinstance(wgu, fn.Fp8Weight):
        xq, xs = fn.quantize_fp8_rowwise(x)
        if 0 < x.shape[0] <= fn._SKINNY_MAX_ROWS and fn._stream_impl():
            return _C().stream_gemm(xq, wgu.q, d, None, xs, wgu.scale, 2, 0, None, 0)
        return ref.swiglu(_C().gemm_fp8(xq, wgu.q, xs, wgu.scale, 0) + d)
    return ref.swiglu(d.addmm_(x, wgu.t()))


# --------------------------------------------------------------------------------------------
# one adapter, trained
# --------------------------------------------------------------------------------------------
def _lora_reference(x, w, parts, widths, scale, bias, residual, interleaved):
    """The plain form, which autograd differentiates: library products."""
    deltas = [torch.nn.functional.linear(torch.nn.functional.linear(x, p[0].to(x.dtype)), p[1].to(x.dtype)) if p is not None
              else x.new_zeros(*x.shape[:-1], m) for p, m in zip(parts, widths)]
    if interleaved:
        lead, f = x.shape[:-1], widths[0]
        d = torch.stack([t.reshape(*lead, f // 128, 128) for t in deltas], dim=-2).reshape(*lead, 2 * f)
    else:
        d = torch.cat(deltas, dim=-1) if len(deltas) > 1 else deltas[0]
    return fn.linear(x, w, bias, residual) + d * scale


def _check_lora(name, x, w, parts, bias=None, residual=None) -> tuple:
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"{name}: rows {tuple(x.shape)} do not fit a projection {tuple(w.shape)}")
    widths = []
    for p in parts:
        if isinstance(p, int):
            widths.append(p)
            continue
        a, b = p
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[1] != w.shape[1] or a.shape[0] < 1:
            raise ValueError(f"{name}: A [rank, {w.shape[1]}] and B [columns, rank] expected, not {tuple(a.shape)} and {tuple(b.shape)}")
        if a.device != x.device or b.device != x.device:
            raise ValueError(f"{name}: adapters on {a.device} and {b.device}, rows on {x.device}")
        widths.append(b.shape[0])
    if not 1 <= len(parts) <= 3 or any(m < 1 for m in widths) or sum(widths) != w.shape[0]:
        raise ValueError(f"{name}: parts of {widths} columns do not make up the projection's {w.shape[0]}")
    if bias is not None and bias.shape != w.shape[:1] or residual is not None and residual.shape != (*x.shape[:-1], w.shape[0]):
        raise ValueError(f"{name}: bias [N], residual [.., N]")
    return tuple(widths)


def _lora(x, w, parts, widths, scale, bias, residual, swiglu):
    adapters = [None if isinstance(p, int) else p for p in parts]
    kernel = fn._is_kernel_tensor(x) and not fn._cublas() and w.dtype == torch.bfloat16 and fn._g2_ok(*w.shape) and any(p is not None for p in adapters) \
        and x.numel() > 0 and all(t is None or t.dtype == torch.bfloat16 for t in (bias, residual))
    if not kernel:
        y = _lora_reference(x, w, adapters, widths, scale, bias, residual, swiglu)
        return ref.swiglu(y) if swiglu else y
    ab = [t if t is None or t.dtype == x.dtype else t.to(x.dtype) for p in adapters for t in p or (None, None)]
    if x.dim() == 2:
        return _C().lora_linear(x, w, ab, widths, float(scale), bias, residual, swiglu)
    y = _C().lora_linear(x.reshape(-1, x.shape[-1]), w, ab, widths, float(scale), bias, None if residual is None else residual.reshape(-1, w.shape[0]), swiglu)
    return y.reshape(*x.shape[:-1], y.shape[1])


def lora_linear(x: torch.Tensor, w: torch.Tensor, parts, scale: float, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """y = x @ w.T + scale * (x @ A.T) @ B.T (+ bias) (+ residual), with gradients of everything (``w`` is frozen as a rule).

    ``parts``: the projection's slices of columns in order, each an adapter (A [rank, K], B [columns, rank]) or, without one, its number of
    columns: ``[(qa, qb), 1024, (va, vb)]``.  Ranks may differ.  What the adapters add is part of the product's fp32 sums."""
    parts = list(parts)
    return _lora(x, w, parts, _check_lora("lora_linear", x, w, parts, bias, residual), scale, bias, residual, False)


def lora_linear_swiglu(x: torch.Tensor, wgu: torch.Tensor, gate, up, scale: float) -> torch.Tensor:
    """``linear_swiglu`` with adapters on gate and up (each (A [rank, K], B [F, rank]) or None), which act before the activation."""
    f = wgu.shape[0] // 2
    parts = [f if p is None else p for p in (gate, up)]
    if wgu.shape[0] % 256 or _check_lora("lora_linear_swiglu", x, wgu, parts) != (f, f):
        raise ValueError("lora_linear_swiglu: gate and up in blocks of 128 rows each")
    return _lora(x, wgu, parts, (f, f), scale, None, None, True)
