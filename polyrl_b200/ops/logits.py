"""A step's logits under the rules that each request brings: penalties for repeated tokens, biases, stop tokens that may not come yet, and
token masks (csrc/logit_rules.cu; plain PyTorch on CPU tensors).

Reference capability: the sampling parameters ``repetition_penalty``, ``presence_penalty``, ``frequency_penalty``, ``logit_bias`` and
``min_new_tokens`` of the SGLang server that the reference's rollout workers talk to."""
from __future__ import annotations

from dataclasses import dataclass, fields

import torch

MAX_HISTORY = 1 << 20          # tokens of a row's history: what the kernel's counters hold
MAX_BIAS = 2046                # entries of a row's bias list


@dataclass
class LogitRules:
    """Rules of a batch of B rows; a field that is None leaves its rule out.

    A row's history is ``tokens[b, :lens[b]]`` (``lens`` absent: all of it), the first ``prompt_lens[b]`` of them its prompt (absent: none).
    The repetition penalty falls on tokens of the whole history, presence and frequency on output tokens.  Ids outside the vocabulary
    (padding) count for nothing, in ``tokens``, ``bias_ids`` and ``stop_ids``; of bias entries with the same id the last one counts.
    ``masks`` hold a bit a token, 32 to a word, lowest bit first; ``mask_rows`` says which mask a row has (negative: none; absent: row b has
    mask b).  Stop tokens may not come while ``lens[b] < min_lens[b]``.  Where nothing is allowed the row is -inf throughout,
    and there is no token in it that ``sample_tokens`` could choose."""

    tokens: torch.Tensor | None = None         # [B, n] int32, n < 2^20
    lens: torch.Tensor | None = None           # [B] int32
    prompt_lens: torch.Tensor | None = None    # [B] int32
    repetition: torch.Tensor | None = None     # [B] fp32, 1 = none
    presence: torch.Tensor | None = None       # [B] fp32, 0 = none
    frequency: torch.Tensor | None = None      # [B] fp32, 0 = none
    bias_ids: torch.Tensor | None = None       # [B, m] int32, m <= 2046
    bias_values: torch.Tensor | None = None    # [B, m] fp32
    stop_ids: torch.Tensor | None = None       # [B, s] int32
    min_lens: torch.Tensor | None = None       # [B] int32
    masks: torch.Tensor | None = None          # [M, ceil(V / 32)] int32
    mask_rows: torch.Tensor | None = None      # [B] int32


_FLOATS = {"repetition", "presence", "frequency", "bias_values"}
_MATRICES = {"tokens", "bias_ids", "bias_values", "stop_ids", "masks"}
_NAMES = tuple(f.name for f in fields(LogitRules))


def _check(logits: torch.Tensor, r: LogitRules, out: torch.Tensor | None) -> None:
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("adjust_logits: bf16 or fp32 logits [rows, vocabulary]")
    rows, v = logits.shape
    if v >= 1 << 30:
        raise ValueError("adjust_logits: a vocabulary of less than 2^30 tokens")
    for name in _NAMES:
        t = getattr(r, name)
        if t is None:
            continue
        kind = torch.float32 if name in _FLOATS else torch.int32
        if t.dtype != kind or t.dim() != (2 if name in _MATRICES else 1) or t.device != logits.device:
            raise ValueError(f"adjust_logits: {name} must be {'[rows, n]' if name in _MATRICES else '[rows]'} {kind} on {logits.device}, "
                             f"not {t.dtype} {tuple(t.shape)} on {t.device}")
        if t.shape[0] != rows and name != "masks":
            raise ValueError(f"adjust_logits: {name} has {t.shape[0]} rows, the logits have {rows}")
    if r.tokens is None and not (r.repetition is r.presence is r.frequency is None):
        raise ValueError("adjust_logits: penalties need the rows' tokens")
    if r.tokens is not None and r.tokens.shape[1] >= MAX_HISTORY:
        raise ValueError(f"adjust_logits: a history of less than {MAX_HISTORY} tokens")
    if (r.bias_ids is None) != (r.bias_values is None) or (r.bias_ids is not None and r.bias_ids.shape != r.bias_values.shape):
        raise ValueError("adjust_logits: bias_ids and bias_values belong together")
    if r.bias_ids is not None and r.bias_ids.shape[1] > MAX_BIAS:
        raise ValueError(f"adjust_logits: at most {MAX_BIAS} biased tokens a row")
    if (r.stop_ids is None) != (r.min_lens is None) or (r.stop_ids is not None and r.lens is None):
        raise ValueError("adjust_logits: stop_ids, min_lens and lens belong together")
    if r.mask_rows is not None and r.masks is None:
        raise ValueError("adjust_logits: mask_rows without masks")
    if r.masks is not None and (r.masks.shape[1] < (v + 31) // 32 or (r.mask_rows is None and r.masks.shape[0] != rows)):
        raise ValueError("adjust_logits: masks [masks, ceil(vocabulary / 32)], one for each row unless mask_rows says which")
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device):
        raise ValueError("adjust_logits: out must be like the logits")


def adjust_logits(logits: torch.Tensor, rules: LogitRules, out: torch.Tensor | None = None) -> torch.Tensor:
    """``logits`` [B, V] (bf16 or fp32) under ``rules``, in a new tensor, in ``out``, or in place (``out=logits``), which leaves alone what
    no rule touches.  With c the times that a token is among the row's output tokens:

        z -> z / repetition if z > 0 else z * repetition      where the token is in the row's history
          -> z - frequency * c - presence                     where c > 0
          -> z + bias
          -> -inf                                             where the mask, or the least length, does not let it come

    in fp32, rounded once.  The kernel may be captured; no gradient (writing in place counts as a change of the tensor)."""
    if logits.is_cuda:                   # (checks its arguments as _check does)
        from . import ext

        r = rules
        return ext().adjust_logits(logits, out, r.tokens, r.lens, r.prompt_lens, r.repetition, r.presence, r.frequency, r.bias_ids, r.bias_values, r.stop_ids,
                                   r.min_lens, r.masks, r.mask_rows)
    _check(logits, rules, out)
    with torch.no_grad():
        z = _adjust_reference(logits, rules)
        return z if out is None else out.copy_(z)


def _adjust_reference(logits: torch.Tensor, r: LogitRules) -> torch.Tensor:
    z, (rows, v) = logits.float().clone(), logits.shape
    lens = r.lens if r.lens is not None else torch.full((rows,), r.tokens.shape[1] if r.tokens is not None else 0, dtype=torch.int32)
    for b in range(rows):
        if r.tokens is not None:
            n = min(max(int(lens[b]), 0), r.tokens.shape[1])
            p = min(max(int(r.prompt_lens[b]), 0), n) if r.prompt_lens is not None else 0
            hist = r.tokens[b, :n].long()
            inside = (hist >= 0) & (hist < v)
            seen = torch.unique(hist[inside])
            used, times = torch.unique(hist[p:][inside[p:]], return_counts=True)
            if r.repetition is not None and float(r.repetition[b]) != 1.0:
                old = z[b, seen]
                z[b, seen] = torch.where(old > 0, old / r.repetition[b], old * r.repetition[b])
            f = r.frequency[b] if r.frequency is not None else 0.0
            z[b, used] = z[b, used] - f * times.float() - (r.presence[b] if r.presence is not None else 0.0)
        if r.bias_ids is not None:
            last = {int(t): float(x) for t, x in zip(r.bias_ids[b].tolist(), r.bias_values[b].tolist()) if 0 <= t < v}
            if last:
                z[b, list(last)] += torch.tensor(list(last.values()), dtype=torch.float32)
        if r.stop_ids is not None and int(lens[b]) < int(r.min_lens[b]):
            z[b, [t for t in r.stop_ids[b].tolist() if 0 <= t < v]] = float("-inf")
        m = -1 if r.masks is None else int(r.mask_rows[b]) if r.mask_rows is not None else b
        if r.masks is not None and 0 <= m < r.masks.shape[0]:
            bits = (r.masks[m].unsqueeze(1) >> torch.arange(32, dtype=torch.int32)) & 1
            z[b, bits.reshape(-1)[:v] == 0] = float("-inf")
    return z.to(logits.dtype)


def token_mask(ids, vocab: int) -> torch.Tensor:
    """[ceil(vocab / 32)] int32 mask that lets the given tokens come."""
    ids = torch.as_tensor(list(ids), dtype=torch.long)
    if ids.numel() and not (0 <= int(ids.min()) and int(ids.max()) < vocab):
        raise ValueError(f"token ids outside the vocabulary of {vocab}")
    bits = torch.zeros((vocab + 31) // 32 * 32, dtype=torch.int64)
    bits[ids] = 1
    words = (bits.view(-1, 32) << torch.arange(32)).sum(1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
