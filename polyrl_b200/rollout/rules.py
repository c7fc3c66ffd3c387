"""What requests ask of their logits (penalties, biases, least length, allowed tokens), as device state of the engine's batch slots.

The state has fixed addresses, so a decode step that applies it (``ops.adjust_logits``, in place on the step's logits) and moves it on (the
sampled token joins its row's history) is captured once.  Reference capability: the sampling parameters of the SGLang server behind the
reference's rollout workers (rlboost/verl_stream/workers/rollout/sglang_rollout/sglang_rollout_remote.py:103-182)."""
from __future__ import annotations

import math

import torch

from .. import ops
from ..ops.logits import MAX_BIAS, MAX_HISTORY, LogitRules

OVERSHOOT = 8            # tokens that a sequence may ride along after it has ended (engine: steps_per_sync)
LARGEST = 1e20           # of a penalty or a bias: a logit stays finite with all of them, 2^20 times the frequency penalty and a small temperature


def check_params(p, vocab: int, stop_ids, max_len: int) -> None:
    """Refuse what the rules cannot mean, and what could leave a step without a token to sample.  ``stop_ids``: the tokens that end the request;
    ``max_len``: of the engine's sequences."""
    if max_len + OVERSHOOT >= MAX_HISTORY:
        raise ValueError(f"rules on logits need a history of less than {MAX_HISTORY} tokens")
    if not 1 / LARGEST <= p.repetition_penalty <= LARGEST:
        raise ValueError(f"repetition_penalty must be positive, not {p.repetition_penalty}")
    if not (abs(p.presence_penalty) <= LARGEST and abs(p.frequency_penalty) <= LARGEST):
        raise ValueError(f"presence_penalty and frequency_penalty must be finite, up to {LARGEST:g}")
    if p.min_new_tokens < 0:
        raise ValueError("min_new_tokens must not be negative")
    if p.logit_bias:
        if len(p.logit_bias) > MAX_BIAS:
            raise ValueError(f"logit_bias: at most {MAX_BIAS} tokens")
        if any(not 0 <= int(t) < vocab for t in p.logit_bias) or not all(abs(float(v)) <= LARGEST or float(v) == -math.inf for v in p.logit_bias.values()):
            raise ValueError(f"logit_bias: tokens below {vocab} and numbers up to {LARGEST:g} (-inf bans a token)")
    if p.allowed_token_ids is not None and (not p.allowed_token_ids or any(not 0 <= int(t) < vocab for t in p.allowed_token_ids)):
        raise ValueError(f"allowed_token_ids: at least one token, all below {vocab}")
    banned = {int(t) for t, v in (p.logit_bias or {}).items() if float(v) == -math.inf} | (set(stop_ids) if p.min_new_tokens > 0 else set())
    if set(range(vocab) if p.allowed_token_ids is None and len(banned) >= vocab else map(int, p.allowed_token_ids or (-1,))) <= banned:
        raise ValueError("allowed_token_ids, logit_bias and min_new_tokens leave no token to sample")


class RequestRules:
    def __init__(self, slots: int, max_len: int, vocab: int, device):
        self.slots, self.width, self.vocab, self.device = slots, max_len + OVERSHOOT, vocab, device
        i32, f32 = (dict(dtype=t, device=device) for t in (torch.int32, torch.float32))
        self.tokens = torch.zeros(slots, self.width, **i32)
        self.lens = torch.zeros(slots, **i32)
        self.prompt_lens = torch.zeros(slots, **i32)
        self.repetition = torch.ones(slots, **f32)
        self.presence = torch.zeros(slots, **f32)
        self.frequency = torch.zeros(slots, **f32)
        self.min_lens = torch.zeros(slots, **i32)
        # grown when a request first needs them
        self.bias_ids = self.bias_values = self.stop_ids = self.masks = None
        self.mask_rows = torch.full((slots,), -1, **i32)
        self.version = 0                 # of the tensors: graphs captured over others are stale

    # ------------------------------------------------------------------ slots
    def _wide(self, t, need: int, fill, most: int = 1 << 30):
        """Rows of at least ``need`` columns, of ``most`` at most, what is there kept; None as long as nothing is needed."""
        have = 0 if t is None else t.shape[1]
        if need <= have:
            return t
        new = torch.full((self.slots, min(most, max(8, 1 << (need - 1).bit_length()))), fill, dtype=torch.float32 if fill == 0.0 and isinstance(fill, float) else torch.int32,
                         device=self.device)
        if have:
            new[:, :have] = t
        self.version += 1
        return new

    def set(self, slot: int, p, history: list[int], prompt_len: int, stop_ids, continued: int = 0) -> None:
        """Rules of the request that now has ``slot``; ``history``: its tokens so far, the first ``prompt_len`` of them its prompt, whose last
        ``continued`` ones count as output."""
        self.clear(slot)
        n = len(history)
        self.tokens[slot, :n] = torch.tensor(history, dtype=torch.int32).to(self.device)
        self.lens[slot], self.prompt_lens[slot] = n, prompt_len - continued
        self.repetition[slot], self.presence[slot], self.frequency[slot] = p.repetition_penalty, p.presence_penalty, p.frequency_penalty
        if p.logit_bias:
            m = len(p.logit_bias)
            self.bias_ids, self.bias_values = self._wide(self.bias_ids, m, -1, MAX_BIAS), self._wide(self.bias_values, m, 0.0, MAX_BIAS)
            self.bias_ids[slot, :m] = torch.tensor([int(t) for t in p.logit_bias], dtype=torch.int32).to(self.device)
            self.bias_values[slot, :m] = torch.tensor([float(v) for v in p.logit_bias.values()], dtype=torch.float32).to(self.device)
        stops = sorted({int(t) for t in stop_ids if 0 <= t < self.vocab and t == int(t)})        # no other can be sampled
        if p.min_new_tokens > 0 and stops:
            self.stop_ids = self._wide(self.stop_ids, len(stops), -1)
            self.stop_ids[slot, :len(stops)] = torch.tensor(stops, dtype=torch.int32).to(self.device)
            self.min_lens[slot] = prompt_len + min(p.min_new_tokens, p.max_new_tokens)
        if p.allowed_token_ids is not None:
            if self.masks is None:
                self.masks = torch.zeros(self.slots, (self.vocab + 31) // 32, dtype=torch.int32, device=self.device)
                self.version += 1
            self.masks[slot] = ops.token_mask(p.allowed_token_ids, self.vocab).to(self.device)
            self.mask_rows[slot] = slot

    def clear(self, slot: int) -> None:
        """A slot whose request has no rules."""
        self.repetition[slot], self.presence[slot], self.frequency[slot] = 1.0, 0.0, 0.0
        self.lens[slot], self.min_lens[slot], self.mask_rows[slot] = 0, 0, -1
        for t in (self.bias_ids, self.stop_ids):
            if t is not None:
                t[slot] = -1

    def move(self, src: int, dst: int) -> None:
        for t in (self.tokens, self.lens, self.prompt_lens, self.repetition, self.presence, self.frequency, self.min_lens, self.bias_ids, self.bias_values,
                  self.stop_ids, self.masks):
            if t is not None:
                t[dst] = t[src]
        self.mask_rows[dst] = torch.where(self.mask_rows[src] >= 0, dst, -1)
        self.clear(src)

    # ------------------------------------------------------------------ a step
    def _rules(self, pick) -> LogitRules:
        got = lambda t: None if t is None else pick(t)  # noqa: E731
        return LogitRules(tokens=pick(self.tokens), lens=pick(self.lens), prompt_lens=pick(self.prompt_lens), repetition=pick(self.repetition),
                          presence=pick(self.presence), frequency=pick(self.frequency), bias_ids=got(self.bias_ids), bias_values=got(self.bias_values),
                          stop_ids=got(self.stop_ids), min_lens=pick(self.min_lens) if self.stop_ids is not None else None, masks=self.masks,
                          mask_rows=pick(self.mask_rows) if self.masks is not None else None)

    def apply(self, logits: torch.Tensor) -> None:
        """In place, row b under the rules of slot b."""
        bs = logits.shape[0]
        ops.adjust_logits(logits, self._rules(lambda t: t[:bs]), out=logits)

    def apply_to(self, logits: torch.Tensor, slots: torch.Tensor) -> None:
        """In place, row i under the rules of slot ``slots[i]``."""
        ops.adjust_logits(logits, self._rules(lambda t: t.index_select(0, slots)), out=logits)

    def advance(self, tok: torch.Tensor, active: torch.Tensor) -> None:
        """The step's tokens join the histories of the active slots [0, bs)."""
        bs = tok.shape[0]
        at = self.lens[:bs].clamp(max=self.width - 1).long().unsqueeze(1)
        self.tokens[:bs].scatter_(1, at, tok.to(torch.int32).unsqueeze(1))
        self.lens[:bs].add_(active.to(torch.int32))

    def append(self, slots: torch.Tensor, tok: torch.Tensor) -> None:
        """First tokens of the requests in ``slots``."""
        at = self.lens.index_select(0, slots).long()
        self.tokens[slots, at] = tok.to(torch.int32)
        self.lens[slots] = (at + 1).to(torch.int32)
