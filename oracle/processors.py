"""Penalties, biases, grammar masks and temperature on logits, restated on the CPU in 64 bits.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  Token by token from the definition: nothing
is shared with the kernels' counting.
"""

from __future__ import annotations

from collections import Counter
from typing import Optional

import torch


def _of(value, b: int) -> float:
    return float(value[b]) if isinstance(value, torch.Tensor) else float(value)


def process_row(x: torch.Tensor, history: list, prompt: int, repetition: float, presence: float, frequency: float,
                temperature: float, bias: dict, allowed: Optional[torch.Tensor], vocab_start: int = 0,
                vocab_end: Optional[int] = None) -> torch.Tensor:
    """y [V] (float64, differentiable in x) of one row that follows the tokens ``history``."""
    V = x.shape[0]
    end = vocab_start + V if vocab_end is None else min(vocab_end, vocab_start + V)
    seen, count = Counter(history), Counter(history[prompt:])
    cols = {j - vocab_start for j in set(seen) | set(bias) if vocab_start <= j < end}
    y = x.double().clone()
    for c in sorted(cols):
        j = c + vocab_start
        z = x[c].double() + bias.get(j, 0.0)
        if seen[j]:
            z = z / repetition if z > 0 else z * repetition
        z = z - frequency * count[j] - (presence if count[j] else 0.0)
        y[c] = z
    y = y / temperature
    if allowed is not None:
        y = torch.where(allowed, y, torch.full_like(y, -float("inf")))
    return y


def process(x: torch.Tensor, ids: torch.Tensor, P, lengths: Optional[torch.Tensor] = None, vocab_start: int = 0,
            vocab_end: Optional[int] = None) -> torch.Tensor:
    """y [B, R, V] of logits x [B, R, V] under the settings P (their tensors on the CPU)."""
    B, R, V = x.shape
    rows = []
    for b in range(B):
        n = 1 if lengths is None else int(lengths[b])
        prompt = 0 if P.prompt_lengths is None else max(0, int(P.prompt_lengths[b]))
        bias = {}
        if P.bias is not None:
            at = (lambda t: t[b] if t.dim() == 2 else t)
            bias = {int(i): float(v) for i, v in zip(at(P.bias_ids), at(P.bias).float())}
        for r in range(R):
            allowed = None
            if P.grammar_masks is not None:
                m = int(P.grammar_rows[b, r])
                if 0 <= m < P.grammar_masks.shape[0]:
                    v = torch.arange(V)
                    allowed = (P.grammar_masks[m].long()[v // 32] >> (v % 32)) % 2 == 1
            rows.append(process_row(
                x[b, r], ids[b, : max(0, n + r)].tolist(), prompt, _of(P.repetition_penalty, b), _of(P.presence_penalty, b),
                _of(P.frequency_penalty, b), _of(P.temperature, b), bias, allowed, vocab_start, vocab_end))
    return torch.stack(rows).view(B, R, V) if rows else x.double()


def logprobs(x: torch.Tensor, ids: torch.Tensor, P, lengths: Optional[torch.Tensor] = None, rows: Optional[int] = None,
             vocab_start: int = 0, vocab_end: Optional[int] = None) -> torch.Tensor:
    """Logprobs [B, R] (float64, differentiable in x) of the token behind each row: 0 without one, -inf and
    no gradient where nothing is left."""
    B, R, V = x.shape
    R = R if rows is None else rows
    y = process(x[:, :R], ids, P, lengths, vocab_start, vocab_end)
    end = vocab_start + V if vocab_end is None else min(vocab_end, vocab_start + V)
    out = []
    for b in range(B):
        n = 1 if lengths is None else int(lengths[b])
        for r in range(R):
            p = n + r
            t = int(ids[b, p]) if 0 <= p < ids.shape[1] else -1
            if not vocab_start <= t < end:
                out.append(y.new_zeros(()))
            elif bool((y[b, r] == -float("inf")).all()):
                out.append(y.new_full((), -float("inf")))
            else:
                out.append(y[b, r, t - vocab_start] - torch.logsumexp(y[b, r], -1))
    return torch.stack(out).view(B, R) if out else y.new_zeros((B, R))
