"""Dropout from a counter-based generator: the mask is never stored.

Whether an element is kept follows from ``(seed, offset, its number in the tensor)``, so the
backward forms the mask again from the same three (see ``rl_amd/csrc/dropout.hip`` for the
generator).  The adapters of the hidden-state logprobs drop their input by the same rule
(:mod:`rl_amd.distributed.linear_ce_adapters`).
"""

from __future__ import annotations

from typing import Any, Union

import torch
from torch.autograd.function import once_differentiable

from rl_amd import _C

__all__ = ["dropout"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, p, seed, offset):  # type: ignore[override]
        ctx.args = (p, None if isinstance(seed, torch.Tensor) else seed, offset)
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
        return _C.dropout(x, p, seed, offset)

    @staticmethod
    def backward(ctx: Any, dy):  # type: ignore[override]
        # the decorator only where a graph of the backward is asked for: it costs a small call 4 us
        return (_Dropout._once if torch.is_grad_enabled() else _Dropout._grads)(ctx, dy)

    @staticmethod
    def _grads(ctx: Any, dy):
        p, seed, offset = ctx.args
        if seed is None:
            (seed,) = ctx.saved_tensors
        return _C.dropout(dy, p, seed, offset), None, None, None

    _once = staticmethod(once_differentiable(_grads.__func__))


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], offset: int = 0,
            training: bool = True) -> torch.Tensor:
    """``x`` with each element kept with probability ``1 - p`` and multiplied by the inverse of
    that, 0 elsewhere; differentiable.

    ``seed`` (64 bits) and ``offset`` (64 bits: a layer, a step) name the mask; ``seed`` may be a
    one-element int64 tensor on x's device, which a captured graph reads anew at every replay.
    ``p`` is held to 1/65536 and the factor is that of the held value.  Without ``training``, or
    with ``p`` of 0, ``x`` itself is returned.  fp32, bf16 and fp16; the mask goes by the
    element's place in the tensor's own (row-major) order whatever its strides."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"dropout takes fp32, bf16 or fp16, got {x.dtype}")
    if not training or p == 0.0:
        return x
    return _Dropout.apply(x, float(p), seed, int(offset))
