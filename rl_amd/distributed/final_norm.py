"""The norm in front of the output weight: RMS norm with the residual's addition.

What a policy does with its residual stream before the hidden-state logprobs
(:mod:`rl_amd.distributed.linear_ce`): ``h = x + residual``, ``y = h / rms(h) * weight``.
:func:`add_rms_norm` is differentiable; :func:`add_rms_norm_8bit` writes the rows in e4m3
with one scale each, as :func:`~rl_amd.distributed.linear_ce_8bit.from_parallel_8bit_hidden_states_to_logprobs`
reads them, for passes that need no gradient (the previous or the reference policy's
logprobs); :func:`quantize_rows_8bit` does the same to an output weight, once.

Types: rows of fp32, bf16 or fp16; the residual, and with it the returned stream, of the
rows' type or fp32; the weight of the rows' type or fp32.  Sums are fp32, every output is
rounded once, and the norm reads the stream as it is stored, so that ``add_rms_norm`` is an
addition followed by a norm.
"""

from __future__ import annotations

from typing import Any, Optional

import torch
from torch.autograd.function import once_differentiable

from rl_amd import _C

__all__ = ["add_rms_norm", "add_rms_norm_8bit", "quantize_rows_8bit", "rms_norm"]

_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float) -> None:
    dtype, shape = x.dtype, x.shape
    if dtype not in _ROW_DTYPES:
        raise TypeError(f"the norm takes fp32, bf16 or fp16 rows, got {dtype}")
    if not shape or shape[-1] == 0:
        raise ValueError(f"expected rows [..., H], got {tuple(shape)}")
    if weight.shape != shape[-1:]:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match rows of {shape[-1]}")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise TypeError(f"the weight has the rows' type {dtype} or float32, got {weight.dtype}")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} does not match {tuple(shape)}")
        if residual.dtype != dtype and residual.dtype != torch.float32:
            raise TypeError(f"the residual has the rows' type {dtype} or float32, got {residual.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")


class _AddRmsNorm(torch.autograd.Function):
    """(y, h) of x, the residual and the weight.  What is kept for the backward: h, one fp32
    per row, the weight."""

    @staticmethod
    def forward(ctx: Any, x, residual, weight, eps):  # type: ignore[override]
        y, h, rstd, _ = _C.add_rms_norm_fwd(x, residual, weight, eps, True, False)
        ctx.save_for_backward(h, rstd, weight)
        ctx.set_materialize_grads(False)
        ctx.x_dtype = x.dtype
        return y, h

    @staticmethod
    def backward(ctx: Any, dy, dh):  # type: ignore[override]
        # the decorator only where a graph of the backward is asked for: it costs a small call 4 us
        return (_AddRmsNorm._once if torch.is_grad_enabled() else _AddRmsNorm._grads)(ctx, dy, dh)

    @staticmethod
    def _grads(ctx: Any, dy, dh):
        h, rstd, weight = ctx.saved_tensors
        need_x, need_res, need_w = ctx.needs_input_grad[:3]
        if dy is None:  # only the stream has a consumer
            return (dh.to(ctx.x_dtype) if need_x else None), (dh if need_res else None), None, None
        dx, dres, dw = _C.add_rms_norm_bwd(dy, dh, h, rstd, weight, need_x, need_res, need_w)
        return dx, dres, dw, None

    _once = staticmethod(once_differentiable(_grads.__func__))


class _RmsNorm(torch.autograd.Function):
    """y of x and the weight."""

    @staticmethod
    def forward(ctx: Any, x, weight, eps):  # type: ignore[override]
        y, _, rstd, _ = _C.add_rms_norm_fwd(x, None, weight, eps, True, False)
        ctx.save_for_backward(x, rstd, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy):  # type: ignore[override]
        x, rstd, weight = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        dx, _, dw = _C.add_rms_norm_bwd(dy, None, x, rstd, weight, need_x, False, need_w)
        return dx, dw, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)``: the stream ``h = x + residual`` in the residual's type and its RMS norm
    ``y = h / sqrt(mean(h^2) + eps) * weight`` in x's; both differentiable."""
    _check(x, residual, weight, eps)
    return _AddRmsNorm.apply(x, residual, weight, float(eps))


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, differentiable."""
    _check(x, None, weight, eps)
    return _RmsNorm.apply(x, weight, float(eps))


def add_rms_norm_8bit(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y8, scale, h)``: as :func:`add_rms_norm`, with ``y`` in e4m3 (``float8_e4m3fn``) and one
    fp32 scale per row, ``y = y8 * scale``, rounded from the fp32 ``y``.  ``residual`` may be None
    (``h`` is then ``x``).  No gradient passes through: inputs that ask for one are refused
    unless gradients are off."""
    _check(x, residual, weight, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError("an 8-bit norm has no gradient: call it under torch.no_grad() or use add_rms_norm")
    y8, h, _, scale = _C.add_rms_norm_fwd(x, residual, weight, eps, False, True)
    return y8, scale, h


def quantize_rows_8bit(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(x8, scale)``: rows ``[..., H]`` in e4m3 with one fp32 scale each, ``x = x8 * scale``:
    ``scale = max|x| / 448``.  For an output weight, once per set of weights."""
    if x.dtype not in _ROW_DTYPES:
        raise TypeError(f"8-bit rows are made of fp32, bf16 or fp16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"expected rows [..., H], got {tuple(x.shape)}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("8-bit rows have no gradient: call this under torch.no_grad()")
    return _C.quantize_rows(x)
