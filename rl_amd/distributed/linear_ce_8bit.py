"""Token logprobs, and logits, from 8-bit hidden states and an 8-bit output weight.

The form of :func:`~rl_amd.distributed.linear_ce.from_parallel_hidden_states_to_logprobs` for
passes that score (the previous or the reference policy's logprobs) under 8-bit weights:
e4m3 or int8 rows with one fp32 scale each, on the MFMA units at twice the 16-bit rate, the fp32
logits never written.  :func:`from_int8_hidden_states_to_logits` writes them, for what a sampler does next
(:mod:`rl_amd.distributed.logit_processing`).  Sums of int8 products are exact.  The hidden states come from
:func:`~rl_amd.distributed.final_norm.add_rms_norm_8bit`, the weight from
:func:`~rl_amd.distributed.final_norm.quantize_rows_8bit`, once per set of weights.
"""

from __future__ import annotations

from typing import Any, Optional

import torch

from rl_amd import _C

__all__ = ["from_int8_hidden_states_to_logits", "from_parallel_8bit_hidden_states_to_logprobs"]

_MAX_INT8_HIDDEN = (1 << 17) - 256  # sums of products up to 2^14 stay inside 32 bits
_H_ALIGN = 256  # the kernel steps through the hidden dimension 256 elements at a time


def _operand8(x: torch.Tensor, whole: bool) -> torch.Tensor:
    """``x [N, H]`` in 8 bits as the kernel reads it: ``H`` and row strides multiples of 16, a 16-byte-aligned
    start, and with ``whole`` (the hidden states) ``H`` a multiple of 256; the weight also contiguous
    with rows of whole words; otherwise a zero-padded copy (the padding adds exact zeros)."""
    N, H = x.shape
    if not whole and H % 4 == 0 and x.is_contiguous() and x.data_ptr() % 4 == 0:
        return x
    if (H % (_H_ALIGN if whole else 16) == 0 and x.stride(-1) == 1 and x.stride(0) % 16 == 0 and x.stride(0) >= H
            and x.data_ptr() % 16 == 0):
        return x
    out = torch.empty((N, -(-H // _H_ALIGN) * _H_ALIGN), dtype=torch.uint8, device=x.device)
    out[:, :H].copy_(x.view(torch.uint8))
    out[:, H:].zero_()
    return out.view(x.dtype)


def _check_weight(h8: torch.Tensor, w8: torch.Tensor) -> int:
    """The vocabulary of a weight that matches the hidden states."""
    H = h8.shape[-1]
    if w8.dim() != 2 or w8.shape[1] != H or w8.shape[0] == 0:
        raise ValueError(f"weight shape {tuple(w8.shape)} does not match hidden size {H}")
    if h8.dtype == torch.int8 and H > _MAX_INT8_HIDDEN:
        raise ValueError(f"hidden size {H}: sums of more than {_MAX_INT8_HIDDEN} int8 products may pass 32 bits")
    return w8.shape[0]


def _no_gradient_to_scales(*scales: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in scales):
        raise RuntimeError("no gradient passes to the scales of int8 rows: detach them")
    _C.refuse_tangents(*scales)


def _check_scales(hidden_scales: torch.Tensor, shape: tuple, weight_scales: torch.Tensor, V: int) -> None:
    for name, scale, want in (("hidden", hidden_scales, shape), ("weight", weight_scales, (V,))):
        if scale.dtype != torch.float32 or tuple(scale.shape) != want:
            raise ValueError(f"{name} scales are float32 {want}, got {scale.dtype} {tuple(scale.shape)}")


def from_parallel_8bit_hidden_states_to_logprobs(
    hidden_states_8bit: torch.Tensor,
    hidden_scales: torch.Tensor,
    output_weight_8bit: torch.Tensor,
    output_weight_scales: torch.Tensor,
    target: torch.Tensor,
    vocab_start_index: int,
    vocab_end_index: int,
    tp_group: Optional[Any] = None,
    cp_group: Optional[Any] = None,
) -> torch.Tensor:
    """Next-token logprobs ``[B, S-1]`` (fp32) of ``hidden [S, B, H] . weight [V, H]^T``, both e4m3
    (``float8_e4m3fn``) or both ``int8``, with fp32 scales ``[S, B]`` and ``[V]``.

    ``target`` ``[B, S]`` is shifted by one position, as in the 16-bit form; the last position,
    which has no next token, is not computed.  Targets outside ``[vocab_start_index,
    vocab_end_index)`` give 0.  There is no gradient.  Hidden states whose size is not a
    multiple of 256, and a weight whose rows are neither 16-byte aligned nor whole words without
    gaps, are copied into padded buffers in every call."""
    from rl_amd.distributed.model_utils import _group_size, _require_single_rank

    _require_single_rank(tp_group)
    if _group_size(cp_group) != 1:
        raise NotImplementedError("context parallelism is not supported from hidden states")
    h8, w8 = hidden_states_8bit, output_weight_8bit
    if h8.dtype != w8.dtype or h8.dtype not in (torch.float8_e4m3fn, torch.int8):
        raise TypeError(f"expected float8_e4m3fn (or int8) hidden states and weight, got {h8.dtype} and {w8.dtype}")
    if h8.dim() != 3 or h8.shape[-1] == 0:
        raise ValueError(f"expected hidden states [S, B, H], got {tuple(h8.shape)}")
    S, B, H = h8.shape
    V = _check_weight(h8, w8)
    if tuple(target.shape) != (B, S):
        raise ValueError(f"target shape {tuple(target.shape)} does not match [B, S] = {(B, S)}")
    _check_scales(hidden_scales, (S, B), output_weight_scales, V)
    if h8.dtype == torch.int8:
        _no_gradient_to_scales(hidden_scales, output_weight_scales)
    R = max(S - 1, 0)
    out = torch.empty((B, R), dtype=torch.float32, device=h8.device)
    if R * B == 0:
        _C._require_gpu(h8, w8, target)
        return out
    if target.dtype != torch.int64:
        target = target.long()
    rows = _operand8(h8[:R].reshape(R * B, H), True)
    _C.linear_ce_8bit_fwd(rows, hidden_scales[:R].reshape(-1).contiguous(), _operand8(w8, False),
                          output_weight_scales.contiguous(), B, target[:, 1:], vocab_start_index,
                          vocab_end_index, out)
    return out


def from_int8_hidden_states_to_logits(
    hidden_states_8bit: torch.Tensor,
    hidden_scales: torch.Tensor,
    output_weight_8bit: torch.Tensor,
    output_weight_scales: torch.Tensor,
    dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Logits ``[..., V]`` of ``hidden [..., H] . weight [V, H]^T``, both ``int8`` with one fp32 scale per row
    (``[...]`` and ``[V]``): ``float(sum) * weight_scale * hidden_scale``, rounded once to ``dtype`` (fp32, bf16
    or fp16).  ``out`` takes them where it is given (contiguous, of ``dtype``).  There is no gradient (scales that ask
    for one are refused unless gradients are off); operands are copied where :func:`from_parallel_8bit_hidden_states_to_logprobs` copies them."""
    h8, w8 = hidden_states_8bit, output_weight_8bit
    _check_int8(h8, w8)
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits are fp32, bf16 or fp16, got {dtype}")
    V = _check_weight(h8, w8)
    lead, H = tuple(h8.shape[:-1]), h8.shape[-1]
    _check_scales(hidden_scales, lead, output_weight_scales, V)
    _no_gradient_to_scales(hidden_scales, output_weight_scales)
    if out is None:
        out = torch.empty((*lead, V), dtype=dtype, device=h8.device)
    elif out.dtype != dtype or tuple(out.shape) != (*lead, V) or not out.is_contiguous():
        raise ValueError(f"out is a contiguous {dtype} tensor {(*lead, V)}, got {out.dtype} {tuple(out.shape)}")
    elif out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("out asks for a gradient, which these logits have none of")
    if h8.numel() == 0:
        _C._require_gpu(h8, w8, out)
        return out
    operands = _int8_layout(h8, hidden_scales, w8, output_weight_scales)
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    _C.int8_logits(*operands, out.view(-1, V))
    return out


def _check_int8(h8: torch.Tensor, w8: torch.Tensor) -> None:
    if h8.dtype != torch.int8 or w8.dtype != torch.int8:
        raise TypeError(f"expected int8 hidden states and weight, got {h8.dtype} and {w8.dtype}")
    if h8.dim() < 1 or h8.shape[-1] == 0:
        raise ValueError(f"expected hidden states [..., H], got {tuple(h8.shape)}")


def int8_operands(h8: torch.Tensor, hidden_scales: torch.Tensor, w8: torch.Tensor, weight_scales: torch.Tensor
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Hidden rows ``[T, H]`` with their scales and the weight with its, checked and as ``_C.int8_logits`` reads them.  Any run of rows
    (and of their scales) is such an operand as well: a caller that takes them by blocks has them laid out once."""
    _check_int8(h8, w8)
    _check_scales(hidden_scales, tuple(h8.shape[:-1]), weight_scales, _check_weight(h8, w8))
    _no_gradient_to_scales(hidden_scales, weight_scales)
    return _int8_layout(h8, hidden_scales, w8, weight_scales)


def _int8_layout(h8: torch.Tensor, hidden_scales: torch.Tensor, w8: torch.Tensor, weight_scales: torch.Tensor
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return (_operand8(h8.reshape(-1, h8.shape[-1]), True), hidden_scales.reshape(-1).contiguous(), _operand8(w8, False),
            weight_scales.contiguous())
