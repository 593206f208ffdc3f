"""Token logprobs from 8-bit hidden states and an 8-bit output weight.

The form of :func:`~rl_amd.distributed.linear_ce.from_parallel_hidden_states_to_logprobs` for
passes that score (the previous or the reference policy's logprobs) under 8-bit weights:
e4m3 rows with one fp32 scale each, on the MFMA units at twice the 16-bit rate, the fp32
logits never written.  The hidden states come from
:func:`~rl_amd.distributed.final_norm.add_rms_norm_8bit`, the weight from
:func:`~rl_amd.distributed.final_norm.quantize_rows_8bit`, once per set of weights.
"""

from __future__ import annotations

from typing import Any, Optional

import torch

from rl_amd import _C

__all__ = ["from_parallel_8bit_hidden_states_to_logprobs"]

_H_ALIGN = 256  # the kernel steps through the hidden dimension 256 elements at a time


def _operand8(x: torch.Tensor, whole: bool) -> torch.Tensor:
    """``x [N, H]`` e4m3 as the kernel reads it: ``H`` and row strides multiples of 16, a 16-byte-aligned
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
    return out.view(torch.float8_e4m3fn)


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
    (``float8_e4m3fn``) with fp32 scales ``[S, B]`` and ``[V]``.

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
    if h8.dtype != torch.float8_e4m3fn or w8.dtype != torch.float8_e4m3fn:
        raise TypeError(f"expected float8_e4m3fn hidden states and weight, got {h8.dtype} and {w8.dtype}")
    if h8.dim() != 3 or h8.shape[-1] == 0:
        raise ValueError(f"expected hidden states [S, B, H], got {tuple(h8.shape)}")
    S, B, H = h8.shape
    if w8.dim() != 2 or w8.shape[1] != H or w8.shape[0] == 0:
        raise ValueError(f"weight shape {tuple(w8.shape)} does not match hidden size {H}")
    V = w8.shape[0]
    if tuple(target.shape) != (B, S):
        raise ValueError(f"target shape {tuple(target.shape)} does not match [B, S] = {(B, S)}")
    for name, scale, shape in (("hidden", hidden_scales, (S, B)), ("weight", output_weight_scales, (V,))):
        if scale.dtype != torch.float32 or tuple(scale.shape) != shape:
            raise ValueError(f"{name} scales are float32 {shape}, got {scale.dtype} {tuple(scale.shape)}")
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
