"""The end of a policy in one call: residual stream -> final norm -> token logprobs.

``h = x + residual``, ``y = rms_norm(h) * norm_weight``, next-token logprobs of ``y`` under the output
weight: in the weight's type (differentiable, with or without adapters), or in 8 bits for passes
that only score.  What it calls: :mod:`~rl_amd.distributed.final_norm` and the hidden-state logprobs of
:mod:`~rl_amd.distributed.linear_ce`, :mod:`~rl_amd.distributed.linear_ce_adapters` and
:mod:`~rl_amd.distributed.linear_ce_8bit`.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Optional, Union

import torch

from rl_amd.distributed.final_norm import add_rms_norm, add_rms_norm_8bit, rms_norm
from rl_amd.distributed.linear_ce import from_parallel_hidden_states_to_logprobs
from rl_amd.distributed.linear_ce_8bit import from_parallel_8bit_hidden_states_to_logprobs
from rl_amd.distributed.linear_ce_adapters import from_parallel_hidden_states_to_logprobs_with_adapters

__all__ = ["HeadAdapters", "from_residual_stream_to_logprobs"]


@dataclass
class HeadAdapters:
    """Low-rank adapters beside the output weight (see
    :func:`~rl_amd.distributed.linear_ce_adapters.from_parallel_hidden_states_to_logprobs_with_adapters`):
    ``a [N, r, H]``, ``b [N, V, r]``, the batch's ``ids [B]`` (-1: the base model), one scaling or
    ``[N]`` of them, and the dropout of the adapters' input."""

    a: torch.Tensor
    b: torch.Tensor
    ids: torch.Tensor
    scaling: Union[float, torch.Tensor] = 1.0
    dropout_p: float = 0.0
    dropout_seed: Union[int, torch.Tensor] = 0
    dropout_offset: int = 0


def from_residual_stream_to_logprobs(
    x: torch.Tensor,
    residual: Optional[torch.Tensor],
    norm_weight: torch.Tensor,
    output_weight_layer: Union[torch.Tensor, tuple[torch.Tensor, torch.Tensor]],
    target: torch.Tensor,
    vocab_start_index: int,
    vocab_end_index: int,
    eps: float = 1e-6,
    adapters: Optional[HeadAdapters] = None,
    tp_group: Optional[Any] = None,
    inference_only: bool = False,
    cp_group: Optional[Any] = None,
    chunk_size: Optional[int] = None,
) -> torch.Tensor:
    """Next-token logprobs ``[B, S-1]`` (fp32) from the last layer's output ``x [S, B, H]`` and the
    residual stream (or None) under the final norm and the output weight.

    ``output_weight_layer`` is the weight ``[V, H]``, or the pair that
    :func:`~rl_amd.distributed.final_norm.quantize_rows_8bit` makes of it, with which the norm's rows
    are 8-bit as well; that form has no gradient and takes no adapters.  With ``inference_only`` no part
    keeps anything for a backward and the result has none.  The other arguments are those of the
    functions named above."""
    if inference_only and torch.is_grad_enabled():
        with torch.no_grad():
            return from_residual_stream_to_logprobs(
                x, residual, norm_weight, output_weight_layer, target, vocab_start_index, vocab_end_index, eps, adapters,
                tp_group, True, cp_group, chunk_size)
    if isinstance(output_weight_layer, (tuple, list)):
        if adapters is not None:
            raise NotImplementedError("adapters stand beside a 16-bit output weight")
        weight8, weight_scales = output_weight_layer
        y8, scales, _ = add_rms_norm_8bit(x, residual, norm_weight, eps)
        return from_parallel_8bit_hidden_states_to_logprobs(
            y8, scales, weight8, weight_scales, target, vocab_start_index, vocab_end_index, tp_group, cp_group)
    y = rms_norm(x, norm_weight, eps) if residual is None else add_rms_norm(x, residual, norm_weight, eps)[0]
    if adapters is not None:
        return from_parallel_hidden_states_to_logprobs_with_adapters(
            y, output_weight_layer, adapters.a, adapters.b, adapters.ids, adapters.scaling, target, vocab_start_index,
            vocab_end_index, tp_group, inference_only, cp_group, chunk_size, adapters.dropout_p, adapters.dropout_seed,
            adapters.dropout_offset)
    return from_parallel_hidden_states_to_logprobs(
        y, output_weight_layer, True, target, vocab_start_index, vocab_end_index, tp_group, inference_only, cp_group,
        chunk_size)
