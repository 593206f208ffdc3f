"""The end of a policy in one call: residual stream -> final norm -> token logprobs.

``h = x + residual``, ``y = rms_norm(h) * norm_weight``, next-token logprobs of ``y`` under the output
weight: in the weight's type (differentiable, with or without adapters), or in 8 bits for passes
that only score; with 8-bit integers also under a sampler's penalties, biases and grammar masks.  What
it calls: :mod:`~rl_amd.distributed.final_norm`, the hidden-state logprobs of
:mod:`~rl_amd.distributed.linear_ce`, :mod:`~rl_amd.distributed.linear_ce_adapters` and
:mod:`~rl_amd.distributed.linear_ce_8bit`, and :mod:`~rl_amd.distributed.logit_processing`.
"""

from __future__ import annotations

from dataclasses import dataclass, replace
from typing import Any, Optional, Union

import torch

from rl_amd import _C
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors
from rl_amd.distributed.final_norm import add_rms_norm, add_rms_norm_8bit, rms_norm
from rl_amd.distributed.linear_ce import from_parallel_hidden_states_to_logprobs
from rl_amd.distributed.linear_ce_8bit import from_parallel_8bit_hidden_states_to_logprobs, int8_operands
from rl_amd.distributed.linear_ce_adapters import from_parallel_hidden_states_to_logprobs_with_adapters
from rl_amd.distributed.logit_processing import processed_next_token_logprobs
from rl_amd.distributed.model_utils import _check_chunk_size, _require_single_rank

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
    logit_processors: Optional[LogitProcessors] = None,
) -> torch.Tensor:
    """Next-token logprobs ``[B, S-1]`` (fp32) from the last layer's output ``x [S, B, H]`` and the
    residual stream (or None) under the final norm and the output weight.

    ``output_weight_layer`` is the weight ``[V, H]``, or the pair that
    :func:`~rl_amd.distributed.final_norm.quantize_rows_8bit` makes of it, with which the norm's rows
    are 8-bit of the same type; that form has no gradient and takes no adapters.  ``logit_processors`` (with
    an ``int8`` pair only) are those of the sampler that drew ``target``: blocks of ``chunk_size`` positions (by
    default of about 1 GiB) are written as fp32 logits and scored under them.  With ``inference_only`` no part
    keeps anything for a backward and the result has none.  The other arguments are those of the
    functions named above."""
    if inference_only and torch.is_grad_enabled():
        with torch.no_grad():
            return from_residual_stream_to_logprobs(
                x, residual, norm_weight, output_weight_layer, target, vocab_start_index, vocab_end_index, eps, adapters,
                tp_group, True, cp_group, chunk_size, logit_processors)
    if isinstance(output_weight_layer, (tuple, list)):
        if adapters is not None:
            raise NotImplementedError("adapters stand beside a 16-bit output weight")
        weight8, weight_scales = output_weight_layer
        if logit_processors is not None and weight8.dtype != torch.int8:
            raise NotImplementedError("logit processors take an int8 output weight")
        y8, scales, _ = add_rms_norm_8bit(x, residual, norm_weight, eps, weight8.dtype)
        if logit_processors is not None:
            _require_single_rank(tp_group, cp_group)
            return _processed_int8(y8, scales, weight8, weight_scales, target, vocab_start_index, vocab_end_index,
                                   chunk_size, logit_processors)
        return from_parallel_8bit_hidden_states_to_logprobs(
            y8, scales, weight8, weight_scales, target, vocab_start_index, vocab_end_index, tp_group, cp_group)
    if logit_processors is not None:
        raise NotImplementedError("logit processors take an int8 output weight")
    y = rms_norm(x, norm_weight, eps) if residual is None else add_rms_norm(x, residual, norm_weight, eps)[0]
    if adapters is not None:
        return from_parallel_hidden_states_to_logprobs_with_adapters(
            y, output_weight_layer, adapters.a, adapters.b, adapters.ids, adapters.scaling, target, vocab_start_index,
            vocab_end_index, tp_group, inference_only, cp_group, chunk_size, adapters.dropout_p, adapters.dropout_seed,
            adapters.dropout_offset)
    return from_parallel_hidden_states_to_logprobs(
        y, output_weight_layer, True, target, vocab_start_index, vocab_end_index, tp_group, inference_only, cp_group,
        chunk_size)


_CHUNK_BYTES = 1 << 30


def _processed_int8(y8, scales, weight8, weight_scales, target, vocab_start, vocab_end, chunk_size, processors):
    """The logprobs of int8 rows ``[S, B, H]`` under a sampler's processors, block by block of positions."""
    if y8.dim() != 3:
        raise ValueError(f"expected hidden states [S, B, H], got {tuple(y8.shape)}")
    _check_chunk_size(chunk_size)
    S, B, _ = y8.shape
    if tuple(target.shape) != (B, S):
        raise ValueError(f"target shape {tuple(target.shape)} does not match [B, S] = {(B, S)}")
    V, R = weight8.shape[0], max(S - 1, 0)
    out = torch.empty((B, R), dtype=torch.float32, device=y8.device)
    if R * B == 0:
        return out
    rows, row_scales, weight, col_scales = int8_operands(y8, scales, weight8, weight_scales)
    step, logits = chunk_size or max(1, _CHUNK_BYTES // (4 * B * V)), None
    for s0 in range(0, R, step):
        s1 = min(s0 + step, R)
        if logits is None or logits.shape[0] != s1 - s0:
            logits = torch.empty((s1 - s0, B, V), dtype=torch.float32, device=y8.device)
        _C.int8_logits(rows[s0 * B:s1 * B], row_scales[s0 * B:s1 * B], weight, col_scales, logits.view(-1, V))
        block = processors
        if processors.grammar_rows is not None:
            block = replace(processors, grammar_rows=processors.grammar_rows[:, s0:s1])
        lengths = torch.full((B,), s0 + 1, dtype=torch.int64, device=y8.device)
        out[:, s0:s1] = processed_next_token_logprobs(logits.transpose(0, 1), target, block, lengths, True, vocab_start, vocab_end)
    return out
