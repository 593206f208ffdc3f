"""What a sampler does to logits ahead of top-k and top-p, on the gfx950 kernels: penalties for
repeated tokens, biases of single tokens, grammar masks, and the temperature behind them.

:func:`process_logits` writes the processed logits out (differentiable, or in place), and
:func:`processed_next_token_logprobs` forms the next tokens' logprobs of processed logits that are
never written, with their gradient: what a sampler that had penalties or a grammar drew its
tokens from.  The settings are :class:`~rl_amd.algorithms.logits_sampling_utils.LogitProcessors`.

Row r of sample b follows the first ``n_b + r`` of its tokens: ``n_b`` is 1 for the rows of a
sequence itself (row r has read tokens 0 .. r) and the length of the history for rows behind one (a
single new token, or several drafted ones).  With ``c`` a token's count among those at or behind
``prompt_lengths[b]``, ``seen`` if it occurs at all (in the prompt as well), its logit x becomes

    z = x + bias;  z = z / repetition if z > 0 else z * repetition, where seen
    z = z - frequency * c - presence * [c > 0]
    y = z / temperature where the row's grammar allows the token, -inf elsewhere

in fp32, rounded once where it is written.  A masked logit may hold anything, and so may its bias.
"""

from __future__ import annotations

import math
from typing import Any, Optional

import torch
from torch.autograd.function import once_differentiable

from rl_amd import _C

__all__ = ["process_logits", "processed_next_token_logprobs"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MAX_TOKENS, _MAX_BIAS, _MAX_VOCAB = (1 << 20) - 1, 2047, 1 << 24  # what the kernels' words and tables hold
# the settings with one value per sample, in the kernels' order: field, least value (excluded)
_PER_SAMPLE = (("repetition_penalty", 0.0), ("presence_penalty", None), ("frequency_penalty", None), ("temperature", 0.0))


def _int64(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype == torch.int64:
        return t
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{name} holds whole numbers, got {t.dtype}")
    return t.long()


def _per_sample(t: Any, name: str, B: int) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (B,):
        raise ValueError(f"{name} is a tensor [{B}], got {tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__}")
    t = _int64(t, name)
    return t if t.is_contiguous() else t.contiguous()


def _f32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _no_grad(t: torch.Tensor, name: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"no gradient passes to {name}: detach it")


class _Call:
    """The checked settings of one call: the tensors that the kernels read, in their order, and the numbers."""

    __slots__ = ("ids", "tensors", "scalars", "vocab")

    def __init__(self, logits: torch.Tensor, input_ids: torch.Tensor, P: Any, history_lengths: Optional[torch.Tensor],
                 R: int, vocab: tuple[int, int]):
        dev, (B, _, V) = logits.device, logits.shape
        if logits.dtype not in _DTYPES:
            raise TypeError(f"logit processors take fp32, bf16 or fp16 logits, got {logits.dtype}")
        if not 0 < V <= _MAX_VOCAB:
            raise ValueError(f"a vocabulary of {V} tokens: 1 to {_MAX_VOCAB} are taken")
        if input_ids.dim() != 2 or input_ids.shape[0] != B:
            raise ValueError(f"expected input_ids [B, L] of {B} samples, got {tuple(input_ids.shape)}")
        self.ids = ids = _int64(input_ids, "input_ids")
        L = ids.shape[1]
        if L > _MAX_TOKENS:
            raise ValueError(f"{L} tokens of a sample: at most {_MAX_TOKENS} are counted")
        lengths = prompts = bias_ids = bias = masks = rows = None
        if history_lengths is not None:
            lengths = _per_sample(history_lengths, "history_lengths", B)
        elif L < R:
            raise ValueError(f"{R} rows of logits for {L} tokens: give history_lengths for rows behind a history")
        if P.prompt_lengths is not None:
            prompts = _per_sample(P.prompt_lengths, "prompt_lengths", B)
        penalties, scalars = [], []
        for field, least in _PER_SAMPLE:
            value = getattr(P, field)
            if isinstance(value, torch.Tensor):
                _no_grad(value, field)
                if tuple(value.shape) != (B,) or not value.dtype.is_floating_point:
                    raise ValueError(f"{field} is a number or a floating tensor [{B}], got {value.dtype} {tuple(value.shape)}")
                penalties.append(_f32(value))
                scalars.append(1.0)
            else:
                value = float(value)
                if not math.isfinite(value) or (least is not None and value <= least):
                    raise ValueError(f"{field} must be finite{'' if least is None else ' and positive'}, got {value}")
                penalties.append(None)
                scalars.append(value)
        if (P.bias_ids is None) != (P.bias is None):
            raise ValueError("bias_ids and bias come together")
        if P.bias is not None:
            _no_grad(P.bias, "bias")
            shape = tuple(P.bias.shape)
            if tuple(P.bias_ids.shape) != shape or len(shape) not in (1, 2) or (len(shape) == 2 and shape[0] != B):
                raise ValueError(f"bias_ids and bias are [K] or [{B}, K], got {tuple(P.bias_ids.shape)} and {shape}")
            if not P.bias.dtype.is_floating_point:
                raise TypeError(f"bias is floating, got {P.bias.dtype}")
            if shape[-1] > _MAX_BIAS:
                raise ValueError(f"{shape[-1]} biases of a sample: at most {_MAX_BIAS} are held (a grammar mask rules out any number)")
            if shape[-1]:
                bias_ids, bias = _int64(P.bias_ids, "bias_ids").contiguous(), _f32(P.bias)
        if (P.grammar_masks is None) != (P.grammar_rows is None):
            raise ValueError("grammar_masks and grammar_rows come together")
        if P.grammar_masks is not None:
            masks, rows = P.grammar_masks, _int64(P.grammar_rows, "grammar_rows")
            if masks.dtype != torch.int32 or masks.dim() != 2 or masks.shape[1] < -(-V // 32):
                raise ValueError(f"grammar_masks are int32 [M, W] with W >= {-(-V // 32)} words for {V} tokens, got {masks.dtype} {tuple(masks.shape)}")
            if rows.dim() != 2 or rows.shape[0] != B or rows.shape[1] < R:
                raise ValueError(f"grammar_rows name the masks of {B} x {R} rows, got {tuple(rows.shape)}")
            if not masks.shape[0]:
                masks = rows = None
            elif masks.stride(1) != 1 or (masks.stride(0) < masks.shape[1] and masks.shape[0] > 1):
                masks = masks.contiguous()
        self.tensors = (lengths, prompts, *penalties, bias_ids, bias, masks, rows)
        self.scalars, self.vocab = tuple(scalars), vocab
        _C.refuse_tangents(logits, *self.tensors)
        for t in (logits, ids, *self.tensors):
            if t is not None and (not t.is_cuda or t.device != dev):
                _C._require_gpu(logits, ids, *self.tensors)

    def args(self) -> "_C.LogitProcessorArgs":
        return _C.processor_args(self.ids, self.tensors, self.scalars, self.vocab)


class _ProcessedLogprob(torch.autograd.Function):
    """Logprobs [B, R] of the tokens behind the first R rows.  Kept for the backward: the logits, eight
    bytes a row, what the call was given."""

    @staticmethod
    def forward(ctx: Any, logits: torch.Tensor, R: int, call: _Call) -> torch.Tensor:  # type: ignore[override]
        out, stats, table = _C.processed_logprob_fwd(logits, R, call.args(), True)
        ctx.save_for_backward(logits, stats, table, call.ids, *call.tensors)
        ctx.numbers = (call.scalars, call.vocab)
        return out

    @staticmethod
    def backward(ctx: Any, grad: torch.Tensor):  # type: ignore[override]
        # the decorator only where a graph of the backward is asked for: it costs a small call 4 us
        return (_ProcessedLogprob._once if torch.is_grad_enabled() else _ProcessedLogprob._grads)(ctx, grad)

    @staticmethod
    def _grads(ctx: Any, grad: torch.Tensor):
        logits, stats, table, ids, *tensors = ctx.saved_tensors
        args = _C.processor_args(ids, tuple(tensors), *ctx.numbers)
        return _C.processed_logprob_bwd(logits, args, table, stats, grad.float()), None, None

    _once = staticmethod(once_differentiable(_grads.__func__))


class _ProcessLogits(torch.autograd.Function):
    """Processed logits as a new tensor.  The backward reads the logits of the tokens that occur."""

    @staticmethod
    def forward(ctx: Any, logits: torch.Tensor, call: _Call) -> torch.Tensor:  # type: ignore[override]
        out, table = _C.process_logits(logits, call.args(), False)
        ctx.save_for_backward(logits, table, call.ids, *call.tensors)
        ctx.numbers = (call.scalars, call.vocab)
        return out

    @staticmethod
    def backward(ctx: Any, grad: torch.Tensor):  # type: ignore[override]
        return (_ProcessLogits._once if torch.is_grad_enabled() else _ProcessLogits._grads)(ctx, grad)

    @staticmethod
    def _grads(ctx: Any, grad: torch.Tensor):
        logits, table, ids, *tensors = ctx.saved_tensors
        return _C.process_logits_bwd(logits, _C.processor_args(ids, tuple(tensors), *ctx.numbers), table, grad), None

    _once = staticmethod(once_differentiable(_grads.__func__))


class _ProcessLogitsF32(torch.autograd.Function):
    """(processed logits in fp32, whether anything is left in a row)."""

    @staticmethod
    def forward(ctx: Any, logits: torch.Tensor, call: _Call):  # type: ignore[override]
        out, left, table = _C.process_logits_f32(logits, call.args())
        ctx.save_for_backward(logits, table, call.ids, *call.tensors)
        ctx.numbers = (call.scalars, call.vocab)
        ctx.mark_non_differentiable(left)
        ctx.set_materialize_grads(False)
        return out, left

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: Optional[torch.Tensor], _: Any):  # type: ignore[override]
        if grad is None:
            return None, None
        logits, table, ids, *tensors = ctx.saved_tensors
        return _C.process_logits_bwd(logits, _C.processor_args(ids, tuple(tensors), *ctx.numbers), table, grad, True), None


def _rows_meet(x: torch.Tensor) -> bool:
    """Whether two rows of ``x [B, R, V]`` (unit stride in V) have an element in common."""
    (n, s), (m, t) = sorted(zip(x.shape[:2], x.stride()[:2]), key=lambda d: d[1])  # the lesser stride first
    V = x.shape[2]
    if (n > 1 and s < V) or (m > 1 and t < V):
        return True
    if n <= 1 or m <= 1 or t >= (n - 1) * s + V:
        return False
    # rows that are i of the one stride and j of the other apart
    return any(abs(i * t - j * s) < V for i in range(1, m) for j in (i * t // s, i * t // s + 1) if j < n)


def _grad_needed(logits: torch.Tensor) -> bool:
    return logits.requires_grad and torch.is_grad_enabled()


def processed_next_token_logprobs(
    logits: torch.Tensor,
    input_ids: torch.Tensor,
    processors: Any,
    history_lengths: Optional[torch.Tensor] = None,
    inference_only: bool = False,
    vocab_start_index: int = 0,
    vocab_end_index: Optional[int] = None,
) -> torch.Tensor:
    """fp32 logprobs ``[B, R]`` of the token behind each row of ``logits [B, R, V]`` under ``processors``.

    Without ``history_lengths`` the rows are those of the sequence: row r is scored against
    ``input_ids[:, r + 1]``, and there are ``min(R, L - 1)`` results.  With ``history_lengths [B]`` row r
    follows the first ``history_lengths[b] + r`` tokens and is scored against the token behind them; a
    row whose token ``input_ids`` does not hold gives 0, as does a token outside ``[vocab_start_index,
    vocab_end_index)``: a constant, without a gradient (the logprobs of unprocessed logits, whose ranges may be the
    parts of a sharded vocabulary, leave the probabilities' gradient there).  A token that its row does not
    allow gives -inf, and a row that allows nothing has no gradient."""
    if logits.dim() != 3:
        raise ValueError(f"expected logits of shape [B, R, V], got {tuple(logits.shape)}")
    R = logits.shape[1]
    if history_lengths is None and input_ids.dim() == 2:
        R = min(R, max(input_ids.shape[1] - 1, 0))
    if logits.stride(-1) != 1:
        logits = logits.contiguous()
    end = vocab_start_index + logits.shape[2] if vocab_end_index is None else vocab_end_index
    call = _Call(logits, input_ids, processors, history_lengths, R, (int(vocab_start_index), int(end)))
    if inference_only or not _grad_needed(logits):
        return _C.processed_logprob_fwd(logits, R, call.args(), False)[0]
    return _ProcessedLogprob.apply(logits, R, call)


def filtered_processed_logprobs(
    logits: torch.Tensor,
    target: torch.Tensor,
    processors: Any,
    top_k: Optional[int],
    top_p: Optional[float],
    inference_only: bool,
    vocab_start_index: int,
    vocab_end_index: Optional[int],
) -> torch.Tensor:
    """fp32 logprobs ``[B, S - 1]`` of the next tokens of ``target [B, S]`` under the processors and the filter behind
    them, from ``logits [B, >= S, V]``.  Ids count from ``vocab_start_index``, for the processors and for the next tokens; one
    that is no column is not among those kept: -inf.

    The processed logits are written once, in fp32 whatever the type of the logits: what is held in 16 bits between the two would
    be off by half a step there (2^-4 at 16), and the cut would be decided on that.  Top-p is therefore
    decided in fp32, as a sampler decides it.  A row in which nothing is left gives -inf and has no gradient."""
    from rl_amd.distributed.sampling import filtered_row_logprobs

    x = logits[:, : max(target.shape[1] - 1, 0)]
    start = int(vocab_start_index)
    end = start + x.shape[2] if vocab_end_index is None else int(vocab_end_index)
    call = _Call(x, target, processors, None, x.shape[1], (start, end))
    if inference_only or not _grad_needed(logits):
        y, left, _ = _C.process_logits_f32(x, call.args())
    else:
        y, left = _ProcessLogitsF32.apply(x, call)
    tokens = call.ids[:, 1:]
    if start != 0 or end < x.shape[2]:
        tokens = torch.where((tokens >= start) & (tokens < end), tokens - start, -1)
    logprobs = filtered_row_logprobs(y, tokens, top_k, top_p, inference_only=inference_only)
    return logprobs.masked_fill(left == 0, -math.inf)


def process_logits(
    logits: torch.Tensor,
    input_ids: torch.Tensor,
    processors: Any,
    history_lengths: Optional[torch.Tensor] = None,
    inplace: bool = False,
) -> torch.Tensor:
    """``apply_logit_processors`` of :mod:`rl_amd.algorithms.logits_sampling_utils`."""
    if logits.dim() not in (2, 3):
        raise ValueError(f"expected logits of shape [B, V] or [B, R, V], got {tuple(logits.shape)}")
    if logits.dim() == 2 and history_lengths is None:
        raise ValueError("logits [B, V] are one row behind each history: give history_lengths")
    x = logits if logits.dim() == 3 else logits.unsqueeze(1)
    if inplace:
        if _grad_needed(logits):
            raise RuntimeError("in place there is no gradient: the backward needs the logits as they were")
        if x.stride(2) != 1 and x.shape[2] > 1:
            raise ValueError("in place, the vocabulary has unit stride")
        if _rows_meet(x):
            raise ValueError("in place, no two rows share memory")
    elif x.stride(2) != 1:
        x = x.contiguous()
    call = _Call(x, input_ids, processors, history_lengths, x.shape[1], (0, x.shape[2]))
    if not inplace and _grad_needed(logits):
        y = _ProcessLogits.apply(x, call)
        return y if logits.dim() == 3 else y.squeeze(1)
    y, _ = _C.process_logits(x, call.args(), inplace)
    if inplace:
        if not logits.is_inference():
            torch.autograd.graph.increment_version(logits)
        return logits
    return y if logits.dim() == 3 else y.squeeze(1)
