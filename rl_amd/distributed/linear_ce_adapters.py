"""Token logprobs from hidden states with low-rank adapters of several requests beside the output weight.

:func:`~rl_amd.distributed.linear_ce.from_parallel_hidden_states_to_logprobs` for a policy whose
output weight carries adapters: sample ``b`` of the batch is under adapter ``adapter_ids[b]``, or
under the base model for an id outside ``[0, N)``, so that one batch holds several policies, or a
policy and its reference:

    d = dropout(h),  U = scaling[a] * (d . A_a^T),  x = h . W^T + U . B_a^T

* forward: the rows are sorted by adapter (on the device) and their ``U`` formed in fp32 by a
  kernel that gathers them; the tile loop takes ``U . B_a^T`` as a few more hidden elements of
  each 256 x 256 tile, and reduces the fp32 logits to logprobs without writing them.
* backward: over the rows with a non-zero upstream gradient, in blocks as the base path's; gradients of
  the hidden states and of the adapters, the output weight is frozen.  ``G = onehot - softmax`` is
  held in the operand type without the rows' gradients; every sum is fp32 and every result
  rounded once.

The hidden states, the weight and the adapters are bf16 or fp16 of one type.
"""

from __future__ import annotations

from typing import Any, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from rl_amd import _C
from rl_amd.distributed.linear_ce import (
    _BLOCK_CHUNKS,
    _H_ALIGN,
    _K_ALIGN,
    _block_rows,
    _dh_splits,
    _kernel_operand,
    _padded_width,
    _round_up,
    _weight_transposed,
)

__all__ = ["from_parallel_hidden_states_to_logprobs_with_adapters"]

_MAX_RANK = 1024
_DU_WAVES = 16384  # waves that dU's product is split into (half of them past the active rows)


def _padded_last(x: torch.Tensor) -> torch.Tensor:
    """``x [N, M, K]`` contiguous, 16-byte aligned and with K a multiple of 8 (zeros past K)."""
    if x.is_contiguous() and x.shape[2] % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    K = x.shape[2]
    out = torch.empty((*x.shape[:2], _round_up(K, 8)), dtype=x.dtype, device=x.device)
    out[:, :, :K].copy_(x)
    out[:, :, K:].zero_()
    return out


def _weight_operand(w: torch.Tensor) -> torch.Tensor:
    """``w [V, H]`` as the tile loop reads it against zero-padded hidden rows: ``H`` and the row stride
    multiples of 8 and a 16-byte-aligned start, or a padded copy."""
    H, ld = w.shape[1], w.stride(0)
    return w if H % 8 == 0 and ld % 8 == 0 and ld >= H and w.data_ptr() % 16 == 0 else _kernel_operand(w)


class _AdapterLogprobs(torch.autograd.Function):
    """``[B, R]`` logprobs of the first R positions of ``hidden [S, B, H]``."""

    @staticmethod
    def forward(ctx: Any, hidden, a, b, weight, ids, scaling, target, vs, ve, chunk_size, drop_args, keep):  # type: ignore[override]
        S, B, H = hidden.shape
        R = target.shape[1]
        dev = hidden.device
        h2 = hidden.view(S * B, H)
        drop = _C.Dropped(*drop_args, dev)
        bk = _padded_last(b)
        rows = _C.AdapterRows(ids, a.shape[0], target)
        h, planes, u = _C.adapter_down(h2, rows, _padded_last(a), bk, scaling, drop, _round_up(H, _H_ALIGN), keep)
        out = torch.empty((B, R), dtype=torch.float32, device=dev)
        stats = torch.empty((R * B, 2), dtype=torch.float32, device=dev) if keep else None
        _C.adapter_ce_fwd(h, _weight_operand(weight), rows, planes, bk, target, vs, ve, out, stats)
        if keep:
            p, seed, offset = drop_args
            seed_t = seed if isinstance(seed, torch.Tensor) else None
            ctx.save_for_backward(hidden, a, b, weight, ids, scaling, target, stats, u, rows.bad, seed_t)
            ctx.rest = (vs, ve, chunk_size, (p, None if seed_t is not None else seed, offset))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad):  # type: ignore[override]
        hidden, a, b, weight, ids, scaling, target, stats, u, bad, seed_t = ctx.saved_tensors
        vs, ve, chunk_size, (p, seed, offset) = ctx.rest
        need_h, need_a, need_b = ctx.needs_input_grad[:3]
        S, B, H = hidden.shape
        T = target.numel()
        N, r, _ = a.shape
        V = weight.shape[0]
        dev = hidden.device
        drop = _C.Dropped(p, seed if seed_t is None else seed_t, offset, dev)
        ak, bk, wk = _padded_last(a), _padded_last(b), _weight_operand(weight)
        rows = _C.AdapterRows(ids, N, target, grad, stats, bad)
        h2 = hidden.view(S * B, H)
        h, planes = _C.adapter_gather(h2, rows, u, _round_up(H, _H_ALIGN))
        Vp = _round_up(V, _K_ALIGN)
        n_rows = _block_rows(T, chunk_size, _BLOCK_CHUNKS * B, V)
        bT = torch.empty((N, bk.shape[2], Vp), dtype=b.dtype, device=dev)
        _C.transpose16(bk, V, bk.shape[2], bT)
        hT = None
        if need_a:
            hT = torch.empty((1, H, _padded_width(T)), dtype=hidden.dtype, device=dev)
            _C.transpose16(h.unsqueeze(0), T, H, hT, count=rows.count, perm=rows.perm, drop=drop)
        wT, wT_ready = _weight_transposed(weight.view(torch.bfloat16), Vp) if need_h else (None, None)
        dh = torch.zeros((S * B, H), dtype=hidden.dtype, device=dev) if need_h else None
        da = torch.zeros((N, r, H), dtype=torch.float32, device=dev) if need_a else None
        db = torch.zeros((N, V, r), dtype=torch.float32, device=dev) if need_b else None
        G = torch.empty((n_rows, Vp), dtype=hidden.dtype, device=dev)
        if Vp > V:
            G[:, V:].zero_()
        Gt = torch.empty((V, _padded_width(n_rows)), dtype=hidden.dtype, device=dev)
        for r0 in range(0, T, n_rows):
            n = min(n_rows, T - r0)
            Gc = G[:n]
            _C.adapter_ce_grad(h, wk, rows, planes, bk, vs, ve, r0, Gc, Gt)
            part = None
            if need_h:
                part = torch.empty((_dh_splits(n, H, Vp, count_known=False), n, H), dtype=torch.float32, device=dev)
                if wT_ready is not None:
                    torch.cuda.current_stream(dev).wait_event(wT_ready)
                    wT_ready = None
                if hidden.dtype == torch.float16:
                    _C.gemm_f16_abt(Gc, wT.view(torch.float16), Vp, part, count=rows.count, count_off=r0)
                else:
                    _C.gemm_bf16_abt(Gc, wT, Vp, part, k_splits=part.shape[0], count=rows.count, count_off=r0,
                                     count_axis=_C.COUNT_ROWS)
            splits = max(1, min(_DU_WAVES // (4 * -(-n // 128)), Vp // 1024))
            _C.adapter_block_grads(rows, r0, V, H, r, scaling, Gc, Gt, bT, ak, hT, u, drop, splits, part, dh, da, db)
            del part
        return (None if dh is None else dh.view(S, B, H), None if da is None else da.to(a.dtype),
                None if db is None else db.to(b.dtype)) + (None,) * 9


def from_parallel_hidden_states_to_logprobs_with_adapters(
    tensor_parallel_hidden_states: torch.Tensor,
    output_weight_layer: torch.Tensor,
    adapter_a: torch.Tensor,
    adapter_b: torch.Tensor,
    adapter_ids: torch.Tensor,
    adapter_scaling: Union[float, torch.Tensor],
    target: torch.Tensor,
    vocab_start_index: int,
    vocab_end_index: int,
    tp_group: Optional[Any] = None,
    inference_only: bool = False,
    cp_group: Optional[Any] = None,
    chunk_size: Optional[int] = None,
    dropout_p: float = 0.0,
    dropout_seed: Union[int, torch.Tensor] = 0,
    dropout_offset: int = 0,
) -> torch.Tensor:
    """Next-token logprobs ``[B, S-1]`` (fp32) of ``hidden [S, B, H]`` under ``weight [V, H]`` and, for
    sample b, adapter ``adapter_ids[b]`` of ``adapter_a [N, r, H]`` and ``adapter_b [N, V, r]``.

    ``adapter_ids`` (int64 ``[B]``): an id outside ``[0, N)``, such as -1, is the base model.
    ``adapter_scaling`` is one factor or a float32 tensor ``[N]``; no gradient reaches it.  With
    ``dropout_p`` the adapters' input is dropped as :func:`~rl_amd.distributed.counter_dropout.dropout`
    drops ``hidden`` under the same seed and offset.  Differentiable in the hidden states and the
    adapters; a weight that asks for a gradient is refused, the adapters stand on a frozen one.
    ``target [B, S]`` is shifted by one position, and targets outside ``[vocab_start_index,
    vocab_end_index)`` give 0; the last position is not computed.  ``inference_only`` keeps nothing for a
    backward.  ``chunk_size`` bounds the rows that the backward handles at a time, as in the
    base path, and never changes a row's logprob."""
    from rl_amd.distributed.model_utils import _group_size, _require_single_rank

    _require_single_rank(tp_group)
    if _group_size(cp_group) != 1:
        raise NotImplementedError("context parallelism is not supported from hidden states")
    hidden, weight, a, b = tensor_parallel_hidden_states, output_weight_layer, adapter_a, adapter_b
    if chunk_size is not None and int(chunk_size) <= 0:
        raise ValueError("chunk_size must be positive")
    if hidden.dim() != 3 or hidden.shape[-1] == 0:
        raise ValueError(f"expected hidden states [S, B, H], got {tuple(hidden.shape)}")
    S, B, H = hidden.shape
    if hidden.dtype not in (torch.bfloat16, torch.float16) or any(t.dtype != hidden.dtype for t in (weight, a, b)):
        raise TypeError("hidden states, weight and adapters are bfloat16 or float16 of one type, got "
                        f"{hidden.dtype}, {weight.dtype}, {a.dtype} and {b.dtype}")
    if weight.dim() != 2 or weight.shape[1] != H or weight.shape[0] == 0:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match hidden size {H}")
    V = weight.shape[0]
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] == 0 or a.shape[1] == 0 or a.shape[2] != H or tuple(b.shape) != (a.shape[0], V, a.shape[1]):
        raise ValueError(f"adapters [N, r, {H}] and [N, {V}, r] expected, got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.shape[1] > _MAX_RANK:
        raise ValueError(f"adapters of rank {a.shape[1]} are not supported (at most {_MAX_RANK})")
    if tuple(target.shape) != (B, S):
        raise ValueError(f"target shape {tuple(target.shape)} does not match [B, S] = {(B, S)}")
    if adapter_ids.dtype != torch.int64 or tuple(adapter_ids.shape) != (B,):
        raise ValueError(f"adapter ids are int64 [{B}], got {adapter_ids.dtype} {tuple(adapter_ids.shape)}")
    if not 0.0 <= dropout_p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {dropout_p}")
    keep = not inference_only and torch.is_grad_enabled() and any(t.requires_grad for t in (hidden, a, b, weight))
    if keep and weight.requires_grad:
        raise NotImplementedError("the output weight beside adapters is frozen: pass it without requires_grad")
    dev = _C._require_gpu(hidden, weight, a, b, adapter_ids, target)
    if isinstance(adapter_scaling, torch.Tensor):
        if adapter_scaling.dtype != torch.float32 or tuple(adapter_scaling.shape) != (a.shape[0],):
            raise ValueError(f"adapter scaling is a number or float32 [{a.shape[0]}], got {adapter_scaling.dtype} "
                             f"{tuple(adapter_scaling.shape)}")
        scaling = adapter_scaling.detach().contiguous()
    else:
        scaling = torch.full((a.shape[0],), float(adapter_scaling), dtype=torch.float32, device=dev)
    R = max(S - 1, 0)
    if R * B == 0:
        # no row: an empty result that the inputs' graph still reaches
        return (hidden[:R].sum(-1).t().float() + 0.0 * (a.sum() + b.sum()).float()) if keep else torch.empty(
            (B, R), dtype=torch.float32, device=dev)
    hidden = hidden.contiguous()
    if weight.stride(1) != 1:
        weight = weight.contiguous()
    target = target.long()[:, 1:]
    return _AdapterLogprobs.apply(
        hidden, a, b, weight, adapter_ids.contiguous(), scaling, target, int(vocab_start_index), int(vocab_end_index),
        None if chunk_size is None else int(chunk_size), (float(dropout_p), dropout_seed, int(dropout_offset)), keep)
