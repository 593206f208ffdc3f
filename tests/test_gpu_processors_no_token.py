"""Rows of processed logprobs without a next token: the result is the constant 0, so no gradient passes, whatever
comes from upstream.  Bounds as derived in test_gpu_processors.py."""

import pytest
import torch

from oracle import processors as oracle
from rl_amd.distributed.model_utils import from_parallel_logits_to_logprobs, processed_next_token_logprobs
from tests.test_gpu_processors import DTYPES, check_grad, check_logprobs, cuda, least_t, magnitude, make

pytestmark = pytest.mark.gpu


def compare(x, P, A, want, lp, t, xo, dtype, seed):
    g = torch.randn(want.shape, generator=torch.Generator().manual_seed(seed))
    assert bool((g != 0).all()) and bool((want == 0).any())
    T = least_t(P)
    check_logprobs(lp.detach(), want.detach(), A, T)
    (dx,) = torch.autograd.grad([lp], [t], [g.cuda()], retain_graph=True)
    (dxo,) = torch.autograd.grad([want], [xo], [g.double()])
    R = want.shape[1]
    assert not dx[:, R:].any()
    check_grad(dx[:, :R], dxo[:, :R], A, T, dtype, g, P.repetition_penalty.max().item() / T)
    assert not dx[:, :R].cpu()[want == 0].any()
    (summed,) = torch.autograd.grad([lp.sum()], [t])  # an expanded upstream gradient
    assert not summed[:, :R].cpu()[want == 0].any() and summed.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,R", [(515, 3), (5003, 1), (70001, 4)])
def test_behind_the_last_token_of_a_history(dtype, V, R):
    B, L = 5, 30
    x, ids, P, lengths = make(B, R, L, V, dtype, seed=V + R, K=3, behind=True)
    P.bias[:, 0] = 0.5
    lengths[:4] = torch.tensor([L, L - 1, 0, L + 7])  # no token at all, one, all, none
    t, xo = x.cuda().requires_grad_(True), x.double().requires_grad_(True)
    lp = processed_next_token_logprobs(t, ids.cuda(), cuda(P), history_lengths=lengths.cuda())
    compare(x, P, magnitude(x, P, L), oracle.logprobs(xo, ids, P, lengths), lp, t, xo, dtype, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,end", [(0, 700), (0, 600), (1000, 1700), (1000, 1650)])
def test_tokens_that_are_no_columns(dtype, start, end):
    B, S, V = 3, 40, 700
    x, ids, P, _ = make(B, S, S, V, dtype, seed=end, K=3)
    P.bias[:, 0] = 0.5
    ids, P.bias_ids = ids + start, P.bias_ids + start
    ids[0, 3], ids[0, 39], ids[1, 20:], ids[2, 1], ids[2, 2] = -1, -100, -1, 10**12, start + V  # padding, and worse
    t, xo = x.cuda().requires_grad_(True), x.double().requires_grad_(True)
    lp = from_parallel_logits_to_logprobs(t, ids.cuda(), start, end, None, logit_processors=cuda(P))
    want = oracle.logprobs(xo, ids, P, rows=S - 1, vocab_start=start, vocab_end=end)
    compare(x, P, magnitude(x, P, S), want, lp, t, xo, dtype, 2)
