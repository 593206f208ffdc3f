"""Edges of the logit processors.  Bounds as derived in test_gpu_processors.py."""

import dataclasses

import pytest
import torch

from oracle import processors as oracle
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors, apply_logit_processors
from rl_amd.distributed.model_utils import from_parallel_logits_to_logprobs, processed_next_token_logprobs
from tests.test_gpu_processors import DTYPES, INF, check_logprobs, check_values, cuda, least_t, magnitude, make, pack_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [520, 70001])
def test_a_masked_token_s_bias_takes_no_part(dtype, V):
    """More biased tokens in 512 columns than a wave holds apart, half of them masked, with biases of infinity and NaN there."""
    B, S, K = 2, 40, 400
    x, ids, P, _ = make(B, S, S, V, dtype, seed=V)
    v = torch.arange(V)
    P.bias_ids = torch.arange(K)
    P.bias = torch.randn(K, generator=torch.Generator().manual_seed(1))
    P.grammar_masks, P.grammar_rows = pack_masks((v % 2 == 0)[None]), torch.zeros(B, S, dtype=torch.int64)
    Q = dataclasses.replace(P, bias=torch.where(v[:K] % 2 == 0, P.bias, torch.where(v[:K] % 4 == 1, INF, float("nan"))))
    outs = []
    for settings in (P, Q):
        t = x.cuda().requires_grad_(True)
        lp = from_parallel_logits_to_logprobs(t, ids.cuda(), 0, V, None, logit_processors=cuda(settings))
        g = torch.where(lp.detach().isfinite(), 1.0, 0.0)
        (dx,) = torch.autograd.grad([lp], [t], [g])
        outs.append((lp.detach(), dx, apply_logit_processors(t.detach(), ids.cuda(), cuda(settings))))
    check_logprobs(outs[0][0], oracle.logprobs(x, ids, P, rows=S - 1), magnitude(x, P, S), least_t(P))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_lengths_at_the_end_of_their_type():
    B, L, R, V = 4, 8, 3, 300
    x, ids, P, _ = make(B, R, L, V, torch.float32, seed=3)
    n = torch.tensor([2**63 - 1, 2**63 - 2, -(2**63), 5])
    A, T = magnitude(x, P, L), least_t(P)
    near = n.clamp(-5, L)  # (as far as a history reaches, the same)
    check_values(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P), history_lengths=n.cuda()), oracle.process(x, ids, P, near), A, T, torch.float32)
    check_logprobs(processed_next_token_logprobs(x.cuda(), ids.cuda(), cuda(P), history_lengths=n.cuda()), oracle.logprobs(x, ids, P, near), A, T)


@pytest.mark.parametrize("dtype,integer,signalling", [(torch.float32, torch.int32, 0x7F800001), (torch.bfloat16, torch.int16, 0x7F81),
                                                      (torch.float16, torch.int16, 0x7C01)])
def test_in_place_leaves_the_bits_of_what_does_not_change(dtype, integer, signalling):
    """Signalling NaN in groups of eight tokens of which none has a penalty or a bias: arithmetic makes quiet ones of them, as
    the written-out form does, and the call in place does not touch them."""
    B, V = 3, 5000
    ids = torch.randint(0, 700, (B, 40), generator=torch.Generator().manual_seed(2))
    lengths = torch.tensor([40, 13, 0])
    P = LogitProcessors(repetition_penalty=1.3, presence_penalty=0.5, bias_ids=torch.tensor([4999, 17, -1]), bias=torch.tensor([1.0, 2.0, 3.0]))
    quiet = torch.ones(B, V, dtype=torch.bool)
    for b in range(B):
        for j in [*ids[b, : lengths[b]].tolist(), 4999, 17]:
            quiet[b, j // 8 * 8: j // 8 * 8 + 8] = False
    assert bool(quiet.any(1).all())
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(3)).to(dtype)
    bits = x.view(integer).clone()
    bits[quiet] = signalling
    place = bits.cuda().view(dtype)
    out = apply_logit_processors(place, ids.cuda(), cuda(P), history_lengths=lengths.cuda())
    assert bool((out.view(integer).cpu()[quiet] != signalling).all())  # the forms can be told apart
    apply_logit_processors(place, ids.cuda(), cuda(P), history_lengths=lengths.cuda(), inplace=True)
    assert bool((place.view(integer).cpu()[quiet] == signalling).all())
    assert torch.equal(place.cpu()[~quiet], out.cpu()[~quiet])


@pytest.mark.parametrize("inplace", [False, True])
def test_quotients_are_rounded_once(inplace):
    """Temperature and repetition penalty divide: fp32 results are those of a division to the nearest, not of a product with the
    rounded reciprocal (off by an ulp in a third of them)."""
    B, V = 40, 3000
    g = torch.Generator().manual_seed(5)
    T, rp = 0.3 + 1.7 * torch.rand(B, generator=g), 1 + torch.rand(B, generator=g)
    x = torch.randn(B, V, generator=g) * 5
    x[:, 7], x[:, 8], x[:, 9] = INF, -INF, float("nan")
    ids = torch.arange(V).expand(B, V)
    none, all_ = torch.zeros(B, dtype=torch.int64), torch.full((B,), V)
    for P, lengths, want in ((LogitProcessors(temperature=T), none, x / T[:, None]),
                             (LogitProcessors(repetition_penalty=rp), all_, torch.where(x > 0, x / rp[:, None], x * rp[:, None]))):
        got = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P), history_lengths=lengths.cuda(), inplace=inplace).cpu()
        assert torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5)) and torch.equal(got.isnan(), want.isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inplace", [False, True])
def test_zeros_keep_their_signs(dtype, inplace):
    x = torch.zeros(2, 600)
    x[:, ::3] = -0.0
    P = LogitProcessors(repetition_penalty=1.3, temperature=0.7)
    ids, lengths = torch.arange(0, 600, 2).expand(2, 300), torch.tensor([300, 0])  # zeros of tokens that occurred, and not
    for settings in (P, LogitProcessors()):
        got = apply_logit_processors(x.to(dtype).cuda(), ids.cuda(), settings, history_lengths=lengths.cuda(), inplace=inplace).cpu()
        assert not got.any() and torch.equal(got.signbit(), x.signbit())
