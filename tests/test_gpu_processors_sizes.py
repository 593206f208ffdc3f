"""The logit processors at the sizes where they change form or could go wrong: many distinct tokens, wide
slices, long histories, the largest vocabulary, logits past 2^31 elements.  Bounds as derived in
test_gpu_processors.py."""

import dataclasses

import pytest
import torch

from oracle import processors as oracle
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors, apply_logit_processors
from rl_amd.distributed.model_utils import from_parallel_logits_to_logprobs, processed_next_token_logprobs
from tests.test_gpu_processors import check_grad, check_logprobs, check_values, cuda, least_t, magnitude, make, pack_masks

pytestmark = pytest.mark.gpu


def gradient(x, ids, P, g, **kw):
    t = x.cuda().requires_grad_(True)
    lp = from_parallel_logits_to_logprobs(t, ids.cuda(), 0, x.shape[2], None, logit_processors=cuda(P), **kw)
    (dx,) = torch.autograd.grad([lp], [t], [g.cuda()])
    return lp.detach(), dx


# more than 64 tokens with a word in 512 columns (and more than a wave lists as the rows go on), wide slices
# (16-bit rows past 4096 x 2048 columns), a last slice of any width
@pytest.mark.parametrize("dtype,B,S,V,K,M", [
    (torch.float32, 1, 300, 520, 0, 0), (torch.bfloat16, 2, 150, 1001, 9, 2), (torch.float16, 1, 200, 4099, 300, 0),
    (torch.bfloat16, 2, 71, 70001, 40, 0), (torch.float16, 2, 71, 65543, 40, 3), (torch.float16, 3, 50, 61440, 0, 2)])
def test_many_tokens_and_wide_slices(dtype, B, S, V, K, M):
    x, ids, P, _ = make(B, S, S, V, dtype, seed=S + V, K=K, M=M)
    h = torch.Generator().manual_seed(7)
    ids = torch.where(torch.rand(B, S, generator=h) < 0.5, torch.randint(0, min(V, 500), (B, S), generator=h), ids)
    g = torch.randn(B, S - 1, generator=torch.Generator().manual_seed(1))
    g[:, 5:40] = 0
    xo = x.double().requires_grad_(True)
    want = oracle.logprobs(xo, ids, P, rows=S - 1)
    g = torch.where(want.detach().isfinite(), g, torch.zeros_like(g))
    lp, dx = gradient(x, ids, P, g)
    A, T = magnitude(x, P, S), least_t(P)
    check_logprobs(lp, want.detach(), A, T)
    (dxo,) = torch.autograd.grad([torch.where(g != 0, want, torch.zeros_like(want)).mul(g.double()).sum()], [xo])
    check_grad(dx[:, :-1], dxo[:, :-1].nan_to_num(0.0), A, T, dtype, g, P.repetition_penalty.max().item() / T)
    check_values(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P)), oracle.process(x, ids, P), A, T, dtype)


def test_a_history_of_the_largest_length():
    L = (1 << 20) - 1
    ids = torch.randint(0, 3, (1, L), generator=torch.Generator().manual_seed(0))
    x = torch.randn(1, 1, 9, generator=torch.Generator().manual_seed(1))
    P = LogitProcessors(frequency_penalty=1e-6, presence_penalty=0.25, repetition_penalty=1.5, prompt_lengths=torch.tensor([1000]))
    lengths = torch.tensor([L])
    y = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P), history_lengths=lengths.cuda()).cpu()
    check_values(y, oracle.process(x, ids, P, lengths), magnitude(x, P, 1) + 1.1, 1.0, torch.float32)


@pytest.mark.parametrize("lengths", [[-5, 0, 7, 8, 9, 10**12]])
def test_lengths_out_of_range(lengths):
    B, L, R, V = len(lengths), 8, 2, 300
    x, ids, P, _ = make(B, R, L, V, torch.float32, seed=3)
    n = torch.tensor(lengths)
    clipped = n.clamp(-5, L)
    A, T = magnitude(x, P, L), least_t(P)
    check_values(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P), history_lengths=n.cuda()), oracle.process(x, ids, P, clipped), A, T, torch.float32)
    check_logprobs(processed_next_token_logprobs(x.cuda(), ids.cuda(), cuda(P), history_lengths=n.cuda()),
                   oracle.logprobs(x, ids, P, clipped), A, T)


def test_the_largest_vocabulary():
    V = 1 << 24
    x = torch.zeros(1, 1, V, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([[0, 5, V - 1, V - 1, 3]], device="cuda")
    P = LogitProcessors(presence_penalty=1.0, frequency_penalty=0.5, bias_ids=torch.tensor([V - 2], device="cuda"), bias=torch.tensor([2.0], device="cuda"))
    y = apply_logit_processors(x, ids, P, history_lengths=torch.tensor([4], device="cuda"))
    at = {0: -1.5, 5: -1.5, V - 1: -2.0, V - 2: 2.0}
    for j, v in at.items():
        assert y[0, 0, j].item() == v
        y[0, 0, j] = 0
    assert not y.any()
    lp = processed_next_token_logprobs(x, ids, P, history_lengths=torch.tensor([4], device="cuda"))
    assert abs(lp.item() + torch.tensor(V, dtype=torch.float64).log().item()) < 1e-5


def test_biases_of_the_largest_number():
    K, V = 2047, 5000
    x, ids, P, _ = make(2, 2, 2, V, torch.float32, seed=1)
    P.bias_ids = torch.randint(0, V, (2, K), generator=torch.Generator().manual_seed(4))
    P.bias = torch.randn(2, K, generator=torch.Generator().manual_seed(5))
    check_values(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P)), oracle.process(x, ids, P), magnitude(x, P, 2), least_t(P), torch.float32)


def test_logits_past_2_31_elements():
    B, S, V = 3, 5000, 151936
    x = torch.empty(B, S, V, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    ids = torch.randint(0, V, (B, S), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    P = LogitProcessors(repetition_penalty=1.2, frequency_penalty=0.1, temperature=0.9)
    lp = from_parallel_logits_to_logprobs(x, ids, 0, V, None, logit_processors=P)
    rows = [0, 31, 32, 2500, S - 2]
    for b in range(B):
        for r in rows:  # a row by itself, behind its history
            one = processed_next_token_logprobs(x[b:b + 1, r:r + 1], ids[b:b + 1], P, history_lengths=torch.tensor([r + 1], device="cuda"))
            assert abs(one.item() - lp[b, r].item()) <= 64 * 8 / 0.9 * 2**-24 + 2**-18
    t = x.requires_grad_(True)
    out = from_parallel_logits_to_logprobs(t, ids, 0, V, None, logit_processors=P)
    g = torch.zeros(B, S - 1, device="cuda")
    g[-1, -1] = 1.0
    (dx,) = torch.autograd.grad([out], [t], [g])
    row = x[-1:, S - 2:S - 1].detach().clone().requires_grad_(True)
    one = processed_next_token_logprobs(row, ids[-1:], P, history_lengths=torch.tensor([S - 1], device="cuda"))
    (d,) = torch.autograd.grad([one.sum()], [row])
    assert (dx[-1, S - 2].float() - d[0, 0].float()).abs().max() <= 2**-8 * d.abs().max()
    assert not dx[:-1].any() and not dx[-1, :S - 2].any() and not dx[-1, S - 1].any()


def test_expanded_and_scaled_upstream_gradients():
    x, ids, P, _ = make(2, 6, 6, 700, torch.float32, seed=4, K=2)
    P.bias[:, 0] = 0.5
    a = x.cuda().requires_grad_(True)
    from_parallel_logits_to_logprobs(a, ids.cuda(), 0, 700, None, logit_processors=cuda(P)).sum().backward()
    _, dx = gradient(x, ids, P, torch.ones(2, 5))
    assert torch.equal(a.grad, dx)
    b = x.cuda().requires_grad_(True)
    apply_logit_processors(b, ids.cuda(), cuda(P)).sum().backward()  # an expanded gradient
    c = x.cuda().requires_grad_(True)
    y = apply_logit_processors(c, ids.cuda(), cuda(P))
    (dc,) = torch.autograd.grad([y], [c], [torch.ones_like(y)])
    assert torch.equal(b.grad, dc)


def test_what_the_backward_reads_is_not_changed_between():
    for change in ("ids", "settings"):
        x, ids, P, _ = make(1, 4, 4, 60, torch.float32, seed=2, K=1)
        ids, P = ids.cuda(), cuda(P)
        t = x.cuda().requires_grad_(True)
        lp = from_parallel_logits_to_logprobs(t, ids, 0, 60, None, logit_processors=P)
        if change == "ids":
            ids[0, 1] += 1
        else:
            P.repetition_penalty.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            lp.sum().backward()


def test_graphs_do_not_share_what_they_write():
    """Two captured steps, replayed in turn, and the same settings for both."""
    a, ids, P, _ = make(3, 1, 30, 2500, torch.bfloat16, seed=8, K=3, M=2, behind=True)
    lengths = torch.tensor([30, 4, 0]).cuda()
    a, ids, P = a.cuda(), ids.cuda(), cuda(P)
    b = torch.randn_like(a)
    graphs, outs = [], []
    for x in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            processed_next_token_logprobs(x, ids, P, history_lengths=lengths)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((processed_next_token_logprobs(x, ids, P, history_lengths=lengths),
                         apply_logit_processors(x, ids, P, history_lengths=lengths)))
        graphs.append(graph)
    for k in range(4):
        lengths.copy_(torch.tensor([k, 5 * k + 2, 29 - k]))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, (lp, y) in zip((a, b), outs):
            want = apply_logit_processors(x, ids, P, history_lengths=lengths)
            assert torch.equal(y, want)
            assert torch.equal(lp, processed_next_token_logprobs(x, ids, P, history_lengths=lengths))


def test_no_masks_in_the_table():
    x, ids, P, _ = make(1, 3, 3, 100, torch.float32, seed=3)
    Q = dataclasses.replace(P, grammar_masks=torch.zeros(0, 4, dtype=torch.int32), grammar_rows=torch.zeros(1, 3, dtype=torch.int64))
    assert torch.equal(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P)), apply_logit_processors(x.cuda(), ids.cuda(), cuda(Q)))
    allowed = torch.ones(2, 100, dtype=torch.bool)
    wide = torch.cat([pack_masks(allowed), torch.zeros(2, 5, dtype=torch.int32)], 1)  # wider than the vocabulary
    W = dataclasses.replace(P, grammar_masks=wide, grammar_rows=torch.tensor([[0, 1, 7]]))  # 7: no such mask
    assert torch.equal(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P)), apply_logit_processors(x.cuda(), ids.cuda(), cuda(W)))


def test_one_mask_of_any_stride_and_inference_mode():
    x, ids, P, _ = make(2, 3, 3, 70, torch.float32, seed=6, K=2)
    mask = pack_masks(torch.rand(1, 70, generator=torch.Generator().manual_seed(3)) < 0.7)
    P = dataclasses.replace(P, grammar_masks=mask, grammar_rows=torch.zeros(2, 3, dtype=torch.int64))
    want = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P))
    odd = dataclasses.replace(cuda(P), grammar_masks=mask.cuda().as_strided((1, 3), (1, 1)))
    assert torch.equal(apply_logit_processors(x.cuda(), ids.cuda(), odd), want)
    with torch.inference_mode():
        place = x.cuda()
        apply_logit_processors(place, ids.cuda(), cuda(P), inplace=True)
        assert torch.equal(place, want)
        lp = from_parallel_logits_to_logprobs(x.cuda(), ids.cuda(), 0, 70, None, logit_processors=cuda(P))
    assert torch.equal(lp, from_parallel_logits_to_logprobs(x.cuda(), ids.cuda(), 0, 70, None, logit_processors=cuda(P)))


def test_saved_tensor_hooks_may_move_what_is_kept():
    x, ids, P, _ = make(2, 5, 5, 900, torch.float32, seed=7, K=3, M=3)
    g = torch.ones(2, 4)
    _, want = gradient(x, ids, P, g)
    with torch.autograd.graph.save_on_cpu():
        _, got = gradient(x, ids, P, g)
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# histories of several lists of tokens, rows that cross from one to the next, and one that ends with it
@pytest.mark.parametrize("dtype,V,R,K,M", [(torch.float32, 700, 3, 0, 0), (torch.bfloat16, 5003, 3, 9, 3), (torch.float16, 2049, 1, 300, 0),
                                           (torch.bfloat16, 141001, 30, 40, 0), (torch.float16, 141001, 30, 0, 3)])
def test_histories_of_several_lists(dtype, V, R, K, M):
    lengths = torch.tensor([8191, 12290] if V > 100000 else [0, 4095, 4096, 4097, 8190, 8193, 12290])
    B, L = len(lengths), 12291 + R
    x, ids, P, _ = make(B, R, L, V, dtype, seed=V + K, K=K, M=M)
    h = torch.Generator().manual_seed(8)
    some = torch.randint(0, V, (120,), generator=h)  # (the oracle takes one token at a time)
    ids = torch.where(torch.rand(B, L, generator=h) < 0.4, some[torch.randint(0, 120, (B, L), generator=h)], ids % 7 + V // 2)
    if K:
        P.bias_ids[:, K // 2:] = P.bias_ids[:, : K - K // 2]  # of two of one token the later holds
    P.prompt_lengths = (lengths - 4200).clamp(min=1)
    A, T = magnitude(x, P, L), least_t(P)
    want = oracle.process(x, ids, P, lengths)
    args = (ids.cuda(), cuda(P), lengths.cuda())
    check_values(apply_logit_processors(x.cuda(), *args), want, A, T, dtype)
    check_values(apply_logit_processors(x.cuda(), *args, inplace=True), want, A, T, dtype)
    t = x.cuda().requires_grad_(True)
    lp = processed_next_token_logprobs(t, *args)
    xo = x.double().requires_grad_(True)
    lpo = oracle.logprobs(xo, ids, P, lengths)
    check_logprobs(lp.detach(), lpo.detach(), A, T)
    g = torch.where(lpo.detach().isfinite(), torch.randn(B, R, generator=torch.Generator().manual_seed(2)), torch.zeros(()))
    (dx,) = torch.autograd.grad([lp], [t], [g.cuda()])
    (dxo,) = torch.autograd.grad([torch.where(g != 0, lpo, torch.zeros_like(lpo)).mul(g.double()).sum()], [xo])
    check_grad(dx, dxo.nan_to_num(0.0), A, T, dtype, g, P.repetition_penalty.max().item() / T)
    y = apply_logit_processors(t, *args)
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
    (da,) = torch.autograd.grad([y], [t], [dy.cuda()])
    yo = oracle.process(xo, ids, P, lengths)
    (dao,) = torch.autograd.grad([torch.where(yo.isfinite(), yo, torch.zeros_like(yo)).mul(dy.double()).sum()], [xo])
    # dy times two factors, three roundings in fp32 and one to the type
    fine = yo.detach().isfinite()
    half = torch.finfo(dtype).eps / 2
    assert bool(((da.double().cpu() - dao).abs() <= dao.abs() * (half + 2**-21) + torch.finfo(dtype).smallest_normal)[fine].all())
