"""Logits and logprobs from 8-bit integers with a scale per token and per column, against 64 bits.

Bounds.  The integer sums are exact; a logit is that sum rounded to fp32 and two products, off by
3 x 2^-24 of itself, then rounded once to its type.  A logprob adds the rounding of exponents of
magnitude A and of its sums: 16 A 2^-24 + 2^-18 (A: the row's largest logit).
"""

import pytest
import torch

from oracle import processors as oracle
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors, TrainingSamplingParams, apply_logit_processors
from rl_amd.distributed.model_utils import (
    add_rms_norm_8bit,
    from_int8_hidden_states_to_logits,
    from_parallel_8bit_hidden_states_to_logprobs,
    from_parallel_logits_to_logprobs,
    from_residual_stream_to_logprobs,
    quantize_rows_8bit,
)

pytestmark = pytest.mark.gpu


def operands(N, H, V, seed=0, lead=None):
    g = torch.Generator().manual_seed(seed)
    h8 = torch.randint(-128, 128, (N, H), generator=g).to(torch.int8)
    w8 = torch.randint(-128, 128, (V, H), generator=g).to(torch.int8)
    hs = torch.rand(N, generator=g) * 0.02 / H**0.5
    ws = torch.rand(V, generator=g) * 0.02
    return h8, hs, w8, ws


def exact(h8, hs, w8, ws):
    return (h8.double() @ w8.double().t()) * ws.double() * hs.double()[:, None]


# rows below and above 128 (the two kernels), whole and ragged tiles, hidden sizes at stage borders
SHAPES = [(1, 1, 1), (1, 4, 3), (3, 16, 129), (64, 128, 128), (65, 200, 257), (128, 256, 1000), (129, 257, 255), (300, 1000, 515),
          (257, 512, 1031), (512, 4096, 300), (7, 4096, 2000)]


@pytest.mark.parametrize("N,H,V", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logits(N, H, V, dtype):
    h8, hs, w8, ws = operands(N, H, V, seed=N + H + V)
    got = from_int8_hidden_states_to_logits(h8.cuda(), hs.cuda(), w8.cuda(), ws.cuda(), dtype)
    assert got.dtype == dtype and got.shape == (N, V)
    want = exact(h8, hs, w8, ws)
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    bound = want.abs() * (3 * 2**-24 * (1 + half) + half) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((got.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("H", [(1 << 17) - 256, (1 << 17) - 257])
def test_sums_are_exact_up_to_the_largest_hidden_size(H):
    h8 = torch.full((2, H), -128, dtype=torch.int8)
    h8[1] = 127
    w8 = torch.full((3, H), -128, dtype=torch.int8)
    w8[1] = 127
    w8[2, ::2] = 127
    one = torch.ones(3)
    got = from_int8_hidden_states_to_logits(h8.cuda(), one[:2].cuda(), w8.cuda(), one.cuda(), torch.float32).cpu()
    assert torch.equal(got, (h8.long() @ w8.long().t()).float())


@pytest.mark.parametrize("S,B,H,V", [(2, 1, 4, 3), (2, 64, 256, 1031), (9, 5, 1000, 515), (130, 3, 300, 700), (65, 4, 512, 256), (1, 3, 64, 50)])
def test_logprobs(S, B, H, V):
    h8, hs, w8, ws = operands(S * B, H, V, seed=S + V)
    target = torch.randint(0, V, (B, S), generator=torch.Generator().manual_seed(1))
    got = from_parallel_8bit_hidden_states_to_logprobs(
        h8.view(S, B, H).cuda(), hs.view(S, B).cuda(), w8.cuda(), ws.cuda(), target.cuda(), 0, V).double().cpu()
    x = exact(h8, hs, w8, ws).view(S, B, V)[:-1]
    want = (x.gather(2, target[:, 1:].t()[..., None])[..., 0] - torch.logsumexp(x, -1)).t()
    assert got.shape == (B, max(S - 1, 0))
    if got.numel():
        assert (got - want).abs().max().item() <= 16 * x.abs().max().item() * 2**-24 + 2**-18
        part = from_parallel_8bit_hidden_states_to_logprobs(
            h8.view(S, B, H).cuda(), hs.view(S, B).cuda(), w8.cuda(), ws.cuda(), target.cuda(), 1, V - 1).cpu()
        outside = (target[:, 1:] < 1) | (target[:, 1:] >= V - 1)
        assert not part[outside].any()


def test_strided_and_unaligned_operands():
    h8, hs, w8, ws = operands(200, 96, 300, seed=5)
    want = from_int8_hidden_states_to_logits(h8.cuda(), hs.cuda(), w8.cuda(), ws.cuda(), torch.float32)
    wide_h = torch.full((200, 2, 130), 99, dtype=torch.int8, device="cuda")
    wide_w = torch.full((300, 131), 99, dtype=torch.int8, device="cuda")
    wide_h[:, 1, 7:103], wide_w[:, 3:99] = h8.cuda(), w8.cuda()
    assert torch.equal(from_int8_hidden_states_to_logits(wide_h[:, 1, 7:103], hs.cuda(), wide_w[:, 3:99], ws.cuda(), torch.float32), want)
    out = torch.zeros(200, 300, device="cuda")
    assert from_int8_hidden_states_to_logits(h8.cuda(), hs.cuda(), w8.cuda(), ws.cuda(), torch.float32, out) is out
    assert torch.equal(out, want)
    for off in (1, 3):  # 16-bit logits whose rows start at any even address
        h, s, w, v = operands(150, 64, 257 + off, seed=off)
        a = from_int8_hidden_states_to_logits(h.cuda(), s.cuda(), w.cuda(), v.cuda(), torch.float16)
        b = from_int8_hidden_states_to_logits(h.cuda(), s.cuda(), w.cuda(), v.cuda(), torch.float32)
        assert torch.equal(a, b.half())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,H", [(1, 1), (5, 7), (3, 1021), (2, 4096), (2, 20001)])
def test_rows(dtype, R, H):
    g = torch.Generator().manual_seed(R + H)
    x, res = (torch.randn(R, H, generator=g) * 3).to(dtype), torch.randn(R, H, generator=g).to(dtype)
    x[0] = 0
    x8, scale = quantize_rows_8bit(x.cuda(), torch.int8)
    assert x8.dtype == torch.int8 and scale.shape == (R,)
    amax = x.double().abs().amax(-1)
    want = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    assert bool(((scale.double().cpu() - want).abs() <= want * 2**-24).all())
    # x * (1 / s): the quotient off by 2^-23 of at most 127, then half a step
    assert bool(((x8.double().cpu() - x.double() / want[:, None]).abs() <= 0.5 + 127 * 2**-22).all())
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(dtype)
    y8, s, h = add_rms_norm_8bit(x.cuda(), res.cuda(), w.cuda(), 1e-6, torch.int8)
    e8, es, eh = add_rms_norm_8bit(x.cuda(), res.cuda(), w.cuda(), 1e-6)
    assert torch.equal(h, eh)
    hd = h.double().cpu()
    y = hd / (hd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    # y's largest magnitude is off by 2^-22 (its norm's sum over a lane's terms and a few products), the scale as well
    assert bool(((s.double().cpu() * 127 - y.abs().amax(-1)).abs() <= y.abs().amax(-1) * 2**-20).all())
    assert bool(((y8.double() * s.double()[:, None]).cpu() - y).abs().le(s.double().cpu()[:, None] * (0.5 + 127 * 2**-20)).all())
    assert (s * 127 - es * 448).abs().max() <= 448 * es.max() * 2**-22


def test_rows_with_a_nan_or_an_infinity_give_no_number():
    x = torch.randn(4, 64)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    x8, s = quantize_rows_8bit(x.cuda(), torch.int8)
    w8, ws = quantize_rows_8bit(torch.randn(40, 64).cuda(), torch.int8)
    logits = from_int8_hidden_states_to_logits(x8, s, w8, ws, torch.float32).cpu()
    assert logits[[0, 3]].isfinite().all() and not logits[[1, 2]].isfinite().any()


@pytest.mark.parametrize("S,B", [(2, 70), (9, 3)])
def test_the_run_of_the_sampler_s_head(S, B):
    """Residual stream -> norm in 8 bits -> int8 logits -> processors -> logprobs (whole and in blocks)."""
    H, V = 200, 1031
    g = torch.Generator().manual_seed(S)
    x, res = torch.randn(S, B, H, generator=g).bfloat16(), torch.randn(S, B, H, generator=g).bfloat16()
    norm, weight = (1 + 0.1 * torch.randn(H, generator=g)).bfloat16(), torch.randn(V, H, generator=g) * 0.1
    ids = torch.randint(0, 40, (B, S), generator=g)
    P = LogitProcessors(repetition_penalty=1.0 + torch.rand(B, generator=g), presence_penalty=0.3, frequency_penalty=0.2,
                        temperature=0.8, prompt_lengths=torch.randint(0, S, (B,), generator=g),
                        bias_ids=torch.randint(0, V, (B, 4), generator=g), bias=torch.randn(B, 4, generator=g),
                        grammar_masks=torch.randint(-2**31, 2**31, (3, 33), generator=g).to(torch.int32),
                        grammar_rows=torch.randint(-1, 3, (B, S - 1), generator=g))
    Pc = LogitProcessors(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in vars(P).items()})
    x, res, norm, ids_c = x.cuda(), res.cuda(), norm.cuda(), ids.cuda()
    pair = quantize_rows_8bit(weight.cuda(), torch.int8)
    y8, scale, _ = add_rms_norm_8bit(x, res, norm, dtype=torch.int8)
    logits = exact(y8.view(-1, H).cpu(), scale.view(-1).cpu(), pair[0].cpu(), pair[1].cpu()).view(S, B, V).transpose(0, 1)
    want = oracle.logprobs(logits, ids, P, rows=S - 1)
    A = 2 * logits.abs().max().item() + 10 + 0.2 * S
    for chunk in (None, 1, 4):
        with torch.no_grad():
            got = from_residual_stream_to_logprobs(x, res, norm, pair, ids_c, 0, V, chunk_size=chunk, logit_processors=Pc).double().cpu()
        assert torch.equal(got == -float("inf"), want == -float("inf"))
        fine = want.isfinite()
        assert (got - want)[fine].abs().max().item() <= 40 * A / 0.8 * 2**-24 + 2**-18
    # step by step, one new token of each request
    step = from_int8_hidden_states_to_logits(y8[-1], scale[-1], *pair, dtype=torch.float32)
    one = LogitProcessors(**{**vars(Pc), "grammar_masks": None, "grammar_rows": None})
    lengths = torch.full((B,), S, device="cuda")
    apply_logit_processors(step, ids_c, one, history_lengths=lengths, inplace=True)
    assert step.shape == (B, V) and step.isfinite().all()
    # without processors: the plain head in the same type, and the filter behind written-out logits
    with torch.no_grad():
        plain = from_residual_stream_to_logprobs(x, res, norm, pair, ids_c, 0, V)
    written = from_int8_hidden_states_to_logits(y8, scale, *pair, dtype=torch.float32).transpose(0, 1)
    assert (plain - from_parallel_logits_to_logprobs(written, ids_c, 0, V, None)).abs().max() <= 40 * A * 2**-24 + 2**-18
    kept = from_parallel_logits_to_logprobs(written, ids_c, 0, V, None, sampling_params=TrainingSamplingParams(top_k=5), logit_processors=one)
    assert kept.shape == (B, S - 1)


def test_a_captured_graph_replays():
    h8, hs, w8, ws = (t.cuda() for t in operands(70, 256, 900, seed=2))
    target = torch.randint(0, 900, (35, 2), device="cuda")

    def step():
        logits = from_int8_hidden_states_to_logits(h8, hs, w8, ws)
        return logits, from_parallel_8bit_hidden_states_to_logprobs(h8.view(2, 35, 256), hs.view(2, 35), w8, ws, target, 0, 900)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        h8.copy_(operands(70, 256, 900, seed=10 + k)[0].cuda())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)
