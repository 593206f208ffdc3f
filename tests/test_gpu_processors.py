"""Penalties, biases, grammar masks and temperature on logits against the 64-bit oracle.

Bounds.  A processed logit is formed in at most 8 fp32 operations on values of magnitude at most A (the
largest logit, bias and penalty of the row together), each off by 2^-24 A, and divided by T: off by
8 A / T 2^-24.  A logprob subtracts two such (the target's and the log of the sum, whose exponents are
as far off, each also rounded once or twice more in base 2) and sums at most a few hundred terms a lane in order:
32 A / T 2^-24 + 2^-18.  Results in 16 bits are rounded once more.
"""

import dataclasses

import pytest
import torch

from oracle import processors as oracle
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors, TrainingSamplingParams, apply_logit_processors
from rl_amd.distributed.model_utils import from_parallel_logits_to_logprobs, processed_next_token_logprobs

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def pack_masks(allowed: torch.Tensor) -> torch.Tensor:
    """bool [M, V] -> int32 [M, ceil(V / 32)], token v bit v % 32 of word v // 32."""
    M, V = allowed.shape
    bits = torch.zeros(M, -(-V // 32) * 32, dtype=torch.int64)
    bits[:, :V] = allowed.long()
    words = (bits.view(M, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)


def make(B, R, L, V, dtype, seed=0, K=0, M=0, behind=False, tensors=True, T=True):
    """(logits, ids, settings, lengths) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, R, V, generator=g) * 3).to(dtype)
    ids = torch.where(torch.rand(B, L, generator=g) < 0.6, torch.randint(0, min(V, 7), (B, L), generator=g),
                      torch.randint(0, V, (B, L), generator=g))
    lengths = torch.randint(0, max(1, L - R + 1), (B,), generator=g) if behind else None
    prompts = torch.randint(0, L + 1, (B,), generator=g)
    P = LogitProcessors(
        repetition_penalty=1.0 + torch.rand(B, generator=g) if tensors else 1.25,
        presence_penalty=torch.randn(B, generator=g) if tensors else 0.5,
        frequency_penalty=torch.rand(B, generator=g) * 0.5 if tensors else -0.25,
        temperature=(0.5 + torch.rand(B, generator=g) if tensors else 0.7) if T else 1.0,
        prompt_lengths=prompts)
    if K:
        P.bias_ids = torch.randint(-1, V, (B, K), generator=g)
        P.bias = torch.randn(B, K, generator=g) * 4
        P.bias[:, 0] = -INF
    if M:
        allowed = torch.rand(M, V, generator=g) < torch.tensor([0.05, 0.5, 0.97])[torch.arange(M) % 3][:, None]
        allowed[0] = False  # a mask that leaves nothing
        P.grammar_masks = pack_masks(allowed)
        P.grammar_rows = torch.randint(-1, M, (B, R), generator=g)
    return x, ids, P, lengths


def cuda(P):
    return dataclasses.replace(P, **{f.name: v.cuda() for f in dataclasses.fields(P) if isinstance(v := getattr(P, f.name), torch.Tensor)})


def magnitude(x, P, L):
    fine = x.double().abs()
    A = fine[fine.isfinite()].max().item() if fine.isfinite().any() else 0.0
    if P.bias is not None:
        A += P.bias[P.bias.isfinite()].abs().max().item() if P.bias.isfinite().any() else 0.0
    rp = P.repetition_penalty.max().item() if isinstance(P.repetition_penalty, torch.Tensor) else P.repetition_penalty
    big = lambda v: v.abs().max().item() if isinstance(v, torch.Tensor) else abs(v)  # noqa: E731
    return A * rp + big(P.frequency_penalty) * L + big(P.presence_penalty)


def least_t(P):
    return P.temperature.min().item() if isinstance(P.temperature, torch.Tensor) else P.temperature


def same_special(got, want):
    """The same places are infinite and NaN; returns the finite ones."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got == -INF, want == -INF) and torch.equal(got == INF, want == INF)
    return want.isfinite()


def check_logprobs(got, want, A, T):
    got = got.double().cpu()
    fine = same_special(got, want)
    err = (got - want)[fine].abs()
    assert err.numel() == 0 or err.max().item() <= 32 * A / T * 2**-24 + 2**-18, err.max().item()


def check_values(got, want, A, T, dtype):
    """Values formed in fp32 and rounded once."""
    got = got.double().cpu()
    want16 = want
    over = want.abs() > torch.finfo(dtype).max  # rounded to infinity
    want16 = torch.where(over, torch.sign(want) * INF, want)
    fine = same_special(got, want16)
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = 8 * A / T * 2**-24 * (1 + half) + want.abs() * half + tiny
    assert bool(((got - want).abs() <= bound)[fine].all()), ((got - want).abs() / bound)[fine].max().item()


def check_grad(got, want, A, T, dtype, g, slope):
    """Gradients (onehot - p) g slope: p is off by its exponent, 32 A / T 2^-24 + 2^-18 relatively."""
    got = got.double().cpu()
    half = torch.finfo(dtype).eps / 2
    rel = 32 * A / T * 2**-24 + 2**-18
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0**-120
    scale = g.abs()[..., None].double() * slope
    p = torch.minimum(want.abs() / scale.clamp(min=1e-30), torch.ones(()).double())
    near_one = torch.maximum(p, 1 - p)  # the target's 1 - p is off by p's error
    bound = want.abs() * (half + rel + 2**-20) + scale * torch.where(want * g[..., None].sign() > 0, near_one, torch.zeros(()).double()) * rel + tiny
    assert torch.equal(got.isnan(), want.isnan())
    ok = (got - want).abs() <= bound
    assert bool(ok[~want.isnan()].all()), ((got - want).abs() / bound).max().item()


# sizes: one token, a slice of 2048 columns less and more than whole, odd rows, several slices and chunks of rows
SHAPES = [(1, 1, 1, 1), (1, 2, 2, 7), (2, 5, 5, 33), (3, 9, 9, 2047), (2, 70, 70, 515), (1, 3, 3, 2049), (2, 4, 4, 9001), (1, 40, 40, 16411)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,R,L,V", SHAPES)
@pytest.mark.parametrize("K,M", [(0, 0), (5, 0), (0, 4), (3, 4)])
def test_apply_matches_the_definition(dtype, B, R, L, V, K, M):
    x, ids, P, _ = make(B, R, L, V, dtype, seed=B + R + V + K + M, K=K, M=M)
    got = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P))
    assert got.dtype == dtype and got.shape == x.shape
    check_values(got, oracle.process(x, ids, P), magnitude(x, P, L), least_t(P), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,R,L,V", SHAPES[1:])
@pytest.mark.parametrize("K,M", [(0, 0), (4, 4)])
def test_logprobs_and_gradient_match_the_definition(dtype, B, R, L, V, K, M):
    x, ids, P, _ = make(B, R, L, V, dtype, seed=2 * B + R + V + K + M, K=K, M=M)
    xg = x.cuda().requires_grad_(True)
    lp = from_parallel_logits_to_logprobs(xg, ids.cuda(), 0, V, None, logit_processors=cuda(P))
    xo = x.double().requires_grad_(True)
    want = oracle.logprobs(xo, ids, P, rows=R - 1)
    A, T = magnitude(x, P, L), least_t(P)
    check_logprobs(lp.detach(), want.detach(), A, T)
    g = torch.randn(B, R - 1, generator=torch.Generator().manual_seed(1))
    g[:, ::3] = 0  # rows that are not read
    (dx,) = torch.autograd.grad([lp], [xg], [g.cuda()])
    fine = (want.detach() > -INF) & (g != 0)
    total = torch.where(fine, want, torch.zeros_like(want)).mul(g.double()).sum() + 0.0 * xo.sum()
    dxo = torch.autograd.grad([total], [xo], retain_graph=True)[0].nan_to_num(0.0)
    # a row whose token is not allowed still has its probabilities' gradient
    for b, r in ((want.detach() == -INF) & (g != 0)).nonzero().tolist():
        y = oracle.process(xo[b:b + 1, : r + 1], ids[b:b + 1], dataclasses.replace(P, **{
            f.name: v[b:b + 1] for f in dataclasses.fields(P) if isinstance(v := getattr(P, f.name), torch.Tensor)
            and f.name != "grammar_masks"}))[0, r]
        if not bool((y == -INF).all()):
            keep = y.isfinite()
            (d,) = torch.autograd.grad([-torch.logsumexp(y[keep], 0) * g[b, r].double()], [xo])
            dxo[b, r] = d[b, r]
    rp = P.repetition_penalty.max().item()
    assert dx.dtype == dtype and dx.shape == x.shape and not dx[:, -1].any()
    check_grad(dx[:, :-1], dxo[:, :-1], A, T, dtype, g, rp / T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,R,L,V,K,M", [(4, 1, 30, 5003, 3, 3), (3, 3, 17, 2051, 0, 0), (70, 1, 9, 4099, 2, 0), (2, 2, 3000, 700, 4, 3)])
def test_rows_behind_histories(dtype, B, R, L, V, K, M):
    x, ids, P, lengths = make(B, R, L, V, dtype, seed=B + L, K=K, M=M, behind=True)
    lengths[0] = 0  # no history at all
    lengths[-1] = L  # nothing behind the last row
    A, T = magnitude(x, P, L), least_t(P)
    want = oracle.process(x, ids, P, lengths)
    out = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P), history_lengths=lengths.cuda())
    check_values(out, want, A, T, dtype)
    if R == 1:
        two = apply_logit_processors(x[:, 0].cuda(), ids.cuda(), cuda(P), history_lengths=lengths.cuda())
        assert torch.equal(two.view(torch.int16 if dtype != torch.float32 else torch.int32),
                           out[:, 0].contiguous().view(torch.int16 if dtype != torch.float32 else torch.int32))
    place = x.cuda()
    assert apply_logit_processors(place, ids.cuda(), cuda(P), history_lengths=lengths.cuda(), inplace=True) is place
    assert torch.equal(place, out)
    lp = processed_next_token_logprobs(x.cuda(), ids.cuda(), cuda(P), history_lengths=lengths.cuda())
    check_logprobs(lp, oracle.logprobs(x, ids, P, lengths), A, T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,R,V,K,M", [(2, 6, 2051, 3, 3), (1, 40, 600, 0, 0)])
def test_apply_gradient(dtype, B, R, V, K, M):
    x, ids, P, _ = make(B, R, R, V, dtype, seed=V, K=K, M=M)
    xg = x.cuda().requires_grad_(True)
    y = apply_logit_processors(xg, ids.cuda(), cuda(P))
    dy = torch.randn(B, R, V, generator=torch.Generator().manual_seed(3)).to(dtype)
    (dx,) = torch.autograd.grad([y], [xg], [dy.cuda()])
    xo = x.double().requires_grad_(True)
    yo = oracle.process(xo, ids, P)
    (want,) = torch.autograd.grad([yo], [xo], [dy.double()])
    want = want.nan_to_num(0.0)
    got = dx.double().cpu()
    # two factors and their product, each rounded in fp32, then to the type
    bound = want.abs() * (4 * 2**-24 + torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((got - want).abs() <= bound).all())


def test_gradient_against_differences():
    """The fp32 gradient against central differences of the fp64 definition (not its derivative)."""
    B, R, V = 1, 5, 37
    x, ids, P, _ = make(B, R, R, V, torch.float32, seed=5, K=2, M=3)
    P.grammar_rows[:] = torch.tensor([[-1, 1, 2, -1, 2]])
    P.bias[:, 0] = 1.0
    xg = x.cuda().requires_grad_(True)
    lp = from_parallel_logits_to_logprobs(xg, ids.cuda(), 0, V, None, logit_processors=cuda(P))
    fine = torch.isfinite(lp.detach().cpu())
    g = torch.where(fine, torch.randn(B, R - 1, generator=torch.Generator().manual_seed(2)), torch.zeros(B, R - 1))
    (dx,) = torch.autograd.grad([lp], [xg], [g.cuda()])
    h = 1e-5

    def value(z):
        w = oracle.logprobs(z, ids, P, rows=R - 1)
        return torch.where(fine, w, torch.zeros_like(w)).mul(g.double()).sum().item()

    for r, j in [(0, 0), (0, int(ids[0, 1])), (1, int(ids[0, 1])), (2, 3), (3, int(ids[0, 4])), (3, 11)]:
        z = x.double()
        up, down = z.clone(), z.clone()
        up[0, r, j] += h
        down[0, r, j] -= h
        assert abs((value(up) - value(down)) / (2 * h) - dx[0, r, j].item()) < 2e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_places_may_hold_anything(dtype):
    x, ids, P, _ = make(2, 4, 4, 1000, dtype, seed=9, M=3)
    P.grammar_rows[:] = torch.tensor([[1, 2, 1, 2]])
    v = torch.arange(1000)
    allowed = (P.grammar_masks[P.grammar_rows].long()[..., v // 32] >> (v % 32)) % 2 == 1
    clean = torch.where(allowed, x, torch.zeros_like(x))
    dirty = torch.where(allowed, x, torch.tensor([float("nan"), INF, -INF, torch.finfo(dtype).min])[v % 4].to(dtype))
    outs = []
    for t in (clean, dirty):
        t = t.cuda().requires_grad_(True)
        lp = from_parallel_logits_to_logprobs(t, ids.cuda(), 0, 1000, None, logit_processors=cuda(P))
        (dx,) = torch.autograd.grad([lp], [t], [torch.ones_like(lp)])
        y = apply_logit_processors(t.detach(), ids.cuda(), cuda(P))
        outs.append((lp.detach(), dx, y))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_infinity_and_lowest_values(dtype):
    low = torch.finfo(dtype).min
    x, ids, P, _ = make(1, 6, 6, 3000, dtype, seed=11, T=False)
    x[0, 0, 17] = float("nan")
    x[0, 1] = -INF  # nothing left by itself
    x[0, 2] = low
    x[0, 3, :2999] = -INF
    x[0, 4, 5] = INF
    want = oracle.logprobs(x, ids, P, rows=5)
    lp = from_parallel_logits_to_logprobs(x.cuda(), ids.cuda(), 0, 3000, None, logit_processors=cuda(P)).cpu()
    assert lp[0, 0].isnan() and lp[0, 1] == -INF and lp[0, 4].isnan()
    fine = [2, 3]
    assert torch.equal(lp[0, fine] == -INF, want[0, fine] == -INF)
    t = x.cuda().requires_grad_(True)
    out = from_parallel_logits_to_logprobs(t, ids.cuda(), 0, 3000, None, logit_processors=cuda(P))
    (dx,) = torch.autograd.grad([out], [t], [torch.ones_like(out)])
    assert dx[0, 0].isnan().any() and not dx[0, 1].any() and not dx[0, 5].any()
    assert not dx[0, 2:4].isnan().any()


def test_settings_as_numbers_and_off():
    x, ids, P, _ = make(2, 7, 7, 900, torch.float32, seed=4, tensors=False)
    check_values(apply_logit_processors(x.cuda(), ids.cuda(), cuda(P)), oracle.process(x, ids, P), magnitude(x, P, 7), 0.7, torch.float32)
    off = LogitProcessors()
    assert torch.equal(apply_logit_processors(x.cuda(), ids.cuda(), off).cpu(), x)
    assert apply_logit_processors(x, ids, None) is x
    plain = from_parallel_logits_to_logprobs(x.cuda(), ids.cuda(), 0, 900, None)
    mine = from_parallel_logits_to_logprobs(x.cuda(), ids.cuda(), 0, 900, None, logit_processors=off)
    assert (plain - mine).abs().max() <= 2**-18


def test_a_later_bias_of_the_same_token_holds():
    x = torch.zeros(1, 1, 50)
    P = LogitProcessors(bias_ids=torch.tensor([3, 7, 3, -1, 50, 7]), bias=torch.tensor([1.0, 2.0, 5.0, 9.0, 9.0, -INF]))
    y = apply_logit_processors(x.cuda(), torch.zeros(1, 1, dtype=torch.int64, device="cuda"), cuda(P)).cpu()
    want = torch.zeros(50)
    want[3], want[7] = 5.0, -INF
    assert torch.equal(y[0, 0], want)


def test_ids_outside_the_vocabulary_and_vocab_start():
    x, ids, P, _ = make(2, 6, 6, 400, torch.float32, seed=8, K=3)
    ids = ids + 1000
    ids[0, 2], ids[1, 1], ids[1, 4] = -1, 10**12, 1400
    P.bias_ids = P.bias_ids + 1000
    for end in (1400, 1300):
        want = oracle.logprobs(x, ids, P, rows=5, vocab_start=1000, vocab_end=end)
        got = from_parallel_logits_to_logprobs(x.cuda(), ids.cuda(), 1000, end, None, logit_processors=cuda(P))
        check_logprobs(got, want, magnitude(x, P, 6), least_t(P))


def test_strides_and_unaligned_rows():
    big = torch.randn(4, 9, 1031, generator=torch.Generator().manual_seed(0))
    for dtype in DTYPES:
        x = big.to(dtype).cuda()
        view = x.transpose(0, 1)[1:8, :3, 5:1027]  # [7, 3, 1022] rows at odd places
        _, ids, P, _ = make(7, 3, 3, 1022, dtype, seed=2, K=2, M=3)
        wide = torch.zeros(7, 6, dtype=torch.int64)
        wide[:, ::2] = ids
        want = oracle.process(view.cpu(), ids, P)
        A, T = magnitude(view.cpu(), P, 3), least_t(P)
        check_values(apply_logit_processors(view, wide.cuda()[:, ::2], cuda(P)), want, A, T, dtype)
        check_logprobs(from_parallel_logits_to_logprobs(view, ids.int().cuda(), 0, 1022, None, logit_processors=cuda(P)),
                       oracle.logprobs(view.cpu(), ids, P, rows=2), A, T)
        swapped = view.transpose(1, 2).contiguous().transpose(1, 2)  # the vocabulary is not the last in memory
        check_values(apply_logit_processors(swapped, ids.cuda(), cuda(P)), want, A, T, dtype)
        around = x.clone()
        apply_logit_processors(view, ids.cuda(), cuda(P), inplace=True)
        check_values(view, want, A, T, dtype)
        same = torch.ones_like(x, dtype=torch.bool)
        same.transpose(0, 1)[1:8, :3, 5:1027] = False
        assert torch.equal(x[same], around[same])


def test_in_place_touches_only_what_changes():
    x, ids, P, _ = make(3, 1, 40, 5000, torch.bfloat16, seed=1, K=3, behind=True, T=False)
    lengths = torch.tensor([40, 13, 1])
    out = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P), history_lengths=lengths.cuda())
    place = x.cuda()
    version = place._version
    apply_logit_processors(place, ids.cuda(), cuda(P), history_lengths=lengths.cuda(), inplace=True)
    assert torch.equal(place, out) and place._version > version


@pytest.mark.parametrize("top_k,top_p", [(20, 1.0), (None, 0.8), (50, 0.9)])
def test_ahead_of_a_filter(top_k, top_p):
    x, ids, P, _ = make(2, 9, 9, 3001, torch.float32, seed=6, K=3)
    S = TrainingSamplingParams(top_k=top_k, top_p=top_p)
    t = x.cuda().requires_grad_(True)
    got = from_parallel_logits_to_logprobs(t, ids.cuda(), 0, 3001, None, sampling_params=S, logit_processors=cuda(P))
    u = x.cuda().requires_grad_(True)
    want = from_parallel_logits_to_logprobs(apply_logit_processors(u, ids.cuda(), cuda(P)), ids.cuda(), 0, 3001, None, sampling_params=S)
    assert torch.equal(got, want)
    g = torch.where(want.detach().isfinite(), torch.ones_like(want), torch.zeros_like(want))
    (a,) = torch.autograd.grad([got], [t], [g])
    (b,) = torch.autograd.grad([want], [u], [g])
    assert torch.equal(a, b)


def test_results_repeat_and_captured_graphs_replay():
    x, ids, P, _ = make(4, 20, 20, 6007, torch.bfloat16, seed=3, K=4, M=3)
    x, ids, P = x.cuda(), ids.cuda(), cuda(P)
    g = torch.randn(4, 19, device="cuda")

    def step(t):
        t = t.detach().requires_grad_(True)
        lp = from_parallel_logits_to_logprobs(t, ids, 0, 6007, None, logit_processors=P)
        (dx,) = torch.autograd.grad([lp], [t], [g])
        return lp.detach(), dx, apply_logit_processors(t.detach(), ids, P)

    first = [t.clone() for t in step(x)]
    for a, b in zip(first, step(x)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        outs = step(static)
    for k in range(4):
        fresh = (x.float() * (1 + k)).to(x.dtype)
        static.copy_(fresh)
        ids[:, 5] = k  # histories change under a captured graph as well
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(fresh)):
            assert torch.equal(a, b)


def test_another_stream():
    x, ids, P, _ = make(2, 8, 8, 4001, torch.float32, seed=12)
    want = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = apply_logit_processors(x.cuda(), ids.cuda(), cuda(P))
    side.synchronize()
    assert torch.equal(got, want)


def test_second_derivatives_are_refused():
    x, ids, P, _ = make(1, 3, 3, 40, torch.float32, seed=1)
    t = x.cuda().requires_grad_(True)
    lp = from_parallel_logits_to_logprobs(t, ids.cuda(), 0, 40, None, logit_processors=cuda(P))
    (dx,) = torch.autograd.grad([lp.sum()], [t], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
