"""Logprobs from hidden states with adapters beside the output weight, and their gradients, against
64 bits (GPU).

Tolerances, all from the inputs: u = 2^-24 (fp32), e = half a step of the type (bf16 2^-8, fp16
2^-11).  A sum of K products in fp32 is off by at most K u times the sum of magnitudes.
* U: H u sum|d a| s, and its two planes hold it to e^2 (fp16: or 2^-24, half the subnormal step
  on either plane); a logit: H u sum|h w| + r u sum|U b| + sum|dev U||b|.  A logprob: the target's
  deviation plus the largest of its row, plus u (|logprob| 8 + 1.5 spread + 150) for the softmax
  (exp2's argument to u |x - m| log2 e, at most 256 / 4 + 20 + V / 2^14 roundings of the sum).
* G: rounded to the type (e |G|; fp16 times 2^15: or 2^-40), its probabilities off by twice the
  largest logit deviation, relatively.  dH, dU, dA and dB: G's deviation through the sums, K u of
  the sums of magnitudes, the planes of dU and g U (e^2; fp16, scaled by the block's largest
  magnitude: or 2^-38 of that), and the result's own rounding e.
"""

import pytest
import torch

from rl_amd.distributed.model_utils import (
    dropout,
    from_parallel_hidden_states_to_logprobs,
    from_parallel_hidden_states_to_logprobs_with_adapters as with_adapters,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0**-24
BF, HF = torch.bfloat16, torch.float16


def inputs(S, B, H, V, N, r, dtype, seed=0, active=0.6, ids=None, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    x = {
        "hidden": torch.randn(S, B, H, generator=g).to(dtype),
        "weight": (torch.randn(V, H, generator=g) * spread / H**0.5).to(dtype),
        "a": (torch.randn(N, r, H, generator=g) / H**0.5).to(dtype),
        "b": (torch.randn(N, V, r, generator=g) * 0.5 / r**0.5).to(dtype),
        "ids": torch.randint(-1, N, (B,), generator=g) if ids is None else torch.tensor(ids),
        "scaling": 0.5 + torch.rand(N, generator=g),
        "target": torch.randint(0, V, (B, S), generator=g),
        "grad": torch.randn(B, max(S - 1, 0), generator=g) * (torch.rand(B, max(S - 1, 0), generator=g) < active),
    }
    return {k: v.to(DEV) for k, v in x.items()}


def run(x, vs=0, ve=None, grads=("hidden", "a", "b"), **kw):
    """(logprobs, {name: gradient})"""
    leaves = {k: x[k].detach().requires_grad_(k in grads) for k in ("hidden", "a", "b")}
    lp = with_adapters(leaves["hidden"], x["weight"], leaves["a"], leaves["b"], x["ids"], x["scaling"], x["target"], vs,
                       x["weight"].shape[0] if ve is None else ve, **kw)
    if not grads:
        return lp, {}
    got = torch.autograd.grad([lp], [leaves[k] for k in grads], [x["grad"]])
    return lp.detach(), dict(zip(grads, got))


def oracle(x, vs=0, ve=None, keep=None, scale=1.0):
    """{name: (value, tolerance)} in 64 bits on the device."""
    dt = x["hidden"].dtype
    e = torch.finfo(dt).eps / 2
    half = dt == HF
    h, w, a, b = (x[k].double() for k in ("hidden", "weight", "a", "b"))
    S, B, H = h.shape
    V, r, R = w.shape[0], a.shape[1], max(S - 1, 0)
    ve = V if ve is None else ve
    f = torch.ones_like(h) if keep is None else keep.double() * scale
    out = {"lp": torch.zeros(B, R, device=DEV, dtype=torch.float64), "lp_tol": torch.zeros(B, R, device=DEV, dtype=torch.float64)}
    z = {"hidden": h, "a": a, "b": b}
    val = {k: torch.zeros_like(v) for k, v in z.items()}
    tol = {k: torch.zeros_like(v) for k, v in z.items()}
    for i in range(B):
        at = int(x["ids"][i])
        on = 0 <= at < a.shape[0]
        s = float(x["scaling"][at]) if on else 0.0
        ai, bi = (a[at], b[at]) if on else (torch.zeros_like(a[0]), torch.zeros_like(b[0]))
        hi, fi, g = h[:R, i], f[:R, i], x["grad"][i].double()[:, None]
        d = hi * fi
        u = s * (d @ ai.t())
        du_ = s * H * U * (d.abs() @ ai.abs().t()) + e * e * u.abs() + (2.0**-24 if half and on else 0.0)
        lg = hi @ w.t() + u @ bi.t()
        err = H * U * (hi.abs() @ w.abs().t()) + (r * U * u.abs() + du_) @ bi.abs().t() + 2 * U * lg.abs()
        t = x["target"][i, 1:]
        off = (t < vs) | (t >= ve) | (t - vs >= V)
        tt = (t - vs).clamp(0, V - 1)[:, None]
        lse = torch.logsumexp(lg, -1, keepdim=True)
        lp = (lg.gather(1, tt) - lse)[:, 0]
        worst = err.amax(-1, keepdim=True)
        sp = (lg.amax(-1) - lg.amin(-1)).clamp(max=100)
        ltol = err.gather(1, tt)[:, 0] + worst[:, 0] + U * (8 * lp.abs() + 1.5 * sp + 150)
        out["lp"][i], out["lp_tol"][i] = torch.where(off, 0.0, lp), torch.where(off, 0.0, ltol)
        p = (lg - lse).exp()
        one = torch.zeros_like(p).scatter_(1, tt, 1.0) * (~off)[:, None]
        G = one - p
        dG = e * G.abs() + p * (2 * worst + U * (1.5 * sp + 160)[:, None]) + U + (2.0**-40 if half else 0.0)
        g_ = g.abs()
        dU, dU_t = s * g * (G @ bi), s * g_ * ((dG + V * U * G.abs()) @ bi.abs())
        peak_u, peak_g = 2.0**-38 * dU.abs().max(), 2.0**-38 * (g * u).abs().max()
        val["hidden"][:R, i] = g * (G @ w) + fi * (dU @ ai)
        tol["hidden"][:R, i] = g_ * ((dG + V * U * G.abs()) @ w.abs()) + fi * ((dU_t + r * U * dU.abs()) @ ai.abs())
        if on:
            n = 2 * x["grad"].numel()
            val["a"][at] += dU.t() @ d
            tol["a"][at] += (dU_t + (e * e + n * U) * dU.abs() + (peak_u if half else 0.0)).t() @ d.abs()
            gu, gu_t = g * u, g_ * du_
            val["b"][at] += G.t() @ gu
            tol["b"][at] += dG.t() @ gu.abs() + G.abs().t() @ (gu_t + (e * e + n * U) * gu.abs() + (peak_g if half else 0.0))
    for k in val:
        out[k], out[k + "_tol"] = val[k], tol[k] + e * val[k].abs() * (1 + 2.0**-7) + (2.0**-25 if half else 0.0)
    return out


def check(got, grads, want):
    for k, v in {"lp": got, **grads}.items():
        assert v.shape == want[k].shape
        diff = (v.double() - want[k]).abs()
        bad = ~(diff <= want[k + "_tol"])
        assert not bad.any(), f"{k}: {int(bad.sum())} of {bad.numel()}, worst {diff[bad].max().item():.3e} over {want[k + '_tol'][bad].min().item():.3e}"


CASES = [(2, 1, 128, 1, 1, 1), (2, 1, 64, 5, 1, 8), (9, 3, 128, 300, 2, 16), (65, 4, 256, 1000, 3, 12), (33, 20, 100, 777, 7, 5),
         (130, 6, 1000, 4097, 3, 24), (300, 2, 128, 2049, 2, 40), (40, 3, 192, 513, 2, 96), (2, 300, 128, 999, 40, 4),
         (5, 64, 136, 1500, 64, 32), (600, 1, 128, 700, 1, 64)]


@pytest.mark.parametrize("S,B,H,V,N,r", CASES)
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
def test_against_64_bits(S, B, H, V, N, r, dtype):
    print("[case]", S, B, H, V, N, r, flush=True)
    x = inputs(S, B, H, V, N, r, dtype, seed=S + V)
    want = oracle(x)
    check(*run(x), want)
    # fewer gradients asked for, none kept
    for some in (("hidden",), ("a",), ("b",)):
        lp, g = run(x, grads=some)
        check(lp, g, want)
    check(*run(x, grads=()), want)
    check(*run(x, grads=(), inference_only=True), want)


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("S,B,H,V,N,r", [(65, 4, 256, 1000, 3, 12), (33, 5, 100, 777, 2, 16)])
def test_dropout_is_the_dropout_operator(S, B, H, V, N, r, dtype):
    x = inputs(S, B, H, V, N, r, dtype, seed=3)
    keep = dropout(torch.ones(S, B, H, device=DEV), 0.3, 77, offset=5) != 0
    scale = 65536 / (65536 - 19661)
    want = oracle(x, keep=keep, scale=scale)
    check(*run(x, dropout_p=0.3, dropout_seed=77, dropout_offset=5), want)
    check(*run(x, dropout_p=0.3, dropout_seed=torch.tensor([77], device=DEV), dropout_offset=5), want)
    everything = run(x, dropout_p=1.0)  # all dropped: the base model
    check(*everything, oracle(x, keep=torch.zeros_like(keep)))


def test_blocks_give_the_same_gradients():
    """A chunk size bounds a block's rows; here the vocabulary is wide enough for several blocks."""
    S, B, H, V, N, r = 1400, 2, 128, 70000, 3, 8
    x = inputs(S, B, H, V, N, r, BF, seed=5, active=0.7, ids=[2, 0])
    lp, whole = run(x)
    lp2, parts = run(x, chunk_size=16)
    assert torch.equal(lp, lp2)
    want = oracle(x)
    check(lp, whole, want)
    check(lp2, parts, want)


def test_all_ids():
    S, B, H, V, N, r = 40, 6, 128, 600, 3, 8
    for ids in ([-1] * 6, [0] * 6, [2] * 6, [2, 1, 0, -1, 1, 2], [7, -5, 3, 1, 2**40, -(2**50)]):
        x = inputs(S, B, H, V, N, r, BF, seed=7, ids=ids)
        clean = dict(x, ids=torch.tensor([i if 0 <= i < N else -1 for i in ids], device=DEV))
        lp, g = run(x)
        check(lp, g, oracle(clean))
    # rows without an adapter: the base model's logprobs (which rounds its logits to bf16)
    x = inputs(S, B, H, V, N, r, BF, seed=7, ids=[-1] * 6)
    base = from_parallel_hidden_states_to_logprobs(x["hidden"], x["weight"], True, x["target"], 0, V, None)
    assert torch.all((run(x, grads=())[0] - base).abs() <= 2.0**-8 * 2 * 12)


def test_no_active_rows_and_single_adapter_rows():
    x = inputs(20, 4, 128, 500, 2, 8, BF, seed=2, active=0.0)
    lp, g = run(x)
    assert not any(v.any() for v in g.values())
    x["grad"][1, 3] = 2.0
    check(*run(x), oracle(x))
    x["grad"][3, 18] = -1.0
    check(*run(x), oracle(x))


def test_vocabulary_slice():
    x = inputs(30, 3, 128, 700, 2, 8, BF, seed=4)
    x["target"] = torch.randint(-100, 2200, (3, 30), generator=torch.Generator().manual_seed(1)).to(DEV)
    for vs, ve in ((700, 1400), (0, 350), (-50, 5000)):
        want = oracle(x, vs, ve)
        # rows whose target is outside: the gradient of -log-sum-exp without a target is not the
        # reference's: a masked target gives 0 - softmax there, which the oracle has as well
        check(*run(x, vs, ve), want)


def test_a_broken_adapter_or_row_stays_to_itself():
    S, B, H, V, N, r = 40, 6, 128, 600, 3, 8
    x = inputs(S, B, H, V, N, r, BF, seed=7, ids=[0, 1, 2, -1, 1, 0], active=1.0)
    ref_lp, ref = run(x)
    for value in (float("nan"), float("inf")):
        for key, place in (("b", (1, 5, 3)), ("a", (1, 2, 100))):
            y = dict(x, **{key: x[key].clone()})
            y[key][place] = value
            lp, g = run(y)
            assert torch.isnan(lp[[1, 4]]).all() and torch.equal(lp[[0, 2, 3, 5]], ref_lp[[0, 2, 3, 5]])
            assert torch.equal(g["hidden"][:, [0, 2, 3, 5]], ref["hidden"][:, [0, 2, 3, 5]])
            for k in ("a", "b"):
                assert torch.equal(g[k][[0, 2]], ref[k][[0, 2]])
    y = dict(x, hidden=x["hidden"].clone())
    y["hidden"][7, 2, 9] = float("nan")  # one row of adapter 2's only sample
    lp, g = run(y)
    assert torch.isnan(lp[2, 7]) and torch.isnan(lp).sum() == 1
    keep = torch.ones(S, B, dtype=torch.bool, device=DEV)
    keep[7, 2] = False
    assert torch.equal(g["hidden"][keep], ref["hidden"][keep])
    assert torch.equal(g["a"][:2], ref["a"][:2]) and torch.equal(g["b"][:2], ref["b"][:2])


def test_layouts_streams_and_repeat():
    x = inputs(21, 4, 136, 900, 3, 12, BF, seed=9)
    ref_lp, ref = run(x)
    wide = torch.zeros(900, 200, dtype=BF, device=DEV)
    wide[:, 3:139] = x["weight"]
    y = dict(x, weight=wide[:, 3:139], hidden=x["hidden"].transpose(0, 1).contiguous().transpose(0, 1),
             a=x["a"].transpose(0, 1).contiguous().transpose(0, 1), b=x["b"].transpose(1, 2).contiguous().transpose(1, 2),
             target=x["target"].t().contiguous().t(), grad=x["grad"].t().contiguous().t())
    lp, g = run(y)
    assert torch.equal(lp, ref_lp) and all(torch.equal(g[k], ref[k]) for k in g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lp, g = run(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(lp, ref_lp) and all(torch.equal(g[k], ref[k]) for k in g)
    # a broadcast upstream gradient, and a scaling given as a number
    z = dict(x, grad=torch.full((1, 1), 0.5, device=DEV).expand(4, 20))
    check(*run(z), oracle(z))
    lp = with_adapters(x["hidden"], x["weight"], x["a"], x["b"], x["ids"], 0.75, x["target"], 0, 900)
    z = dict(x, scaling=torch.full((3,), 0.75, device=DEV))
    assert torch.equal(lp, run(z, grads=())[0])


def test_captured_and_replayed():
    x = inputs(65, 4, 128, 1000, 3, 16, BF, seed=11)
    leaves = [x[k].requires_grad_(True) for k in ("hidden", "a", "b")]
    seed = torch.tensor([3], device=DEV)

    def step():
        lp = with_adapters(x["hidden"], x["weight"], x["a"], x["b"], x["ids"], x["scaling"], x["target"], 0, 1000,
                           dropout_p=0.1, dropout_seed=seed)
        return (lp.detach(), *torch.autograd.grad([lp], leaves, [x["grad"]]))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x["hidden"].mul_(0.9)
            x["ids"].copy_((x["ids"] + 2) % 4 - 1)
            x["grad"].copy_(x["grad"].roll(3, 1))
        seed.add_(1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_empty():
    x = inputs(1, 3, 128, 300, 2, 8, BF)
    lp, g = run(x)
    assert lp.shape == (3, 0) and not any(v.any() for v in g.values())
    assert with_adapters(x["hidden"], x["weight"], x["a"], x["b"], x["ids"], 1.0, x["target"], 0, 300).shape == (3, 0)


@pytest.mark.parametrize("S,B,H,V,N,r", [(70, 2, 128, 300, 2, 200), (4, 3, 5, 90, 2, 8), (20, 2, 64, 130, 1, 1024),
                                         (2, 1000, 64, 257, 1000, 8), (2, 128, 64, 300, 128, 16), (2, 129, 64, 300, 129, 12)])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
def test_ranks_sizes_and_many_adapters(S, B, H, V, N, r, dtype):
    """Ranks over several tiles, a hidden size below a vector, an adapter for every row of a tile."""
    print("[case]", S, B, H, V, N, r, flush=True)
    x = inputs(S, B, H, V, N, r, dtype, seed=r, ids=[(7 * i) % N for i in range(B)], active=1.0)
    check(*run(x), oracle(x))
    check(*run(x, chunk_size=4), oracle(x))


def test_few_rows_with_a_broken_adapter():
    x = inputs(5, 6, 128, 600, 3, 8, BF, seed=7, ids=[0, 1, 2, -1, 1, 0], active=1.0)
    ref_lp, ref = run(x)
    y = dict(x, b=x["b"].clone())
    y["b"][1, 599, 7] = float("-inf")
    lp, g = run(y)
    assert torch.isnan(lp[[1, 4]]).all() and torch.equal(lp[[0, 2, 3, 5]], ref_lp[[0, 2, 3, 5]])
    assert torch.equal(g["hidden"][:, [0, 2, 3, 5]], ref["hidden"][:, [0, 2, 3, 5]])
    # an adapter that no sample is under may hold anything
    y = dict(x, b=x["b"].clone(), a=x["a"].clone(), ids=torch.tensor([0, 2, 2, -1, 2, 0], device=DEV))
    clean = run(dict(x, ids=y["ids"]))
    y["b"][1], y["a"][1] = float("nan"), float("inf")
    lp, g = run(y)
    assert torch.equal(lp, clean[0]) and all(torch.equal(g[k], clean[1][k]) for k in g)


@pytest.mark.parametrize("S", [3, 100])
def test_adapters_of_more_than_2_gib(S):
    """9 adapters of rank 800 over 151936 tokens are 2.19 GB: past 32-bit byte offsets.  The one in use
    alone takes the other route; both are fp32 sums of the same products, off by at most r u sum|U b|
    each (and the logprob by twice that, its own and the log-sum-exp's)."""
    V, H, r = 151936, 128, 800
    g = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    hidden, weight = rnd(S, 2, H).to(BF), (rnd(V, H) * 0.1).to(BF)
    a, b = (rnd(9, r, H) / H**0.5).to(BF), torch.empty(9, V, r, dtype=BF, device=DEV)
    for i in range(9):
        b[i] = (rnd(V, r) * 0.02).to(BF)
    target = torch.randint(0, V, (2, S), generator=g, device=DEV)
    grad = rnd(2, S - 1)

    def go(a, b, ids):
        h, a, b = (t.detach().requires_grad_(True) for t in (hidden, a, b))
        lp = with_adapters(h, weight, a, b, torch.tensor(ids, device=DEV), 1.0, target, 0, V)
        return (lp.detach(), *torch.autograd.grad([lp], [h, a, b], [grad]))

    far = go(a, b, [8, -1])
    near = go(a[8:], b[8:].contiguous(), [0, -1])
    mag = r * 0.02 * 4  # sum|U b| of r terms of order 1 x 0.02, four standard deviations
    assert (far[0] - near[0]).abs().max() <= 4 * r * U * mag
    for p, q in zip(far[1:], (near[1], near[2], near[3])):
        p = p if p.shape == q.shape else p[8:]
        assert (p.float() - q.float()).norm() <= 2.0**-7 * q.float().norm()
    assert not far[2][:8].any() and not far[3][:8].any()


@pytest.mark.parametrize("S", [9, 200])
@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("H,left,wide", [(40, 24, 64), (128 + 8, 0, 256), (200, 56, 256), (1000, 16, 1024), (72, 8, 400)])
def test_nothing_past_the_weights_rows_is_read(S, dtype, H, left, wide):
    """The weight as columns of a wider tensor whose other columns are NaN (its last row may end the
    storage): what a contiguous copy gives, and what zero-padded hidden states, weight and
    adapters give (the padding adds exact zeros)."""
    x = inputs(S, 2, H, 300, 2, 8, dtype, seed=H, ids=[1, 0])
    buf = torch.full((300, wide), float("nan"), dtype=dtype, device=DEV)
    buf[:, left : left + H] = x["weight"]
    pad = -(-H // 128) * 128 - H
    zero_padded = {k: torch.nn.functional.pad(x[k], (0, pad)) for k in ("hidden", "weight", "a")}
    lp, grads = run({**x, "weight": buf[:, left : left + H]})
    lp2, grads2 = run(x)
    assert torch.equal(lp, lp2) and all(torch.equal(grads[k], grads2[k]) for k in grads)
    lp2, grads2 = run({**x, **zero_padded})  # (dH's sum over the vocabulary is split by the padded size)
    assert torch.equal(lp, lp2) and torch.equal(grads["b"], grads2["b"])


@pytest.mark.parametrize("S", [9, 200])
def test_infinity_in_the_next_row_of_the_weight(S):
    """A token that an infinity rules out (logit -inf) leaves the others as without it."""
    H, V = 200, 300
    x = inputs(S, 2, H, V, 2, 8, BF, ids=[1, 0])
    x["hidden"][..., 0] = x["hidden"][..., 0].abs() + 0.5
    x["target"] = x["target"] % 17
    x["b"][:, 17:] = 0
    weight = x["weight"].clone()
    weight[17:, 0] = -float("inf")
    got, _ = run({**x, "weight": weight}, grads=())
    want = oracle({**x, "weight": weight[:17], "b": x["b"][:, :17].contiguous()})
    assert bool(((got.double() - want["lp"]).abs() <= want["lp_tol"]).all())
