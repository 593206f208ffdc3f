"""The end of a policy as it is used: residual stream -> norm -> logprobs -> gradients (GPU).

The single operators are held to 64 bits by their own tests; here the run of them is compared with
torch's fp32 operations on the same inputs.  Tolerances: y is rounded to bf16 (2^-8 of each
element, independent), which moves a logit of standard deviation 1.5 by 2^-9 * 1.5 rms and six
times that at most over these rows; the base path rounds its logits to bf16 as well (2^-8 of the
largest, 9, for the target and the log-sum-exp).  Gradients: three bf16 roundings in a row (y, G, the
result), 2^-9 rms each, so 2^-7 of their norm bounds the whole.  8 bits: e4m3 rounds by 2^-4, 2^-5.3
rms of either factor; six times 1.5 * 2^-5.3 * sqrt(2).
"""

import pytest
import torch

from rl_amd.distributed.model_utils import HeadAdapters, dropout, from_residual_stream_to_logprobs, quantize_rows_8bit

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
S, B, H, V, N, R = 130, 4, 512, 3000, 3, 16


def inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    bf = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).to(torch.bfloat16).to(DEV)
    x = {"x": bf(S, B, H), "res": bf(S, B, H, k=3), "nw": (1 + 0.1 * torch.randn(H, generator=g)).to(torch.bfloat16).to(DEV),
         "w": bf(V, H, k=1.5 / H**0.5), "a": bf(N, R, H, k=H**-0.5), "b": bf(N, V, R, k=0.5 * R**-0.5)}
    x["target"] = torch.randint(0, V, (B, S), generator=g).to(DEV)
    x["grad"] = (torch.randn(B, S - 1, generator=g) * (torch.rand(B, S - 1, generator=g) < 0.5)).to(DEV)
    return x


def plain(x, ids=None, scaling=0.0, keep=None, scale=1.0):
    """fp32 logprobs and gradients by autograd."""
    v = {k: x[k].float().requires_grad_(True) for k in ("x", "res", "nw", "a", "b", "w")}
    h = v["x"] + v["res"]
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * v["nw"]
    logits = y @ v["w"].t()
    if ids is not None:
        d = y if keep is None else torch.where(keep, y * scale, 0.0)
        parts = []
        for i, a in enumerate(ids):
            if a >= 0:
                parts.append(logits[:, i] + scaling * (d[:, i] @ v["a"][a].t()) @ v["b"][a].t())
            else:
                parts.append(logits[:, i])
        logits = torch.stack(parts, 1)
    lp = torch.log_softmax(logits[:-1], -1).gather(-1, x["target"][:, 1:].t()[..., None])[..., 0].t()
    return lp, v


def near(got, want, rel):
    got, want = got.float(), want.float()
    assert (got - want).norm() <= rel * want.norm(), ((got - want).norm() / want.norm()).item()


def leaves(x, *names):
    return [x[k].detach().requires_grad_(True) for k in names]


def test_training_with_adapters():
    x = inputs()
    ids = [1, -1, 2, 1]
    xs, res, nw, a, b = leaves(x, "x", "res", "nw", "a", "b")
    ad = HeadAdapters(a, b, torch.tensor(ids, device=DEV), 0.8, dropout_p=0.1, dropout_seed=5, dropout_offset=2)
    lp = from_residual_stream_to_logprobs(xs, res, nw, x["w"], x["target"], 0, V, adapters=ad, chunk_size=64)
    keep = dropout(torch.ones(S, B, H, device=DEV), 0.1, 5, offset=2) != 0
    want, v = plain(x, ids, 0.8, keep, 65536 / (65536 - 6554))
    assert lp.shape == (B, S - 1) and (lp - want).abs().max() <= 6 * 1.5 * 2.0**-8
    got = torch.autograd.grad([lp], [xs, res, nw, a, b], [x["grad"]])
    ref = torch.autograd.grad([want], [v[k] for k in ("x", "res", "nw", "a", "b")], [x["grad"]])
    for p, q in zip(got, ref):
        near(p, q, 2.0**-7)


def test_training_without_adapters():
    x = inputs(1)
    xs, res, nw, w = leaves(x, "x", "res", "nw", "w")
    lp = from_residual_stream_to_logprobs(xs, res, nw, w, x["target"], 0, V)
    want, v = plain(x)
    assert (lp - want).abs().max() <= 6 * 1.5 * 2.0**-8 + 2 * 9 * 2.0**-8
    got = torch.autograd.grad([lp], [xs, res, nw, w], [x["grad"]])
    ref = torch.autograd.grad([want], [v[k] for k in ("x", "res", "nw", "w")], [x["grad"]])
    for p, q in zip(got, ref):
        near(p, q, 2.0**-6)


@pytest.mark.parametrize("with_residual", [True, False])
def test_scoring_in_8_bits(with_residual):
    x = inputs(2)
    pair = quantize_rows_8bit(x["w"])
    if not with_residual:
        x["x"], x["res"] = (x["x"].float() + x["res"].float()).to(torch.bfloat16), torch.zeros_like(x["res"])
    lp = from_residual_stream_to_logprobs(x["x"], x["res"] if with_residual else None, x["nw"], pair, x["target"], 0, V)
    want, _ = plain(x)
    assert (lp - want).abs().max() <= 6 * 1.5 * 2.0**-5.3 * 2**0.5


def test_policy_and_reference_in_one_batch():
    """One sample twice, under its adapter and under none: the second is the reference policy."""
    x = inputs(3)
    for k in ("x", "res"):
        x[k] = x[k][:, :1].expand(S, 2, H).contiguous()
    x["target"] = x["target"][:1].expand(2, S).contiguous()
    ad = HeadAdapters(x["a"], x["b"], torch.tensor([2, -1], device=DEV))
    lp = from_residual_stream_to_logprobs(x["x"], x["res"], x["nw"], x["w"], x["target"], 0, V, adapters=ad, inference_only=True)
    want, _ = plain(x, [2, -1], 1.0)
    assert (lp - want).abs().max() <= 6 * 1.5 * 2.0**-8
    assert (lp[0] - lp[1]).abs().max() > 0.1


def test_the_whole_step_captured_and_replayed():
    x = inputs(4)
    xs, res, nw, a, b = leaves(x, "x", "res", "nw", "a", "b")
    ids = torch.tensor([0, 1, -1, 2], device=DEV)

    def step():
        lp = from_residual_stream_to_logprobs(xs, res, nw, x["w"], x["target"], 0, V, adapters=HeadAdapters(a, b, ids, 0.5))
        return (lp.detach(), *torch.autograd.grad([lp], [xs, res, nw, a, b], [x["grad"]]))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        with torch.no_grad():
            xs.mul_(0.9)
            b.mul_(1.1)
            ids.copy_(ids.roll(1))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


@pytest.mark.parametrize("form", ["8 bits", "16 bits", "adapters"])
def test_inference_only_of_a_policy_in_training(form):
    """Parameters that ask for gradients, gradients on: the same logprobs as without, and no graph."""
    x = inputs(5)
    xs, res, nw, a, b, w = leaves(x, "x", "res", "nw", "a", "b", "w")
    weight = quantize_rows_8bit(x["w"]) if form == "8 bits" else w
    ids = torch.tensor([0, 1, -1, 2], device=DEV)
    lp = from_residual_stream_to_logprobs(xs, res, nw, weight, x["target"], 0, V, inference_only=True,
                                          adapters=HeadAdapters(a, b, ids) if form == "adapters" else None)
    assert not lp.requires_grad
    with torch.no_grad():
        want = from_residual_stream_to_logprobs(x["x"], x["res"], x["nw"], weight, x["target"], 0, V,
                                                adapters=HeadAdapters(x["a"], x["b"], ids) if form == "adapters" else None)
    assert torch.equal(lp, want)
