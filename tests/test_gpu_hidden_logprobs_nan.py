"""NaN logits of the fused hidden-state logprobs (GPU): a NaN anywhere in a row's vocabulary makes its logprob
NaN, as log_softmax has it, also where it holds all columns that a wave or a tile of the kernels takes
(the last one of a vocabulary one past a tile, a block of neighbouring tokens); a token that is ruled out
(a logit of -inf) leaves the others as they are.  Row counts on both sides of the few-row kernels."""

import pytest
import torch

from rl_amd.distributed.model_utils import (
    from_parallel_8bit_hidden_states_to_logprobs,
    from_parallel_hidden_states_to_logprobs,
    from_parallel_hidden_states_to_logprobs_with_adapters,
    quantize_rows_8bit,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAN = float("nan")
FORMS = ["adapters-bf16", "adapters-f16", "base-bf16", "base-f16", "8bit", "8bit-scale"]
# (V, the tokens that are NaN): one past a tile of 256, past a wave's 32; whole waves, tiles and their neighbours
HOLES = [(257, 256, 257), (32001, 32000, 32001), (129, 128, 129), (700, 32, 64), (700, 128, 256), (700, 256, 512),
         (700, 255, 513), (513, 512, 513)]


def inputs(S, V, H=136, seed=0):
    g = torch.Generator().manual_seed(seed)
    B = 2
    hidden, weight = torch.randn(S, B, H, generator=g), torch.randn(V, H, generator=g) * 0.12
    ids = torch.tensor([1, -1])
    a, b = torch.randn(2, 8, H, generator=g) / H**0.5, torch.randn(2, V, 8, generator=g) * 0.2
    return [t.to(DEV) for t in (hidden, weight, torch.randint(0, V, (B, S), generator=g), ids, a, b)]


def logprobs(form, hidden, weight, target, ids, a, b, first=0, last=0, value=NAN, graph=False):
    """Logprobs with weight rows first .. last (or, "8bit-scale", their scales) of `value`."""
    V = weight.shape[0]
    if form.startswith("8bit"):
        h8, w8 = quantize_rows_8bit(hidden), quantize_rows_8bit(weight)
        w, s = w8[0].clone(), w8[1].clone()
        if form == "8bit":
            w.view(torch.uint8)[first:last] = 0x7F  # e4m3's NaN
        else:
            s[first:last] = value
        return from_parallel_8bit_hidden_states_to_logprobs(*h8, w, s, target, 0, V)
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16}[form.split("-")[1]]
    weight = weight.clone()
    weight[first:last] = value
    h, w = hidden.to(dtype).requires_grad_(graph), weight.to(dtype)
    if form.startswith("base"):
        lp = from_parallel_hidden_states_to_logprobs(h, w, True, target, 0, V, None)
    else:
        lp = from_parallel_hidden_states_to_logprobs_with_adapters(h, w, a.to(dtype), b.to(dtype), ids, 0.5, target, 0, V)
    return (lp.detach(), torch.autograd.grad([lp.sum()], [h])[0]) if graph else lp


@pytest.mark.parametrize("S", [9, 90])
@pytest.mark.parametrize("V,first,last", HOLES)
@pytest.mark.parametrize("form", FORMS)
def test_a_block_of_nan_tokens(form, V, first, last, S):
    print("[case]", form, V, first, last, S, flush=True)
    hidden, weight, target, *rest = inputs(S, V)
    assert torch.isfinite(logprobs(form, hidden, weight, target, *rest)).all()
    # targets elsewhere, so that no logprob is NaN by its own logit
    target = torch.where((target >= first) & (target < last), target % first, target)
    assert torch.isnan(logprobs(form, hidden, weight, target, *rest, first, last)).all()


@pytest.mark.parametrize("S", [9, 90])
@pytest.mark.parametrize("form", FORMS)
def test_everything_is_nan(form, S):
    hidden, weight, target, *rest = inputs(S, 300)
    assert torch.isnan(logprobs(form, hidden, weight, target, *rest, 0, 300)).all()


@pytest.mark.parametrize("S", [9, 90])
@pytest.mark.parametrize("form", ["adapters-bf16", "adapters-f16", "base-bf16", "base-f16"])
def test_a_block_of_ruled_out_tokens(form, S):
    """Whole groups of -inf logits take no part; one NaN among them shows."""
    V = 700
    hidden, weight, target, ids, a, b = inputs(S, V)
    hidden[..., 0] = hidden[..., 0].abs() + 0.5
    weight[:, 0] = 0
    b[:, 256:] = 0
    target = target % 256
    short = weight.clone()[:256]
    want = logprobs(form, hidden, short, target, ids, a, b[:, :256].contiguous())
    weight[256:] = 0
    weight[256:, 0] = -float("inf")
    # the sums of a tile and of waves are the same ones: only their join has more terms, which are 0
    got = logprobs(form, hidden, weight, target, ids, a, b)
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 2.0**-20
    weight[699] = NAN
    assert torch.isnan(logprobs(form, hidden, weight, target, ids, a, b)).all()


@pytest.mark.parametrize("form", ["adapters-bf16", "base-bf16"])
def test_the_gradient_is_nan_where_the_logprob_is(form):
    hidden, weight, target, *rest = inputs(9, 257)
    lp, dh = logprobs(form, hidden, weight, target % 256, *rest, 256, 257, graph=True)
    assert torch.isnan(lp).all() and torch.isnan(dh[:8]).all() and not dh[8].any()
