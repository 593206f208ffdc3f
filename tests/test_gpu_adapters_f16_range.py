"""fp16 adapters whose U passes the type's range (65504) while the logits do not (GPU): U is held in fp32,
so such rows have the logprobs and gradients of the formula.  Inputs, oracle and its tolerances are those of
the adapters' tests.  Their term for U's two planes (2^-22 |u| and 2^-24) holds here as well: a row past the
range enters times a power of two that takes its largest |u| to 2^14 .. 2^15, so that half a subnormal step of a
plane is at most 2^-39 of that |u|, which is less than the 2^-22 |u| of the largest value alone."""

import pytest
import torch

from test_gpu_linear_ce_adapters import check, inputs, oracle, run

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HF = torch.float16

CASES = [(9, 3, 128, 300, 2, 16), (9, 3, 128, 40, 2, 1), (90, 4, 256, 1000, 3, 8), (70, 2, 128, 300, 2, 96), (300, 2, 200, 520, 2, 40)]


def wide_inputs(S, B, H, V, N, r, seed, ids=None):
    """Adapter 1 has U of up to some 2e5 and a B that is as much smaller; gradients that dB in fp16 can hold."""
    x = inputs(S, B, H, V, N, r, HF, seed=seed, ids=[(1 + i) % N for i in range(B)] if ids is None else ids)
    x["scaling"][1] = 60000.0
    x["b"][1] *= 2.0**-9
    x["grad"] *= 2.0**-6
    d = x["hidden"][: S - 1, 0].double() @ x["a"][1].double().t()
    assert x["ids"][0] == 1 and (d.abs() * 60000).max() > 65520
    return x


@pytest.mark.parametrize("S,B,H,V,N,r", CASES)
def test_u_past_the_range(S, B, H, V, N, r):
    print("[case]", S, B, H, V, N, r, flush=True)
    x = wide_inputs(S, B, H, V, N, r, seed=S)
    want = oracle(x)
    check(*run(x), want)
    check(*run(x, grads=()), want)
    check(*run(x, chunk_size=4), want)


@pytest.mark.parametrize("S", [9, 200])
def test_the_other_rows_are_as_before(S):
    """Rows of other adapters and of the base model beside such rows, bit for bit; a broken adapter there
    as well."""
    ids = [1, 0, 2, -1]
    x = wide_inputs(S, 4, 136, 700, 3, 12, seed=3, ids=ids)
    y = dict(x, scaling=x["scaling"].clone())
    y["scaling"][1] = 1.0
    (lp, g), (lp2, g2) = run(x), run(y)
    assert torch.isfinite(lp).all()
    assert torch.equal(lp[1:], lp2[1:]) and torch.equal(g["hidden"][:, 1:], g2["hidden"][:, 1:])
    z = dict(x, b=x["b"].clone())
    z["b"][2, 650, 3] = float("inf")
    lp3, g3 = run(z)
    assert torch.isnan(lp3[2]).all() and torch.equal(lp3[[0, 1, 3]], lp[[0, 1, 3]])
    assert torch.equal(g3["hidden"][:, [0, 1, 3]], g["hidden"][:, [0, 1, 3]])


@pytest.mark.parametrize("S", [9, 200])
@pytest.mark.parametrize("scaling", [1e9, 1e30])
def test_far_past_the_range(S, scaling):
    """A B of zeros takes any finite U out: the base model's logprobs (whose sums in fp32 the scaling by a
    power of two leaves as they are), and no gradient of A."""
    x = inputs(S, 2, 128, 300, 2, 8, HF, seed=5, ids=[1, -1])
    x["b"][1] = 0
    base, _ = run(dict(x, ids=torch.tensor([-1, -1], device=DEV)), grads=())
    x["scaling"][1] = scaling
    lp, g = run(x, grads=("hidden", "a"))
    assert torch.equal(lp, base) and torch.isfinite(g["hidden"]).all() and not g["a"].any()


def test_an_infinite_u_makes_its_row_nan():
    x = inputs(9, 3, 128, 300, 2, 8, HF, seed=6, ids=[1, 0, 1])
    ref, _ = run(x, grads=())
    y = dict(x, hidden=x["hidden"].clone())
    y["hidden"][4, 0, 7] = float("inf")
    lp, _ = run(y, grads=())
    assert torch.isnan(lp[0, 4])
    lp[0, 4] = ref[0, 4]
    assert torch.equal(lp, ref)


def test_captured_and_replayed():
    x = wide_inputs(90, 2, 128, 700, 2, 8, seed=7)
    scaling = x["scaling"]
    leaves = [x[k].requires_grad_(True) for k in ("hidden", "a", "b")]
    from rl_amd.distributed.model_utils import from_parallel_hidden_states_to_logprobs_with_adapters as with_adapters

    def step():
        lp = with_adapters(x["hidden"], x["weight"], x["a"], x["b"], x["ids"], scaling, x["target"], 0, 700)
        return (lp.detach(), *torch.autograd.grad([lp], leaves, [x["grad"]]))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for s in (60000.0, 1.0, 50000.0, 2.0):  # past the range in one replay, within it in the next
        scaling[1] = s
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager)) and torch.isfinite(out[0]).all()
