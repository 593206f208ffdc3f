"""fp16 adapters of far different magnitudes in one backward block (GPU): each adapter's gradients are what they
are without the other's size, bit for bit."""

import pytest
import torch

from test_gpu_linear_ce_adapters import check, inputs, oracle, run

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("S,r", [(9, 12), (200, 12), (40, 96)])
@pytest.mark.parametrize("scaling", [3e4, 1e8, 1e13])
def test_gradients_beside_a_large_adapter(S, r, scaling):
    """Adapter 1's rows have a U of some `scaling` and no B, so their logits are the base model's."""
    x = inputs(S, 6, 136, 700, 3, r, torch.float16, seed=S, ids=[1, 0, 2, -1, 0, 1], active=0.8)
    x["b"][1] = 0
    x["scaling"][1] = 1.0
    want = oracle(x)
    lp, g = run(x)
    check(lp, g, want)
    x["scaling"][1] = scaling
    lp2, g2 = run(x)
    assert torch.equal(lp, lp2) and torch.equal(g["hidden"], g2["hidden"])
    for k in ("a", "b"):
        assert torch.equal(g[k][[0, 2]], g2[k][[0, 2]])
    lp3, g3 = run(x, chunk_size=4)
    check(lp3, {k: g3[k][[0, 2]] for k in ("a", "b")},
          {"lp": lp.double(), "lp_tol": torch.zeros_like(lp), **{k: want[k][[0, 2]] for k in ("a", "a_tol", "b", "b_tol")}})


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_small_gradients_beside_large_ones(dtype):
    """Upstream gradients of some 2^-8 in one adapter's samples beside 2^4 in another's."""
    x = inputs(60, 4, 128, 500, 2, 8, dtype, seed=2, ids=[0, 1, 0, 1], active=1.0)
    small, large = x["grad"].clone() * 2.0**-8, x["grad"].clone()
    y = dict(x, grad=torch.where(x["ids"][:, None] == 0, small, large * 2.0**4))
    z = dict(x, grad=torch.where(x["ids"][:, None] == 0, small, small))
    (_, g), (_, g2) = run(y), run(z)
    assert torch.equal(g["a"][0], g2["a"][0]) and torch.equal(g["b"][0], g2["b"][0]) and g["b"][0].any()
