"""The norm's weight gradient over many rows, against its exact value (GPU).

Rows of ones under eps 0 have rstd 1 exactly, so a column of dw is R times its dy: a constant, chosen
with 24 significant bits, whose running sum rounds in one direction for a whole binade at a time.
Bound: dw adds at most R / 1024 + 37 terms in sequence, each addition off by half a step (u = 2^-24) of
a partial sum that is at most the whole one.  In chains of R / 16 these columns would be off by 240 u of
the sum at R = 16384 and 850 u at R = 60000, where the bound is 53 u and 96 u.
"""

import pytest
import torch

from rl_amd.distributed.model_utils import add_rms_norm, rms_norm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0**-24
C = (1.1248482465744019, 1.224725604057312, 1.3745416402816772, 1.4119956493377686, 1.2372102737426758)


@pytest.mark.parametrize("R,H", [(1, 5), (16, 1), (771, 1021), (1024, 1023), (1025, 64), (1024, 17), (300, 3000), (200, 5000),
                                 (63, 16384), (4097, 250), (16384, 17), (16384, 64), (60000, 17), (1 << 20, 1)])
def test_the_bound_on_the_weight_gradient(R, H):
    print("[case]", R, H, flush=True)
    dy = torch.tensor(C, device=DEV).repeat(-(-H // len(C)))[:H].contiguous()
    x, w = torch.ones(R, H, device=DEV), torch.ones(H, device=DEV, requires_grad=True)
    want = R * dy.double()
    for y in (rms_norm(x, w, eps=0.0), add_rms_norm(x, torch.zeros_like(x), w, eps=0.0)[0]):
        (dw,) = torch.autograd.grad([y], [w], [dy.expand(R, H).contiguous()])
        assert torch.all((dw.double() - want).abs() <= (R / 1024 + 37) * U * want)


@pytest.mark.parametrize("R,H", [(1023, 40), (1024, 40), (1025, 40), (2100, 96), (16384, 17), (3000, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
def test_random_rows(R, H, dtype):
    """Both sides of the rule by which rows are shared out: rstd is within 40 u, a term within 42 u of its
    value, the sum within R / 1024 + 37 u more, and dw is rounded to its type once."""
    g = torch.Generator().manual_seed(R + H)
    x, res, dy = (torch.randn(R, H, generator=g).to(dtype).to(DEV) for _ in range(3))
    w = (1 + 0.3 * torch.randn(H, generator=g)).to(dtype).to(DEV).requires_grad_(True)
    y, h = add_rms_norm(x, res, w, eps=1e-5)
    (dw,) = torch.autograd.grad([y], [w], [dy])
    h = h.double()
    terms = dy.double() * h * (h.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    want = terms.sum(0)
    tol = (R / 1024 + 79) * U * terms.abs().sum(0)
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
    assert torch.all((dw.double() - want).abs() <= tol)
