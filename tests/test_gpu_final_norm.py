"""RMS norm with the residual's addition, its backward and its 8-bit output against 64 bits (GPU).

Tolerances.  u = 2^-24 (half a step of fp32).  A row's sum of squares has positive terms and at
most 16 + 6 + 16 additions in sequence for rows that registers hold and H / 8192 * 8 + 22 for
longer ones (at most 60 here), and the square root halves what the sum is off: rstd is within
40 u, y before its rounding within 45 u < 2^-18 of the value, and the rounding to the type adds
half a step, eps / 2 (2^-25 absolute below fp16's normal range).  dh sums three terms: 2^-18 of
the sum of their magnitudes (the mean's terms have either sign).  dw adds at most R / 1024 + 37
terms in sequence: 2^-18 of the sum of the magnitudes for R <= 4096.  e4m3 rounds by at most 2^-4
of the value, or 2^-10 below its normal range.
"""

import pytest
import torch

from rl_amd.distributed.model_utils import add_rms_norm, add_rms_norm_8bit, quantize_rows_8bit, rms_norm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
F32_TOL = 2.0**-18


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2 if t != BF else 0.0


def rows(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def norm64(h, w, eps):
    h, w = h.double(), w.double()
    return h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * w


def close(got, want, magnitude, dtype):
    want = want.double()
    tol = want.abs() * half_step(dtype) * (1 + 2.0**-10) + magnitude * F32_TOL + tiny(dtype)
    diff = (got.double() - want).abs()
    assert torch.all(diff <= tol), f"max excess {(diff - tol).max().item():.3e}"


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 3, 64), (70, 511), (9, 512), (33, 513), (6, 1021), (3, 1024), (5, 1025),
          (4, 2, 2048), (5, 2049), (2, 5, 4096), (3, 4100), (2, 8192), (3, 8197), (2, 16384), (3, 16385), (2, 40003),
          (2100, 96), (1500, 1536)]
TYPES = [(BF, BF, BF), (BF, FP, FP), (BF, BF, FP), (HF, HF, HF), (HF, FP, HF), (FP, FP, FP)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x)[6:] for x in t))
def test_forward_and_backward(shape, types):
    xt, rt, wt = types
    x, res = rows(shape, xt, 1), rows(shape, rt, 2, 3.0)
    w = (1 + 0.3 * rows(shape[-1:], FP, 3)).to(wt)
    dy, dh_out = rows(shape, xt, 4), rows(shape, rt, 5)
    x, res, w = (t.requires_grad_(True) for t in (x, res, w))
    y, h = add_rms_norm(x, res, w, eps=1e-5)
    assert y.dtype == xt and h.dtype == rt and y.shape == h.shape == x.shape
    assert torch.equal(h, (x.float() + res.float()).to(rt))
    h64 = h.detach().double().requires_grad_(True)
    w64 = w.detach().double().requires_grad_(True)
    y64 = norm64(h64, w64, 1e-5)
    close(y.detach(), y64.detach(), y64.detach().abs(), xt)
    dx, dres, dw = torch.autograd.grad([y, h], [x, res, w], [dy, dh_out])
    dh64, dw64 = torch.autograd.grad([y64], [h64, w64], [dy.double()])
    dh64 = dh64 + dh_out.double()
    rstd = (h64.detach().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    n = h64.detach() * rstd
    wdy = w64.detach() * dy.double()
    mag = rstd * (wdy.abs() + n.abs() * (wdy * n).abs().mean(-1, keepdim=True)) + dh_out.double().abs()
    assert dx.dtype == xt and dres.dtype == rt and dw.dtype == wt
    close(dx, dh64, mag, xt)
    close(dres, dh64, mag, rt)
    close(dw, dw64, (dy.double() * n).abs().reshape(-1, shape[-1]).sum(0), wt)
    # only the norm's output has a consumer; only some inputs ask for a gradient
    y, h = add_rms_norm(x, res.detach(), w.detach(), eps=1e-5)
    (dx,) = torch.autograd.grad([y], [x], [dy])
    close(dx, dh64 - dh_out.double(), mag, xt)
    # only the stream has one
    y, h = add_rms_norm(x, res, w, eps=1e-5)
    dx, dres = torch.autograd.grad([h], [x, res], [dh_out])
    assert torch.equal(dres, dh_out) and torch.equal(dx, dh_out.to(xt))


@pytest.mark.parametrize("shape", [(3, 7), (4, 1021), (3, 2, 4096), (2, 20011)], ids=str)
@pytest.mark.parametrize("types", [(BF, BF), (HF, FP), (FP, FP)], ids=lambda t: str(t[0])[6:])
def test_without_a_residual(shape, types):
    xt, wt = types
    x, w, dy = rows(shape, xt, 1, 2.0), (1 + 0.3 * rows(shape[-1:], FP, 3)).to(wt), rows(shape, xt, 4)
    x.requires_grad_(True), w.requires_grad_(True)
    y = rms_norm(x, w)
    x64, w64 = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    y64 = norm64(x64, w64, 1e-6)
    close(y.detach(), y64.detach(), y64.detach().abs(), xt)
    dx, dw = torch.autograd.grad([y], [x, w], [dy])
    dx64, dw64 = torch.autograd.grad([y64], [x64, w64], [dy.double()])
    rstd = (x64.detach().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    n, wdy = x64.detach() * rstd, w64.detach() * dy.double()
    close(dx, dx64, rstd * (wdy.abs() + n.abs() * (wdy * n).abs().mean(-1, keepdim=True)), xt)
    close(dw, dw64, (dy.double() * n).abs().reshape(-1, shape[-1]).sum(0), wt)


def test_gradient_against_differences():
    x, res, w = rows((3, 40), FP, 1), rows((3, 40), FP, 2), 1 + 0.3 * rows((40,), FP, 3)
    dy, d = rows((3, 40), FP, 4), rows((3, 40), FP, 6)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad([add_rms_norm(x, res, w)[0]], [x], [dy])
    step = 2.0**-6
    f = [(add_rms_norm((x + s * d).detach(), res, w)[0].double() * dy.double()).sum() for s in (step, -step)]
    want = (f[0] - f[1]) / (2 * step)
    # third derivatives: |d|^3 step^2 / 6 of values of order one over 120 elements; fp32 of f: 120 * 2^-20 / step
    assert abs((dx.double() * d.double()).sum() - want) < 0.02 * abs(want) + 0.02


def check_8bit(y8, scale, y64):
    amax = y64.abs().amax(-1)
    want = torch.where(amax > 0, (amax / 448).clamp(min=2.0**-126), torch.ones_like(amax))
    assert torch.all((scale.double() - want).abs() <= want * 2.0**-17)
    v = y64 / scale.double()[..., None]
    diff = (y8.double() - v).abs()
    assert torch.all(diff <= v.abs() * 2.0**-4 * (1 + 2.0**-10) + 2.0**-10 * (1 + 2.0**-10))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("types", [(BF, BF, BF), (HF, FP, FP), (FP, FP, FP)], ids=lambda t: str(t[0])[6:])
def test_8bit(shape, types):
    xt, rt, wt = types
    x, res, w = rows(shape, xt, 1), rows(shape, rt, 2, 3.0), (1 + 0.3 * rows(shape[-1:], FP, 3)).to(wt)
    y8, scale, h = add_rms_norm_8bit(x, res, w)
    assert y8.dtype == torch.float8_e4m3fn and scale.shape == shape[:-1]
    assert torch.equal(h, (x.float() + res.float()).to(rt))
    check_8bit(y8, scale, norm64(h, w, 1e-6))
    y8, scale, h = add_rms_norm_8bit(x, None, w)
    assert h is x
    check_8bit(y8, scale, norm64(x, w, 1e-6))
    q8, scale = quantize_rows_8bit(x)
    check_8bit(q8, scale, x.double())


def test_rows_of_zeros_infinities_and_nan():
    x = rows((6, 520), BF, 1)
    w = torch.ones(520, dtype=BF, device=DEV)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 519] = float("inf")
    x[4] = 2.0**-130
    y = rms_norm(x, w, eps=0.0)
    assert torch.isnan(y[1]).all()  # 0 / 0, as the formula has it
    assert not rms_norm(x, w)[1].any()
    assert torch.isnan(y[2]).all() and torch.isnan(y[3, 519])
    assert torch.isfinite(y[[0, 5]]).all()
    q8, scale = quantize_rows_8bit(x)
    assert scale[1] == 1 and not q8[1].float().any()
    assert torch.isnan(scale[2]) and torch.isnan(q8[2].float()).all()
    assert torch.isinf(scale[3]) and torch.isnan(q8[3].float()[519]) and not q8[3].float()[:519].any()
    assert scale[4] == 2.0**-126 and torch.equal(q8[4].float(), torch.full((520,), 2.0**-4, device=DEV))
    check_8bit(q8[[0, 5]], scale[[0, 5]], x[[0, 5]].double())
    y8, scale, _ = add_rms_norm_8bit(x, x, w)
    assert torch.isnan(scale[2]) and scale[1] == 1 and not y8[1].float().any()


def test_strided_rows_and_empty_batches():
    base, wide = rows((4, 6, 300), BF, 1), rows((4, 6, 901), BF, 2)
    w = 1 + rows((300,), BF, 3) * 0.25
    dy = rows((4, 6, 300), BF, 4)
    want = add_rms_norm(base, wide[..., 301:601].contiguous(), w)
    for x, res in ((base, wide[..., 301:601]), (base.transpose(0, 1).contiguous().transpose(0, 1), wide[..., 301:601])):
        got = add_rms_norm(x, res, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = base.clone().requires_grad_(True)
    y, _ = add_rms_norm(x, wide[..., 301:601], w)
    (a,) = torch.autograd.grad([y], [x], [dy], retain_graph=True)
    (b,) = torch.autograd.grad([y], [x], [dy.transpose(0, 1).contiguous().transpose(0, 1)])
    assert torch.equal(a, b)
    (c,) = torch.autograd.grad([add_rms_norm(x, base, w)[0].sum()], [x])  # a broadcast upstream gradient
    (d,) = torch.autograd.grad([add_rms_norm(x, base, w)[0]], [x], [torch.ones_like(x)])
    assert torch.equal(c, d)
    one = rows((5, 1), BF, 5).expand(5, 300)
    assert torch.equal(rms_norm(one, w), rms_norm(one.contiguous(), w))
    e = torch.empty(0, 300, dtype=BF, device=DEV, requires_grad=True)
    wl = w.clone().requires_grad_(True)
    y, h = add_rms_norm(e, e.detach(), wl)
    de, dw = torch.autograd.grad([y], [e, wl], [torch.empty_like(y)])
    assert de.shape == (0, 300) and not dw.any()
    y8, s, _ = add_rms_norm_8bit(e.detach(), None, w)
    assert y8.shape == (0, 300) and s.shape == (0,)


def test_side_stream_graph_and_repeat():
    x, res, w = rows((300, 2048), BF, 1), rows((300, 2048), BF, 2), rows((2048,), BF, 3)
    dy = rows((300, 2048), BF, 4)
    for t in (x, res, w):
        t.requires_grad_(True)

    def step():
        y, h = add_rms_norm(x, res, w)
        return (y.detach(), h.detach(), *torch.autograd.grad([y, h], [x, res, w], [dy, dy]))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(rows((300, 2048), BF, 10 + k))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_no_second_derivative():
    from rl_amd.distributed.model_utils import dropout

    x, w = rows((3, 40), FP, 1).requires_grad_(True), rows((40,), FP, 3).requires_grad_(True)
    for y in (add_rms_norm(x, x, w)[0], rms_norm(x, w), dropout(x, 0.5, 3)):
        dy = torch.ones_like(y).requires_grad_(True)
        (g,) = torch.autograd.grad([y], [x], [dy], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
