"""A vocabulary of one token, whose single row may carry any stride and still be contiguous (GPU): what the
ordinary strides give, and logprobs of 0 (a sum of one exponential, computed in two factors that are each
within 2 u of their value, u = 2^-24, with one rounding between them: its logarithm is within 6 u of 0)."""

import pytest
import torch

from rl_amd.distributed.model_utils import (
    from_parallel_8bit_hidden_states_to_logprobs,
    from_parallel_hidden_states_to_logprobs_with_adapters,
    quantize_rows_8bit,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0**-24


@pytest.mark.parametrize("S", [3, 200])
def test_8bit_row_of_a_wider_buffer(S):
    g = torch.Generator().manual_seed(1)
    hidden = quantize_rows_8bit(torch.randn(S, 2, 20, generator=g).to(DEV))
    buf = torch.full((3, 41), 0x7F, dtype=torch.uint8, device=DEV)
    w8, ws = quantize_rows_8bit(torch.randn(1, 20, generator=g).to(DEV))
    buf[:1, 8:28] = w8.view(torch.uint8)
    row = buf.view(torch.float8_e4m3fn)[:1, 8:28]
    assert row.is_contiguous() and row.stride(0) == 41
    target = torch.zeros(2, S, dtype=torch.int64, device=DEV)
    got, want = (from_parallel_8bit_hidden_states_to_logprobs(*hidden, w, ws, target, 0, 1) for w in (row, w8))
    assert got.shape == (2, S - 1) and torch.equal(got, want) and (got.abs() <= 6 * U).all()


@pytest.mark.parametrize("S", [3, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_adapters_with_b_transposed(S, dtype):
    g = torch.Generator().manual_seed(2)
    hidden, weight, a, bt = (torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((S, 2, 40), (1, 40), (2, 8, 40), (2, 8, 1)))
    target = torch.zeros(2, S, dtype=torch.int64, device=DEV)
    b = bt.transpose(1, 2)
    assert b.shape == (2, 1, 8) and b.is_contiguous() and b.stride(1) == 1

    def go(b):
        h, a_, b = (t.detach().requires_grad_(True) for t in (hidden, a, b))
        lp = from_parallel_hidden_states_to_logprobs_with_adapters(h, weight, a_, b, torch.tensor([1, -1], device=DEV), 1.0, target, 0, 1)
        return (lp.detach(), *torch.autograd.grad([lp.sum()], [h, a_, b]))

    got, want = go(b), go(bt.reshape(2, 1, 8).clone(memory_format=torch.contiguous_format))
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and (got[0].abs() <= 6 * U).all()
