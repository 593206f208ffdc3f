"""The run of the sampler's head by blocks of positions: operands that have to be laid out anew are laid out once a call."""

import pytest
import torch

from rl_amd.algorithms.logits_sampling_utils import LogitProcessors
from rl_amd.distributed.model_utils import (add_rms_norm_8bit, from_int8_hidden_states_to_logits, from_residual_stream_to_logprobs,
                                            processed_next_token_logprobs, quantize_rows_8bit)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,gap,offset", [(1001, 0, 0), (512, 3, 0), (512, 0, 1)])  # odd rows, rows with gaps, an odd start
def test_the_weight_is_laid_out_once(H, gap, offset):
    S, B, V = 33, 2, 4000
    g = torch.Generator().manual_seed(H)
    x, norm = torch.randn(S, B, H, generator=g).cuda(), torch.ones(H, device="cuda")
    w8, ws = quantize_rows_8bit(torch.randn(V, H, generator=g).cuda(), torch.int8)
    buffer = torch.zeros(V * (H + gap) + 16, dtype=torch.int8, device="cuda")
    weight = buffer[offset:offset + V * (H + gap)].view(V, H + gap)[:, :H]
    weight.copy_(w8)
    ids = torch.randint(0, V, (B, S), generator=g).cuda()
    P = LogitProcessors(repetition_penalty=1.2, temperature=0.8)
    y8, scale, _ = add_rms_norm_8bit(x, None, norm, dtype=torch.int8)
    logits = from_int8_hidden_states_to_logits(y8, scale, w8, ws, torch.float32).transpose(0, 1)
    want = processed_next_token_logprobs(logits, ids, P)
    for chunk in (1, 5, None):
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
        got = from_residual_stream_to_logprobs(x, None, norm, (weight, ws), ids, 0, V, chunk_size=chunk, logit_processors=P)
        taken = torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before
        assert (got - want).abs().max() <= 2**-16  # (the rows of a block may go to another kernel: the same logits, sums in another order)
        # one copy of the weight (rows padded to 256 bytes), the logits of one or two block sizes, and for each block
        # what its logprobs work on (partials, the table: under 4 words a column and 64 KB)
        step = chunk or S - 1
        blocks = -(-(S - 1) // step)
        small = blocks * (B * V * 16 + (1 << 16)) + 2 * step * B * V * 4 + 8 * S * B * 1280
        assert taken <= V * (-(-H // 256) * 256) + small + (1 << 20)
