"""NaN logits (GPU): a NaN anywhere in a row makes its logprobs NaN, as log_softmax has it, also where a lane or
a wave of the kernels meets nothing but NaN before its first other value; rows without one, and tokens that
are ruled out (-inf), are as they are.  The logits' own path, the K-id gather, and the fp32 hidden-state form
and policy head, whose logits go through the same row kernel."""

import pytest
import torch

from rl_amd import _C
from rl_amd.distributed.model_utils import (
    from_parallel_hidden_states_to_logprobs,
    from_parallel_logits_to_logprobs,
    from_residual_stream_to_logprobs,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NAN, INF = float("nan"), float("inf")
# (V, first, last): the last token alone, a vector, neighbouring vectors, a wave's and a workgroup's first reads
HOLES = [(129, 128, 129), (700, 32, 64), (700, 8, 16), (700, 0, 512), (4097, 4096, 4097), (32000, 64, 72), (32000, 0, 8192),
         (40003, 40002, 40003), (151936, 8, 24), (151936, 0, 65536), (257, 1, 257), (9, 8, 9)]


def rows(V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(2, 5, V, generator=g) * 2).to(dtype).to(DEV)
    target = torch.randint(0, V, (2, 5), generator=g).to(DEV)
    return logits, target


@pytest.mark.parametrize("V,first,last", HOLES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
def test_a_block_of_nan_logits(V, first, last, dtype):
    print("[case]", V, first, last, dtype, flush=True)
    logits, target = rows(V, dtype)
    other = (last if last < V else 0) % V  # a token that is not NaN
    target[:] = other
    want = from_parallel_logits_to_logprobs(logits, target, 0, V, None, inference_only=True)
    assert torch.isfinite(want).all()
    bad = logits.clone()
    bad[0, 2, first:last] = NAN
    got = from_parallel_logits_to_logprobs(bad, target, 0, V, None, inference_only=True)
    assert torch.isnan(got[0, 2])
    got[0, 2] = want[0, 2]
    assert torch.equal(got, want)
    # beside ruled-out tokens only, and with everything NaN
    bad = torch.full_like(logits, -INF)
    bad[..., other] = 0.0
    clean = from_parallel_logits_to_logprobs(bad, target, 0, V, None, inference_only=True)
    assert not clean.any()
    bad[..., first] = NAN
    assert torch.isnan(from_parallel_logits_to_logprobs(bad, target, 0, V, None, inference_only=True)).all()
    bad[:] = NAN
    assert torch.isnan(from_parallel_logits_to_logprobs(bad, target, 0, V, None, inference_only=True)).all()


@pytest.mark.parametrize("V,first,last", HOLES)
def test_gathered_logprobs(V, first, last):
    logits, _ = rows(V, torch.bfloat16, 1)
    other = (last if last < V else 0) % V
    ids = torch.full((2, 5, 3), other, device=DEV)
    logits[1, 4, first:last] = NAN
    out = torch.empty(2, 5, 3, device=DEV)
    _C.gather_logprob_fwd(logits, ids, 0, V, out, None)
    assert torch.isnan(out[1, 4]).all() and torch.isnan(out).sum() == 3


@pytest.mark.parametrize("V,first,last", [(129, 128, 129), (700, 32, 64), (700, 256, 512), (32001, 32000, 32001)])
def test_fp32_hidden_states_and_policy_head(V, first, last):
    g = torch.Generator().manual_seed(3)
    x, weight = torch.randn(9, 2, 64, generator=g).to(DEV), (torch.randn(V, 64, generator=g) * 0.2).to(DEV)
    norm, target = torch.ones(64, device=DEV), torch.full((2, 9), 5, device=DEV)
    hidden = lambda: from_parallel_hidden_states_to_logprobs(x, weight, True, target, 0, V, None)
    head = lambda: from_residual_stream_to_logprobs(x, x, norm, weight, target, 0, V)
    assert torch.isfinite(hidden()).all() and torch.isfinite(head()).all()
    weight[first:last] = NAN
    assert torch.isnan(hidden()).all() and torch.isnan(head()).all()
