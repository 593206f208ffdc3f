"""A broken adapter past 2 GiB of the adapters' storage (GPU): an adapter that no sample is under may hold
anything, also where the few-row kernel's last steps lie past the stages that it has."""

import pytest
import torch

from rl_amd.distributed.model_utils import from_parallel_hidden_states_to_logprobs_with_adapters as with_adapters

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("H", [128, 256, 384])  # 2, 4 and 6 stages: two, one and no step past them
def test_a_broken_adapter_past_2_gib(H):
    V, r, N, S = 151936, 800, 9, 3  # 2.19 GB: byte 2^31 lies in adapter 8, token 126689
    g = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    hidden, weight = rnd(S, 2, H).to(torch.bfloat16), (rnd(V, H) * 0.1).to(torch.bfloat16)
    a, b = (rnd(N, r, H) / H**0.5).to(torch.bfloat16), torch.zeros(N, V, r, dtype=torch.bfloat16, device=DEV)
    b[0] = (rnd(V, r) * 0.02).to(torch.bfloat16)
    target = torch.randint(0, V, (2, S), generator=g, device=DEV)
    ids = torch.tensor([0, -1], device=DEV)
    assert b.nbytes > 2**31 and (2**31 // (r * 2)) // V == 8

    def go():
        return with_adapters(hidden, weight, a, b, ids, 1.0, target, 0, V)

    want = go()
    for value in (float("nan"), float("inf")):
        b[8, 126689:] = value
        assert torch.equal(go(), want)
