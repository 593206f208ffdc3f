"""What the policy head's operators refuse, on the CPU: before any kernel runs."""

import pytest
import torch

from rl_amd import _C
from rl_amd.distributed.model_utils import (
    HeadAdapters,
    add_rms_norm,
    add_rms_norm_8bit,
    dropout,
    from_parallel_8bit_hidden_states_to_logprobs,
    from_parallel_hidden_states_to_logprobs_with_adapters,
    from_residual_stream_to_logprobs,
    quantize_rows_8bit,
    rms_norm,
)

X = torch.randn(3, 8)


def test_cpu_tensors_are_refused():
    w = torch.ones(8)
    for call in (lambda: add_rms_norm(X, X, w), lambda: rms_norm(X, w), lambda: add_rms_norm_8bit(X, X, w),
                 lambda: quantize_rows_8bit(X), lambda: dropout(X, 0.5, 1)):
        with pytest.raises(_C.MirlError, match="ROCm GPU"):
            call()


@pytest.mark.parametrize("x,res,w,eps,err", [
    (X, X, torch.ones(7), 1e-6, ValueError), (X, X[:2], torch.ones(8), 1e-6, ValueError),
    (X.double(), X.double(), torch.ones(8), 1e-6, TypeError), (X, X.bfloat16(), torch.ones(8), 1e-6, TypeError),
    (X.bfloat16(), X.half(), torch.ones(8), 1e-6, TypeError), (X.bfloat16(), X, torch.ones(8).half(), 1e-6, TypeError),
    (X, X, torch.ones(8), -1.0, ValueError), (X, X, torch.ones(8), float("nan"), ValueError),
    (X[:, :0], X[:, :0], torch.ones(0), 1e-6, ValueError), (torch.tensor(1.0), torch.tensor(1.0), torch.ones(1), 1e-6, ValueError),
], ids=str)
def test_norm_refusals(x, res, w, eps, err):
    for call in (add_rms_norm, add_rms_norm_8bit):
        with pytest.raises(err):
            call(x, res, w, eps=eps)


def test_8bit_refuses_gradients():
    x = X.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient"):
        add_rms_norm_8bit(x, X, torch.ones(8))
    with pytest.raises(RuntimeError, match="gradient"):
        quantize_rows_8bit(x)
    with pytest.raises(TypeError):
        quantize_rows_8bit(X.double())


def test_dropout_refusals():
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            dropout(X, p, 1)
    with pytest.raises(TypeError):
        dropout(X.double(), 0.5, 1)


F8 = torch.float8_e4m3fn


def args8(**kw):
    a = dict(h8=torch.zeros(4, 2, 32).to(F8), hs=torch.ones(4, 2), w8=torch.zeros(50, 32).to(F8), ws=torch.ones(50),
             target=torch.zeros(2, 4, dtype=torch.long))
    a.update(kw)
    return (*a.values(), 0, 50)


@pytest.mark.parametrize("change,err", [
    (dict(h8=torch.zeros(4, 2, 32)), TypeError), (dict(w8=torch.zeros(50, 32)), TypeError),
    (dict(h8=torch.zeros(4, 32).to(F8)), ValueError), (dict(w8=torch.zeros(50, 31).to(F8)), ValueError),
    (dict(w8=torch.zeros(0, 32).to(F8), ws=torch.ones(0)), ValueError), (dict(target=torch.zeros(4, 2, dtype=torch.long)), ValueError),
    (dict(hs=torch.ones(2, 4)), ValueError), (dict(hs=torch.ones(4, 2).half()), ValueError), (dict(ws=torch.ones(49)), ValueError),
    ({}, _C.MirlError),
], ids=lambda v: str(list(v)) if isinstance(v, dict) else v.__name__)
def test_8bit_logprobs_refusals(change, err):
    with pytest.raises(err):
        from_parallel_8bit_hidden_states_to_logprobs(*args8(**change))


def adapter_args(**kw):
    bf = torch.bfloat16
    a = dict(hidden=torch.zeros(4, 2, 32, dtype=bf), weight=torch.zeros(50, 32, dtype=bf), a=torch.zeros(3, 8, 32, dtype=bf),
             b=torch.zeros(3, 50, 8, dtype=bf), ids=torch.zeros(2, dtype=torch.long), scaling=1.0,
             target=torch.zeros(2, 4, dtype=torch.long))
    a.update(kw)
    return (*a.values(), 0, 50)


BF = torch.bfloat16


@pytest.mark.parametrize("change,err", [
    (dict(hidden=torch.zeros(4, 2, 32)), TypeError), (dict(a=torch.zeros(3, 8, 32)), TypeError),
    (dict(b=torch.zeros(3, 50, 8).half()), TypeError), (dict(hidden=torch.zeros(4, 32, dtype=BF)), ValueError),
    (dict(weight=torch.zeros(50, 31, dtype=BF)), ValueError), (dict(a=torch.zeros(3, 8, 31, dtype=BF)), ValueError),
    (dict(b=torch.zeros(3, 49, 8, dtype=BF)), ValueError), (dict(b=torch.zeros(2, 50, 8, dtype=BF)), ValueError),
    (dict(b=torch.zeros(3, 50, 7, dtype=BF)), ValueError), (dict(a=torch.zeros(0, 8, 32, dtype=BF), b=torch.zeros(0, 50, 8, dtype=BF)), ValueError),
    (dict(a=torch.zeros(3, 1025, 32, dtype=BF), b=torch.zeros(3, 50, 1025, dtype=BF)), ValueError),
    (dict(ids=torch.zeros(3, dtype=torch.long)), ValueError), (dict(ids=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(target=torch.zeros(4, 2, dtype=torch.long)), ValueError), ({}, _C.MirlError),
    (dict(weight=torch.zeros(50, 32, dtype=BF, requires_grad=True)), NotImplementedError),
], ids=lambda v: str(list(v)) if isinstance(v, dict) else v.__name__)
def test_adapter_refusals(change, err):
    with pytest.raises(err):
        from_parallel_hidden_states_to_logprobs_with_adapters(*adapter_args(**change))


@pytest.mark.parametrize("kw", [dict(chunk_size=0), dict(dropout_p=1.5), dict(dropout_p=float("nan"))], ids=str)
def test_adapter_argument_refusals(kw):
    with pytest.raises(ValueError):
        from_parallel_hidden_states_to_logprobs_with_adapters(*adapter_args(), **kw)


def test_head_refusals():
    x = torch.zeros(4, 2, 32)
    pair = (torch.zeros(50, 32).to(F8), torch.ones(50))
    target = torch.zeros(2, 4, dtype=torch.long)
    ad = HeadAdapters(torch.zeros(1, 8, 32), torch.zeros(1, 50, 8), torch.zeros(2, dtype=torch.long))
    with pytest.raises(NotImplementedError):
        from_residual_stream_to_logprobs(x, x, torch.ones(32), pair, target, 0, 50, adapters=ad)
    with pytest.raises(RuntimeError, match="gradient"):
        from_residual_stream_to_logprobs(x.requires_grad_(True), x.detach(), torch.ones(32), pair, target, 0, 50)


def test_c_entries_return_a_status():
    """Bad arguments come back as a status before any device work."""
    lib = _C.load()
    assert lib.mirl_add_rms_norm_fwd(None, 1, 8, None, 1, 8, None, 1, 4, 8, 1e-6, None, None, None, None, None) != 0
    assert "null" in lib.mirl_last_error().decode()
    assert lib.mirl_add_rms_norm_fwd(None, 1, 8, None, 1, 8, None, 2, 4, 8, 1e-6, None, None, None, None, None) != 0
    assert "weight" in lib.mirl_last_error().decode()
    assert lib.mirl_add_rms_norm_fwd(None, 3, 8, None, 3, 8, None, 3, 4, 8, 1e-6, None, None, None, None, None) != 0
    assert lib.mirl_add_rms_norm_fwd(None, 1, 8, None, 1, 8, None, 1, 4, 0, 1e-6, None, None, None, None, None) != 0
    assert lib.mirl_add_rms_norm_bwd(None, 1, 8, None, 8, None, 1, 8, None, None, 1, 4, 8, None, None, None, None, None) != 0
    assert lib.mirl_add_rms_norm_bwd_workspace_elems(5, 8) == 0  # small: formed in the same launch
    assert lib.mirl_add_rms_norm_bwd_workspace_elems(2048, 1024) == 1024 * 1024
    assert lib.mirl_add_rms_norm_bwd_workspace_elems(0, 8) == 0
    assert lib.mirl_quantize_rows(None, 0, 8, 4, 8, None, None, None) != 0
    assert lib.mirl_dropout(None, 0, 8, 1.5, 1, None, 0, None, None) != 0
    assert "probability" in lib.mirl_last_error().decode()
    assert lib.mirl_dropout(None, 3, 8, 0.5, 1, None, 0, None, None) != 0
    assert lib.mirl_linear_ce_8bit_fwd(None, None, 4, 250, 256, None, None, 10, 256, 2, None, 1, 1, 0, 10, None, 1, 1, None, None) != 0
    assert "256" in lib.mirl_last_error().decode()
    assert lib.mirl_linear_ce_8bit_fwd(None, None, 4, 256, 256, None, None, 10, 256, 2, None, 1, 1, 0, 10, None, 1, 1, None, None) != 0
    assert "null" in lib.mirl_last_error().decode()
    assert lib.mirl_lce_x_workspace_elems(4, 300) == 4 * 3 * 2 + 4 and lib.mirl_lce_x_workspace_elems(200, 300) == 200 * 2 * 2 + 200
    assert lib.mirl_adapter_rows(None, 2, 3, 4, *[None] * 1, 0, 0, None, 0, 0, *[None] * 10, None) != 0
    assert lib.mirl_adapter_rows(None, 0, 3, 4, *[None] * 1, 0, 0, None, 0, 0, *[None] * 10, None) != 0
    assert lib.mirl_adapter_block_workspace_bytes(10, 8, 2) > 0 and lib.mirl_adapter_block_workspace_bytes(0, 8, 2) == 0
    assert lib.mirl_gemm_f16_abt(None, 8, None, 8, 4, 4, 100, 1, None, 4, None, 0, None) != 0
    assert lib.mirl_transpose16(None, 1, 0, 4, 4, 3, None, 0, 8, 8, None, None, 0.0, 0, None, 0, None) != 0
    # nothing to do
    assert lib.mirl_dropout(None, 0, 0, 0.5, 1, None, 0, None, None) == 0
    assert lib.mirl_quantize_rows(None, 0, 8, 0, 8, None, None, None) == 0


def test_layouts_that_the_tile_loop_cannot_read():
    """Refused for their layout, before the pointers are looked at."""
    lib = _C.load()

    def fwd8(Hd, ldh, ldw, w=None):
        return lib.mirl_linear_ce_8bit_fwd(None, None, 4, Hd, ldh, w, None, 10, ldw, 2, None, 1, 1, 0, 10, None, 1, 1, None, None)

    for args in ((250, 256, 250), (252, 256, 256), (252, 252, 252), (256, 264, 256), (272, 272, 272), (256, 256, 240), (252, 256, 252, 2),
                 (256, 256, 272, 4), (256, 256, 256, 6)):
        assert fwd8(*args) != 0 and "multiples of 16" in lib.mirl_last_error().decode(), args
    for args in ((252, 256, 252), (256, 256, 272), (272, 512, 272), (4, 256, 4, 4)):  # readable: the null pointers are next
        assert fwd8(*args) != 0 and "null" in lib.mirl_last_error().decode(), args

    def adapters(Hd, ldh, ldw, w=None):
        return lib.mirl_adapter_ce_fwd(None, 1, 4, Hd, ldh, w, 10, ldw, *[None] * 3, 8, 1, *[None] * 3, 2, None, 1, 1, 0, 10, None, 1, 1,
                                       None, None, None)

    for args in ((12, 128, 16), (16, 16, 16), (136, 136, 136), (128, 128, 120), (128, 132, 128), (128, 128, 132)):
        assert adapters(*args) != 0 and "multiples of 8" in lib.mirl_last_error().decode(), args
    assert adapters(128, 128, 128, 8) != 0 and "aligned" in lib.mirl_last_error().decode()
    assert adapters(136, 256, 136) != 0 and "null" in lib.mirl_last_error().decode()
