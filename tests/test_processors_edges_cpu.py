"""Refusals of the logit processors and of the 8-bit integer head beyond those of test_processors_refusals_cpu.py, before
anything is launched."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from rl_amd import _C
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors, TrainingSamplingParams, apply_logit_processors
from rl_amd.distributed.model_utils import (from_int8_hidden_states_to_logits, from_parallel_8bit_hidden_states_to_logprobs,
                                            from_parallel_logits_to_logprobs, from_residual_stream_to_logprobs,
                                            processed_next_token_logprobs)

V = 40


@pytest.fixture(autouse=True)
def no_message_left():
    yield
    assert _C.load().mirl_dropout(None, 0, 0, 0.5, 0, None, 0, None, None) == 0  # (a call that succeeds clears it)


def settings(**fields):
    A = _C.LogitProcessorArgs()
    A.vocab_end = V
    for name, value in fields.items():
        setattr(A, name, value)
    return ctypes.byref(A)


def refused(status, word):
    return status != 0 and word in _C.load().mirl_last_error().decode()


def test_the_fp32_c_entry_points():
    lib = _C.load()
    one = 16  # an address that is never read
    fwd = lambda x=None, dtype=0, b=1, v=V, out=None: lib.mirl_process_logits_f32(x, dtype, b, 1, v, v, v, settings(), one, out, v, v, out, None)  # noqa: E731
    bwd = lambda x=None, dtype=0, b=1, v=V: lib.mirl_process_logits_f32_bwd(x, dtype, b, 1, v, v, v, settings(), one, None, v, v, None, v, v, None)  # noqa: E731
    for call in (fwd, bwd):
        assert refused(call(dtype=3), "dtype") and refused(call(v=0), "shape") and refused(call(b=-1), "shape") and refused(call(), "null")
        assert call(b=0) == 0
    assert refused(fwd(x=one, out=one), "in place")


def test_sizes_that_no_launch_holds():
    """A launch holds fewer than 2^32 threads: of the table 1024 for each list of a sample, of the join 64 a row.  The sizes are
    refused ahead of any launch, and those below end at the missing pointers."""
    lib = _C.load()
    none = (None,) * 5

    def fwd(b, r, v=V, **fields):
        return lib.mirl_processed_logprob_fwd(None, 0, b, r, v, r * v, v, settings(**fields), *none)

    def process(b, r, v=V, **fields):
        return lib.mirl_process_logits(None, 0, b, r, v, r * v, v, settings(**fields), None, None, r * v, v, None)

    def bwd(b, r, v=V, **fields):
        return lib.mirl_processed_logprob_bwd(None, 0, b, r, r, v, r * v, v, settings(**fields), None, None, None, r, 1, None, r * v, v, None)

    some = dict(ids=16, bias_ids=16, bias=16)
    for call in (fwd, process, bwd):
        assert refused(call(1 << 22, 1), "lists") and refused(call((1 << 22) - 1, 1), "null")
        assert refused(call(1 << 21, 1, n_bias=1, **some), "lists") and refused(call((1 << 21) - 1, 1, n_bias=1, **some), "null")
        assert refused(call(1 << 14, 1, n_ids=(1 << 20) - 1, **some), "lists") and refused(call((1 << 14) - 1, 1, n_ids=(1 << 20) - 1, **some), "null")
        assert refused(call(2, 1 << 62), "2^31") and refused(call(1 << 62, 4), "2^31")  # (products past 64 bits)
    assert refused(fwd(1, 1 << 26), "scored") and refused(fwd(1, (1 << 26) - 1), "null")
    assert refused(process(1, 1 << 26), "null")  # (no join)


def test_int8_rows_that_no_launch_merges():
    lib = _C.load()

    def fwd(T):
        return lib.mirl_linear_ce_int8_fwd(None, None, T, 256, 256, None, None, 5, 256, 1, None, 1, 1, 0, 5, None, 1, 1, None, None)

    assert refused(fwd(1 << 26), "scored") and refused(fwd((1 << 26) - 1), "null")


@pytest.mark.parametrize("which", ["hidden", "weight"])
def test_int8_scales_take_no_gradient(which):
    h, w = torch.zeros(2, 2, 16, dtype=torch.int8), torch.zeros(5, 16, dtype=torch.int8)
    hs, ws = torch.ones(2, 2, requires_grad=which == "hidden"), torch.ones(5, requires_grad=which == "weight")
    target = torch.zeros(2, 2, dtype=torch.int64)
    calls = [lambda: from_int8_hidden_states_to_logits(h, hs, w, ws),
             lambda: from_parallel_8bit_hidden_states_to_logprobs(h, hs, w, ws, target, 0, 5)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient passes"):
            call()
        with torch.no_grad(), pytest.raises(_C.MirlError):  # (no GPU here: the call is taken)
            call()
    e4m3 = torch.float8_e4m3fn
    with pytest.raises(_C.MirlError):  # as before
        from_parallel_8bit_hidden_states_to_logprobs(h.to(e4m3), hs, w.to(e4m3), ws, target, 0, 5)


def test_int8_weight_scales_of_the_policy_head_take_no_gradient(monkeypatch):
    w, ws = torch.zeros(5, 16, dtype=torch.int8), torch.ones(5, requires_grad=True)
    rows = (torch.zeros(2, 1, 16, dtype=torch.int8), torch.ones(2, 1), None)
    monkeypatch.setattr("rl_amd.distributed.policy_head.add_rms_norm_8bit", lambda *a: rows)  # (the norm needs a GPU)
    for P in (None, LogitProcessors(temperature=0.7)):
        with pytest.raises(RuntimeError, match="no gradient passes"):
            from_residual_stream_to_logprobs(torch.zeros(2, 1, 16), None, torch.ones(16), (w, ws), torch.zeros(1, 2, dtype=torch.int64), 0, 5, logit_processors=P)


@pytest.mark.parametrize("what", ["logits", "bias", "temperature"])
def test_forward_mode_tangents_are_refused(what):
    """Not taken without their tangents: neither where a graph is recorded nor where none is."""
    ids = torch.zeros(2, 3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        x = torch.zeros(2, 3, V)
        P = LogitProcessors(temperature=torch.ones(2), bias_ids=torch.zeros(4, dtype=torch.int64), bias=torch.zeros(4))
        if what == "logits":
            x = dual(x)
        else:
            setattr(P, what, dual(getattr(P, what)))
        F = TrainingSamplingParams(top_k=3)
        for call in (lambda: apply_logit_processors(x, ids, P), lambda: apply_logit_processors(x, ids, P, inplace=True),
                     lambda: processed_next_token_logprobs(x, ids, P),
                     lambda: from_parallel_logits_to_logprobs(x, ids, 0, V, None, logit_processors=P),
                     lambda: from_parallel_logits_to_logprobs(x, ids, 0, V, None, sampling_params=F, logit_processors=P)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                call()
        h, w, hs, ws = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(5, 16, dtype=torch.int8), torch.ones(2), torch.ones(5)
        with pytest.raises(NotImplementedError, match="tangent"):
            from_int8_hidden_states_to_logits(h, dual(hs), w, ws)
    plain = LogitProcessors(repetition_penalty=1.1)
    with pytest.raises(_C.MirlError):  # (no GPU here: a call without a tangent is taken)
        apply_logit_processors(torch.zeros(2, 3, V), ids, plain)
