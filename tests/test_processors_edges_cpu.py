"""Refusals of the logit processors and of the 8-bit integer head beyond those of test_processors_refusals_cpu.py, before
anything is launched."""

import ctypes

import pytest

from rl_amd import _C

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
