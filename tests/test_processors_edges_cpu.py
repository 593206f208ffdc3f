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
