"""What the logit processors and the 8-bit integer head refuse, before anything is launched."""

import ctypes

import pytest
import torch

from rl_amd import _C
from rl_amd.algorithms.logits_sampling_utils import LogitProcessors, TrainingSamplingParams, apply_logit_processors
from rl_amd.distributed.model_utils import (
    add_rms_norm_8bit,
    from_int8_hidden_states_to_logits,
    from_parallel_8bit_hidden_states_to_logprobs,
    from_parallel_logits_to_logprobs,
    from_residual_stream_to_logprobs,
    get_next_token_logprobs_from_logits,
    processed_next_token_logprobs,
    quantize_rows_8bit,
)

B, R, V = 2, 3, 40


@pytest.fixture(autouse=True)
def no_message_left():
    yield
    assert _C.load().mirl_dropout(None, 0, 0, 0.5, 0, None, 0, None, None) == 0  # (a call that succeeds clears it)


def logits(**kw):
    return torch.zeros(B, R, V, **kw)


def ids():
    return torch.zeros(B, R, dtype=torch.int64)


ROWS = torch.zeros(B, R, dtype=torch.int64)
MASK = torch.zeros(1, 2, dtype=torch.int32)


@pytest.mark.parametrize("settings,error", [
    (dict(repetition_penalty=0.0), ValueError),
    (dict(repetition_penalty=-1.0), ValueError),
    (dict(repetition_penalty=float("nan")), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=float("inf")), ValueError),
    (dict(presence_penalty=float("inf")), ValueError),
    (dict(frequency_penalty=torch.zeros(B + 1)), ValueError),
    (dict(frequency_penalty=torch.zeros(B, dtype=torch.int64)), ValueError),
    (dict(temperature=torch.ones(B, 1)), ValueError),
    (dict(presence_penalty=torch.zeros(B, requires_grad=True)), RuntimeError),
    (dict(prompt_lengths=torch.zeros(B + 1, dtype=torch.int64)), ValueError),
    (dict(prompt_lengths=torch.zeros(B)), TypeError),
    (dict(prompt_lengths=3), ValueError),
    (dict(bias=torch.zeros(4)), ValueError),
    (dict(bias_ids=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(bias_ids=torch.zeros(4, dtype=torch.int64), bias=torch.zeros(5)), ValueError),
    (dict(bias_ids=torch.zeros(B + 1, 4, dtype=torch.int64), bias=torch.zeros(B + 1, 4)), ValueError),
    (dict(bias_ids=torch.zeros(4), bias=torch.zeros(4)), TypeError),
    (dict(bias_ids=torch.zeros(4, dtype=torch.int64), bias=torch.zeros(4, dtype=torch.int64)), TypeError),
    (dict(bias_ids=torch.zeros(4, dtype=torch.int64), bias=torch.zeros(4, requires_grad=True)), RuntimeError),
    (dict(bias_ids=torch.zeros(2048, dtype=torch.int64), bias=torch.zeros(2048)), ValueError),
    (dict(grammar_masks=MASK), ValueError),
    (dict(grammar_rows=ROWS), ValueError),
    (dict(grammar_masks=MASK[:, :1], grammar_rows=ROWS), ValueError),
    (dict(grammar_masks=MASK.long(), grammar_rows=ROWS), ValueError),
    (dict(grammar_masks=MASK[0], grammar_rows=ROWS), ValueError),
    (dict(grammar_masks=MASK, grammar_rows=ROWS[:, :2]), ValueError),
    (dict(grammar_masks=MASK, grammar_rows=ROWS[:1]), ValueError),
    (dict(grammar_masks=MASK, grammar_rows=ROWS.float()), TypeError),
])
def test_settings(settings, error):
    with pytest.raises(error):
        apply_logit_processors(logits(), ids(), LogitProcessors(**settings))
    if "grammar_rows" not in settings or settings["grammar_rows"].shape != (B, 2):  # (two rows are enough for the logprobs)
        with pytest.raises(error):
            processed_next_token_logprobs(logits(), ids(), LogitProcessors(**settings))


def test_tensors():
    P = LogitProcessors(repetition_penalty=1.1)
    for bad, error in ((logits(dtype=torch.float64), TypeError), (logits(dtype=torch.int32), TypeError), (torch.zeros(V), ValueError),
                       (torch.zeros(B, R, 0), ValueError), (torch.zeros(B, V), ValueError), (torch.zeros(1, B, R, V), ValueError)):
        with pytest.raises(error):
            apply_logit_processors(bad, ids(), P)
    for bad, error in ((ids()[:1], ValueError), (ids()[0], ValueError), (ids().float(), TypeError), (ids()[:, :2], ValueError)):
        with pytest.raises(error):
            apply_logit_processors(logits(), bad, P)
    lengths = torch.ones(B, dtype=torch.int64)
    for bad, error in ((lengths[:1], ValueError), (lengths.float(), TypeError), (3, ValueError), (lengths[None], ValueError)):
        with pytest.raises(error):
            apply_logit_processors(logits(), ids(), P, history_lengths=bad)
        with pytest.raises(error):
            processed_next_token_logprobs(logits(), ids(), P, history_lengths=bad)
    with pytest.raises(ValueError):  # 2^20 tokens are more than a word counts
        apply_logit_processors(logits(), torch.zeros(B, 1 << 20, dtype=torch.int64), P)
    with pytest.raises(ValueError):
        apply_logit_processors(torch.zeros(1, 1, 1).expand(1, 1, (1 << 24) + 1), torch.zeros(1, 1, dtype=torch.int64), P)
    with pytest.raises(ValueError):
        processed_next_token_logprobs(torch.zeros(B, V), ids(), P)
    with pytest.raises(ValueError):  # more tokens than rows, as without processors
        from_parallel_logits_to_logprobs(logits(), torch.zeros(B, R + 1, dtype=torch.int64), 0, V, None, logit_processors=P)


def test_in_place():
    P = LogitProcessors(repetition_penalty=1.1)
    with pytest.raises(RuntimeError, match="no gradient"):
        apply_logit_processors(logits(requires_grad=True), ids(), P, inplace=True)
    with pytest.raises(ValueError, match="unit stride"):
        apply_logit_processors(torch.zeros(B, V, R).transpose(1, 2), ids(), P, inplace=True)
    with pytest.raises(ValueError, match="share memory"):
        apply_logit_processors(torch.zeros(1, R, V).expand(B, R, V), ids(), P, inplace=True)


@pytest.mark.parametrize("strides", [(V, V), (R * V, V), (V, B * V), (R * V - 1, V), (5 * V, 2 * V), (2 * V, 5 * V), (4 * V, 2 * V)])
def test_in_place_rows_that_nest(strides):
    x = torch.zeros(40 * V).as_strided((B, R, V), (*strides, 1))
    places = {i * strides[0] + j * strides[1] + v for i in range(B) for j in range(R) for v in range(V)}
    shared = len(places) < B * R * V
    with pytest.raises(ValueError if shared else _C.MirlError, match="share memory" if shared else None):
        apply_logit_processors(x, ids(), LogitProcessors(repetition_penalty=1.1), inplace=True)


def test_valid_calls_end_at_the_device():
    P = LogitProcessors(repetition_penalty=torch.full((B,), 1.1), bias_ids=torch.zeros(3, dtype=torch.int64), bias=torch.zeros(3),
                        grammar_masks=MASK, grammar_rows=ROWS)
    for call in (lambda: apply_logit_processors(logits(), ids(), P),
                 lambda: processed_next_token_logprobs(logits(), ids(), P),
                 lambda: get_next_token_logprobs_from_logits(ids(), logits(), logit_processors=P),
                 lambda: from_parallel_logits_to_logprobs(logits(), ids(), 0, V, None, logit_processors=P,
                                                          sampling_params=TrainingSamplingParams(top_k=3))):
        with pytest.raises(_C.MirlError):
            call()
    x = logits()
    assert apply_logit_processors(x, ids(), None) is x


def test_the_c_entry_points():
    lib = _C.load()
    A = _C.LogitProcessorArgs()
    A.n_ids, A.vocab_end = 5, V
    none = (None,) * 6

    def fwd(dtype=0, b=1, r=1, v=V, args=A):
        return lib.mirl_processed_logprob_fwd(None, dtype, b, r, v, v, v, ctypes.byref(args) if args is not None else None, *none[:5])

    for call, word in ((lambda: fwd(dtype=3), "dtype"), (lambda: fwd(v=0), "shape"), (lambda: fwd(b=-1), "shape"),
                       (lambda: fwd(v=(1 << 24) + 1), "vocabulary"), (lambda: fwd(args=None), "null"), (fwd, "null")):
        assert call() != 0 and word in lib.mirl_last_error().decode()
    for field, value, word in (("n_ids", 1 << 20, "tokens"), ("n_bias", 2048, "biases"), ("n_masks", 1, "masks"), ("n_bias", -1, "biases")):
        bad = _C.LogitProcessorArgs()
        bad.vocab_end = V
        setattr(bad, field, value)
        assert fwd(args=bad) != 0 and word in lib.mirl_last_error().decode()
    assert fwd(b=0) == 0 and fwd(r=0) == 0
    one = 16  # an address that is never read
    assert lib.mirl_process_logits(one, 0, 2, 1, V, V, V, ctypes.byref(_C.LogitProcessorArgs()), one, one, V + 1, V, None) != 0
    assert "in place" in lib.mirl_last_error().decode()
    assert lib.mirl_processed_logprob_bwd(None, 0, 1, 3, 2, V, V, V, ctypes.byref(_C.LogitProcessorArgs()), *none[:3], 1, 1, None, V, V, None) != 0
    # a sample's head, where the three buckets of each list begin and the last ends (tokens, 4096 a list; biases), the entries
    assert lib.mirl_logit_processors_table_elems(2, 5000, 10, 3) == 2 * (8 + 2 * (3 + 1) + 10 + 3)
    assert lib.mirl_logit_processors_table_elems(2, 5000, 0, 0) == 2 * (8 + 3 + 1)
    assert lib.mirl_logit_processors_table_elems(1, 5000, 4097, 0) == 8 + 2 * (3 + 1) + 4097


# ---------------------------------------------------------------------------
# 8-bit integers
# ---------------------------------------------------------------------------
def test_int8_operands():
    h, w = torch.zeros(4, 16, dtype=torch.int8), torch.zeros(5, 16, dtype=torch.int8)
    hs, ws = torch.ones(4), torch.ones(5)
    f8 = torch.float8_e4m3fn
    for args, error in (((h.float(), hs, w, ws), TypeError), ((h, hs, w.to(f8), ws), TypeError), ((h.to(f8), hs, w.to(f8), ws), TypeError),
                        ((h, hs, w[:, :8], ws), ValueError), ((h, hs, w[0], ws), ValueError), ((h, hs, w[:0], ws[:0]), ValueError),
                        ((h, hs[:3], w, ws), ValueError), ((h, hs, w, ws.double()), ValueError), ((h[:, :0], hs, w[:, :0], ws), ValueError)):
        with pytest.raises(error):
            from_int8_hidden_states_to_logits(*args)
    wide = torch.zeros(1, 1, dtype=torch.int8).expand(1, (1 << 17) - 255)
    with pytest.raises(ValueError, match="32 bits"):
        from_int8_hidden_states_to_logits(wide, hs[:1], wide, ws[:1])
    with pytest.raises(TypeError):
        from_int8_hidden_states_to_logits(h, hs, w, ws, torch.float64)
    for out in (torch.zeros(4, 5), torch.zeros(5, 4, dtype=torch.bfloat16).t(), torch.zeros(4, 6, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            from_int8_hidden_states_to_logits(h, hs, w, ws, torch.bfloat16, out)
    with pytest.raises(RuntimeError):
        from_int8_hidden_states_to_logits(h, hs, w, ws, torch.float32, torch.zeros(4, 5, requires_grad=True))
    with pytest.raises(_C.MirlError):
        from_int8_hidden_states_to_logits(h, hs, w, ws)
    target = torch.zeros(2, 2, dtype=torch.int64)
    with pytest.raises(TypeError):
        from_parallel_8bit_hidden_states_to_logprobs(h.view(2, 2, 16), hs.view(2, 2), w.to(f8), ws, target, 0, 5)
    with pytest.raises(_C.MirlError):
        from_parallel_8bit_hidden_states_to_logprobs(h.view(2, 2, 16), hs.view(2, 2), w, ws, target, 0, 5)


def test_int8_rows():
    for dtype in (torch.uint8, torch.float16, torch.float8_e5m2):
        with pytest.raises(TypeError):
            quantize_rows_8bit(torch.zeros(2, 4), dtype)
        with pytest.raises(TypeError):
            add_rms_norm_8bit(torch.zeros(2, 4), None, torch.ones(4), 1e-6, dtype)


def test_processors_of_the_policy_head_need_an_int8_weight():
    x, w = torch.zeros(2, 1, 16), torch.zeros(5, 16)
    target = torch.zeros(1, 2, dtype=torch.int64)
    P = LogitProcessors(temperature=0.7)
    with pytest.raises(NotImplementedError):
        from_residual_stream_to_logprobs(x, None, torch.ones(16), w, target, 0, 5, logit_processors=P)
    with pytest.raises(NotImplementedError):
        from_residual_stream_to_logprobs(x, None, torch.ones(16), (w.to(torch.float8_e4m3fn), torch.ones(5)), target, 0, 5, logit_processors=P)


def test_the_int8_c_entry_points():
    lib = _C.load()
    call = lambda T=4, H=16, ldh=256, V=5, ldw=16, dtype=0, ldo=5: lib.mirl_int8_logits(  # noqa: E731
        None, None, T, H, ldh, None, None, V, ldw, None, dtype, ldo, None)
    for kw, word in ((dict(dtype=7), "dtype"), (dict(H=0), "shape"), (dict(V=0), "shape"), (dict(H=1 << 17, ldh=1 << 17, ldw=1 << 17), "32 bits"),
                     (dict(ldh=16), "multiples"), (dict(H=18, ldw=20), "multiples"), (dict(ldh=1 << 22), "strides"), ({}, "null")):
        assert call(**kw) != 0 and word in lib.mirl_last_error().decode(), kw
    assert call(T=0) == 0
    assert lib.mirl_linear_ce_int8_fwd(None, None, 4, 16, 256, None, None, 5, 16, 3, None, 1, 1, 0, 5, None, 1, 1, None, None) != 0
    assert "multiple of the batch" in lib.mirl_last_error().decode()
    assert lib.mirl_add_rms_norm_int8_fwd(None, 0, 8, None, 0, 0, None, 0, 2, 8, 1e-6, None, None, None, None) != 0
    assert lib.mirl_quantize_rows_int8(None, 9, 8, 2, 8, None, None, None) != 0
