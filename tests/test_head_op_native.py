"""How the calls of rotary positions, attention and log probabilities are taken by the Python interface's native code, on the CPU: tensors wrap a made-up
address, and every call that reaches an operator is refused by it before any launch. What is of another type than the native code takes, or missing
where it must not be, is handed on to the Python call, which says so."""
import importlib

import numpy as np
import pytest

from test_row_op_validation import BF16, F32, INVALID_ARGUMENT, fake

S32, S64 = np.int32, np.int64


@pytest.fixture
def api(cv, monkeypatch):
    api = importlib.import_module("cvcuda_amd.pyapi")
    # the current device, and its default stream
    monkeypatch.setattr(api.torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(api.torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    monkeypatch.setattr(api, "_followed", {})
    return api


def tensors(cv, api):
    return lambda *args, **kw: api.Tensor(_wrap=fake(cv, *args, **kw))


def operators(cv, api):
    """(name, operator, arguments that only the operator refuses, which of them may be None, where another type of number is)."""
    t = tensors(cv, api)
    heads, keys = t([6, 4, 16], BF16), t([6, 2, 16], BF16)
    offsets, lengths, lse, one = t([3], S32), t([2], S32), t([4, 6]), t([1], np.uint8)
    logits, tokens, row, values, words = t([6, 50]), t([6], S64), t([6]), t([6, 5]), t([6, 5], S32)
    few = t([5])
    # (each with something that no optional argument changes: a position too many, results of other heads, a small workspace, a row too few)
    return [
        ("rotary", cv.Rotary(), [heads, t([7], S64), heads, 16, 1e4, 1.0, 0.0, 1.0, 4.0, 1.0, False, True], (), {3: 1 << 40, 4: 10000, 9: None, 10: 0, 11: 1}),
        ("attention", cv.Attention(), [heads, keys, keys, offsets, offsets, lengths, keys, lse, one, 0.25, True], (4, 5, 7, 8), {9: 1, 10: 1}),
        ("attention's gradient", cv.AttentionGrad(), [heads, heads, keys, keys, heads, lse, offsets, offsets, lengths, heads, keys, keys, one, 0.25, False],
         (7, 8, 12), {13: None, 14: None}),
        ("log probabilities", cv.LogProbs(), [logits, tokens, few, row, row, values, words, 1.0], (3, 4, 5, 6), {7: 1}),
        ("their gradient", cv.LogProbsGrad(), [logits, tokens, few, row, row, row, logits, 1.0], (3, 5), {7: True}),
    ]


def calls(cv, api, monkeypatch, op, args):
    """(status of the refusal, whether the call was handed on)"""
    handed = []

    def submit(*a):
        handed.append(a)
        raise LookupError

    monkeypatch.setattr(api, "_submit", submit)
    try:
        api._run(None, [], [], op, *args)
    except LookupError:
        assert len(handed) == 1 and list(handed[0][4:]) == list(args)
        return None, True
    except api.Error as e:
        assert not handed and str(e)
        return e.status, False
    raise AssertionError("neither refused nor handed on")


def test_what_the_native_code_takes_is_refused_by_the_operators(cv, api, monkeypatch):
    for name, op, args, optional, _ in operators(cv, api):
        assert calls(cv, api, monkeypatch, op, args) == (INVALID_ARGUMENT, False), name
        for place in optional:
            assert calls(cv, api, monkeypatch, op, args[:place] + [None] + args[place + 1:]) == (INVALID_ARGUMENT, False), (name, place)


def test_what_it_does_not_take_is_handed_on(cv, api, monkeypatch):
    for name, op, args, optional, others in operators(cv, api):
        for place, value in enumerate(args):
            if isinstance(value, api.Tensor):
                for other in ([] if place in optional else [None]) + [1, "tensor", value._t]:
                    assert calls(cv, api, monkeypatch, op, args[:place] + [other] + args[place + 1:]) == (None, True), (name, place, other)
        for place, other in others.items():
            assert calls(cv, api, monkeypatch, op, args[:place] + [other] + args[place + 1:]) == (None, True), (name, place, other)
        assert calls(cv, api, monkeypatch, op, args[:-1]) == (None, True), name
        assert calls(cv, api, monkeypatch, op, args + [True]) == (None, True), name


def test_what_is_handed_on_is_refused_in_python(cv, api):
    """The whole way, with the call's own _submit."""
    t = tensors(cv, api)
    heads, keys, offsets, logits, tokens, row = t([6, 4, 16], BF16), t([6, 2, 16], BF16), t([3], S32), t([6, 50]), t([6], S64), t([6])
    room = t([cv.AttentionGrad.workspace(6, 6, 2, 4, 2, 16)], np.uint8)
    refusals = [
        lambda: api.rotary_into(heads, heads, None),
        lambda: api.attention_into(heads, heads, keys, None, offsets),
        lambda: api.attention_into(None, heads, keys, keys, offsets),
        lambda: api.attention_grad_into(heads, keys, None, heads, heads, keys, keys, heads, t([4, 6]), offsets, workspace=room),
        lambda: api.attention_grad_into(heads, keys, keys, heads, heads, keys, keys, heads, None, offsets, workspace=room),
        lambda: api.log_probs_into(row, logits, None),
        lambda: api.log_probs_into(row, logits, tokens, top_values=t([6, 5])),
        lambda: api.log_probs_grad_into(logits, logits, tokens, None, row),
        lambda: api.log_probs_grad_into(logits, logits, tokens, row, row, grad_entropy=row),
    ]
    for call in refusals:
        with pytest.raises(api.Error) as e:
            call()
        assert e.value.status == INVALID_ARGUMENT and str(e.value)
