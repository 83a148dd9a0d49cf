"""What rotary positions, attention and log probabilities (cvcuda/Rotary.h, Attention.h, LogProbs.h) refuse, on the CPU: tensors wrap a
made-up device address, every case is rejected on the host before any launch."""
import importlib

import numpy as np
import pytest

from test_row_op_validation import BF16, F16, F32, FAKE, INVALID_ARGUMENT, NOT_COMPATIBLE, fake, refused

S32, S64, NAN, INF = np.int32, np.int64, float("nan"), float("inf")


def test_rotary_refusals(cv):
    op = cv.Rotary()
    x, y, at = fake(cv, [6, 4, 10]), fake(cv, [6, 4, 10]), fake(cv, [6], S64)
    refused(cv, op, 0, None, at, y, 10)
    refused(cv, op, 0, x, None, y, 10)
    refused(cv, op, 0, x, at, None, 10)
    refused(cv, op, 0, fake(cv, [24, 10]), at, fake(cv, [24, 10]), 10)             # dimensions
    refused(cv, op, 0, fake(cv, [6, 4, 10], np.float64), at, fake(cv, [6, 4, 10], np.float64), 10)
    refused(cv, op, 0, x, at, fake(cv, [6, 4, 10], F16), 10)                         # type
    refused(cv, op, 0, x, at, fake(cv, [6, 4, 12]), 10)
    refused(cv, op, 0, x, at, fake(cv, [6, 5, 10]), 10)
    refused(cv, op, 0, x, fake(cv, [6], F32), y, 10)
    refused(cv, op, 0, x, fake(cv, [7], S64), y, 10)
    refused(cv, op, 0, x, fake(cv, [2, 3], S64, "NW", strides=[4, 1]), y, 10)          # positions with gaps
    refused(cv, op, 0, fake(cv, [6, 4, 10], at=FAKE + 2), at, y, 10)                 # between elements
    for dims in (0, -2, 3, 12, 1 << 30):
        refused(cv, op, 0, x, at, y, dims)
    refused(cv, op, 0, fake(cv, [6, 4, 600]), at, fake(cv, [6, 4, 600]), 258)
    for name in ("base", "factor", "magnitude"):
        for value in (0.0, -1.0, NAN, INF):
            refused(cv, op, 0, x, at, y, 10, **{name: value})
    refused(cv, op, 0, x, at, y, 10, magnitude=1e39)
    for scaling in ((-1.0, 1.0, 4.0), (NAN, 1.0, 4.0), (8192.0, 4.0, 4.0), (8192.0, -1.0, 4.0), (8192.0, 1.0, NAN), (8192.0, 1.0, INF)):
        refused(cv, op, 0, x, at, y, 10, original=scaling[0], low=scaling[1], high=scaling[2])
    assert cv._cv.cvcudaxRotaryCreate(None) == INVALID_ARGUMENT
    cv.last_error()
    refused(cv, lambda: cv.check(cv._cv.cvcudaxRotarySubmit(op.handle, 0, x.handle, at.handle, y.handle, None)))
    args = cv.capi.RotaryArgs(10000.0, 1.0, 0.0, 0.0, 0.0, 1.0, 10, 0, 0)
    refused(cv, lambda: cv.check(cv._cv.cvcudaxRotarySubmit(cv.Reformat().handle, 0, x.handle, at.handle, y.handle, args)), status=NOT_COMPATIBLE)


def attention_parts(cv, dtype=BF16, rows=6, keys=6, heads=4, key_heads=2, d=16, sequences=2):
    made = dict(q=fake(cv, [rows, heads, d], dtype), k=fake(cv, [keys, key_heads, d], dtype), v=fake(cv, [keys, key_heads, d], dtype),
                offsets=fake(cv, [sequences + 1], S32), key_offsets=None, key_lengths=None, out=fake(cv, [rows, heads, d], dtype),
                lse=fake(cv, [heads, rows]), workspace=None, scale=0.25)
    return made


@pytest.mark.parametrize("gradient", [False, True])
def test_attention_refusals(cv, gradient):
    op = cv.AttentionGrad() if gradient else cv.Attention()
    good = attention_parts(cv)
    if gradient:
        room = cv.AttentionGrad.workspace(6, 6, 2, 4, 2, 16)
        good.update(grad=good["out"], grad_q=good["out"], grad_k=good["k"], grad_v=good["v"], workspace=fake(cv, [room], np.uint8))

    def no(**change):
        refused(cv, op, 0, **dict(good, **change))

    for name in ("q", "k", "v", "offsets", "out") + (("grad", "lse", "grad_q", "grad_k", "grad_v", "workspace") if gradient else ()):
        no(**{name: None})
    no(q=fake(cv, [24, 16], BF16))
    no(q=fake(cv, [6, 4, 16], F16))
    no(q=fake(cv, [6, 5, 16], BF16), out=fake(cv, [6, 5, 16], BF16), lse=fake(cv, [5, 6]))        # heads in no groups
    no(q=fake(cv, [6, 1, 16], BF16), out=fake(cv, [6, 1, 16], BF16), lse=fake(cv, [1, 6]))
    no(v=fake(cv, [7, 2, 16], BF16))
    no(v=fake(cv, [6, 1, 16], BF16))
    no(out=fake(cv, [6, 4, 24], BF16))
    no(k=fake(cv, [6, 2, 24], BF16), v=fake(cv, [6, 2, 24], BF16))
    no(offsets=fake(cv, [3], S64))
    no(offsets=fake(cv, [2, 2], S32, "NW", strides=[4, 1]))
    no(key_offsets=fake(cv, [2], S32))
    no(key_offsets=fake(cv, [3], S64))
    no(key_lengths=fake(cv, [2], S32))                                                      # without key offsets
    no(key_offsets=fake(cv, [3], S32), key_lengths=fake(cv, [3], S32))
    no(lse=fake(cv, [6, 3]))
    no(lse=fake(cv, [4, 6], F16))
    for scale in (0.0, -1.0, NAN, INF):
        no(scale=scale)
    # addresses and distances of whole 16 bytes
    no(q=fake(cv, [6, 4, 16], BF16, at=FAKE + 8))
    no(k=fake(cv, [6, 2, 16], BF16, "TWE", strides=[36, 16, 1]))
    no(v=fake(cv, [6, 2, 16], BF16, "TWE", strides=[60, 20, 1]))
    no(out=fake(cv, [6, 4, 16], BF16, "TWE", strides=[68, 16, 1]))
    if gradient:
        no(grad_v=fake(cv, [6, 2, 16], BF16, at=FAKE + 2))
        no(workspace=fake(cv, [room - 1], np.uint8))
        no(workspace=fake(cv, [room], np.uint8, at=FAKE + 8))
        no(grad=fake(cv, [6, 4, 16], F16))
        no(grad_k=fake(cv, [6, 4, 16], BF16))
    for d in (4, 12, 136, 256):
        parts = attention_parts(cv, d=d)
        refused(cv, op, 0, **dict(good, **{k: parts[k] for k in ("q", "k", "v", "out")}))
    parts = attention_parts(cv, dtype=F32)
    refused(cv, op, 0, **dict(good, **{k: parts[k] for k in ("q", "k", "v", "out")}))


def test_attention_of_few_rows_needs_a_workspace(cv):
    need = cv.Attention.workspace(1, 5000, 1, 4, 2, 16)
    assert need > 0 and need % 4 == 0
    parts = attention_parts(cv, rows=1, keys=5000, sequences=1)
    op = cv.Attention()
    refused(cv, op, 0, **parts)
    refused(cv, op, 0, **dict(parts, workspace=fake(cv, [need - 1], np.uint8)))
    refused(cv, op, 0, **dict(parts, workspace=fake(cv, [need], F32)))
    refused(cv, op, 0, **dict(parts, workspace=fake(cv, [need], np.uint8, at=FAKE + 4)))


@pytest.mark.parametrize("name", ["Attention", "AttentionGrad"])
def test_workspace_refusals(cv, name):
    workspace = getattr(cv, name).workspace
    for sizes in ((-1, 1, 1, 4, 2, 16), (1, -1, 1, 4, 2, 16), (1, 1, -1, 4, 2, 16), (1, 1, 1, 0, 1, 16), (1, 1, 1, 4, 3, 16), (1, 1, 1, 4, 0, 16),
                  (1, 1, 1, 4, 2, 0), (1, 1, 1, 4, 2, 20), (1, 1, 1, 4, 2, 136), (1 << 30, 1, 1, 4, 2, 16), (1, 1 << 31, 1, 4, 2, 16)):
        refused(cv, workspace, *sizes)
    assert workspace(0, 0, 0, 4, 2, 16) >= 0
    # of no more than the sizes need, whatever they are
    for rows in (1, 7, 100, 100000):
        for keys in (1, 1000, 1000000):
            for sequences in (1, 3, 1000):
                need = cv.Attention.workspace(rows, keys, sequences, 32, 8, 128)
                assert need % (rows * 32 * 129 * 4) == 0 and need // (rows * 32 * 129 * 4) in [0] + list(range(2, 65))


def test_log_probs_refusals(cv):
    op = cv.LogProbs()
    x, tokens, out = fake(cv, [6, 50]), fake(cv, [6], S64), fake(cv, [6])
    values, words = fake(cv, [6, 5]), fake(cv, [6, 5], S32)
    refused(cv, op, 0, None, tokens, out)
    refused(cv, op, 0, x, None, out)
    refused(cv, op, 0, x, tokens, None)
    refused(cv, op, 0, fake(cv, [6, 50], np.float64), tokens, out)
    refused(cv, op, 0, x, fake(cv, [6], F32), out)
    refused(cv, op, 0, x, fake(cv, [5], S64), out)
    refused(cv, op, 0, x, tokens, fake(cv, [7]))
    refused(cv, op, 0, x, tokens, fake(cv, [6], F16))
    refused(cv, op, 0, x, tokens, out, fake(cv, [5]))
    refused(cv, op, 0, x, tokens, out, None, fake(cv, [6], F16))
    refused(cv, op, 0, x, tokens, out, None, None, values, None)
    refused(cv, op, 0, x, tokens, out, None, None, None, words)
    refused(cv, op, 0, x, tokens, out, None, None, fake(cv, [6, 4]), words)
    refused(cv, op, 0, x, tokens, out, None, None, values, fake(cv, [6, 5], S64))
    refused(cv, op, 0, x, tokens, out, None, None, fake(cv, [6, 33]), fake(cv, [6, 33], S32))
    refused(cv, op, 0, x, tokens, out, None, None, fake(cv, [4]), fake(cv, [4], S32))
    refused(cv, op, 0, fake(cv, [6, 4]), tokens, out, None, None, values, words)     # more than there are logits
    for scale in (0.0, -1.0, NAN, INF):
        refused(cv, op, 0, x, tokens, out, scale=scale)
    refused(cv, op, 0, fake(cv, [3, 4, 5, 50], layout="ABDW", strides=[10000, 1100, 60, 1]), fake(cv, [60], S64), fake(cv, [60]))
    assert cv._cv.cvcudaxLogProbsCreate(None) == INVALID_ARGUMENT
    cv.last_error()


def test_log_probs_gradient_refusals(cv):
    op = cv.LogProbsGrad()
    x, dx, tokens, s = fake(cv, [6, 50]), fake(cv, [6, 50]), fake(cv, [6], S64), fake(cv, [6])
    refused(cv, op, 0, None, tokens, s, None, s, None, dx)
    refused(cv, op, 0, x, None, s, None, s, None, dx)
    refused(cv, op, 0, x, tokens, None, None, s, None, dx)
    refused(cv, op, 0, x, tokens, s, None, None, None, dx)
    refused(cv, op, 0, x, tokens, s, None, s, None, None)
    refused(cv, op, 0, x, tokens, s, None, s, s, dx)                                   # its entropy is missing
    refused(cv, op, 0, x, tokens, fake(cv, [5]), None, s, None, dx)
    refused(cv, op, 0, x, tokens, s, None, fake(cv, [6], F16), None, dx)
    refused(cv, op, 0, x, tokens, s, None, s, None, fake(cv, [6, 50], F16))
    refused(cv, op, 0, x, tokens, s, None, s, None, fake(cv, [6, 51]))
    refused(cv, op, 0, x, fake(cv, [6], np.uint8), s, None, s, None, dx)
    refused(cv, op, 0, x, tokens, s, None, s, None, dx, scale=0.0)


def test_native_calls_are_handed_on(cv):
    """Arguments that the native part does not take are the Python call's to refuse."""
    api = importlib.import_module("cvcuda_amd.pyapi")
    q = api.Tensor.__new__(api.Tensor)
    with pytest.raises((api.Error, TypeError, ValueError, AttributeError)):
        api.attention(q, q, q, q)
    with pytest.raises((api.Error, TypeError, ValueError, AttributeError)):
        api.rotary(None, None)
    with pytest.raises((api.Error, TypeError, ValueError, AttributeError)):
        api.log_probs(None, None)


@pytest.mark.parametrize("gradient", [False, True])
def test_attention_refuses_what_its_addresses_do_not_reach(cv, gradient):
    op = cv.AttentionGrad() if gradient else cv.Attention()
    good = attention_parts(cv)
    if gradient:
        room = cv.AttentionGrad.workspace(6, 6, 2, 4, 2, 16)
        good.update(grad=good["out"], grad_q=good["out"], grad_k=good["k"], grad_v=good["v"], workspace=fake(cv, [room], np.uint8))

    def no(**change):
        refused(cv, op, 0, **dict(good, **change))

    far = (1 << 23) + 8                                                        # elements: 2^24 bytes and 16
    no(k=fake(cv, [6, 2, 16], BF16, "TWE", strides=[far, 16, 1]))
    no(v=fake(cv, [6, 2, 16], BF16, "TWE", strides=[far, 16, 1]))
    no(out=fake(cv, [6, 4, 16], BF16, "TWE", strides=[far, 16, 1]))
    # a single token, whose heads alone lie too far from one another
    one = attention_parts(cv, rows=1, keys=1, sequences=1)
    refused(cv, cv.Attention(), 0, **dict(one, q=fake(cv, [1, 4, 16], BF16, "TWE", strides=[4 * ((1 << 21) + 8), (1 << 21) + 8, 1])))
    no(scale=2e30)


@pytest.mark.parametrize("name", ["Attention", "AttentionGrad"])
def test_sizes_that_kernels_cannot_count(cv, name):
    workspace = getattr(cv, name).workspace
    for sizes in ((1 << 27, 1, 1, 4, 2, 16), (1, 1 << 28, 1, 4, 2, 16), (1, 1, 1 << 20, 4, 2, 16), (1 << 62, 1, 1, 4, 2, 16), (1, 1 << 62, 1, 4, 2, 16),
                  (1, 1, 1 << 62, 4, 2, 16)):
        refused(cv, workspace, *sizes)
    assert workspace((1 << 27) - 1, (1 << 28) - 1, (1 << 20) - 1, 4, 2, 16) >= 0
