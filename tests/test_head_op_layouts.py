"""The orders of tokens and heads that tensors of rotary positions and attention can have: a token lies behind all heads of the one before, which the
kernels rest on. (The CPU: addresses are made up.)"""
import pytest

from test_row_op_validation import BF16, INVALID_ARGUMENT, fake


@pytest.mark.parametrize("layout", ["", "TWE"])
@pytest.mark.parametrize("strides", [[16, 96, 1], [0, 16, 1], [16, 16, 1], [48, 16, 1], [64, 0, 1], [-64, 16, 1]])
def test_heads_before_tokens_are_refused(cv, strides, layout):
    with pytest.raises(cv.Error) as e:
        fake(cv, [6, 4, 16], BF16, layout, strides=strides)
    assert e.value.status == INVALID_ARGUMENT


def test_gaps_between_heads_and_tokens_are_taken(cv):
    for strides in ([64, 16, 1], [80, 16, 1], [96, 24, 1], [128, 32, 1]):
        assert fake(cv, [6, 4, 16], BF16, "TWE", strides=strides).strides == [2 * s for s in strides]


@pytest.mark.parametrize("tokens,heads,strides", [(1, 4, [16, 16, 1]), (1, 4, [0, 24, 1]), (6, 1, [16, 0, 1]), (6, 1, [40, 640, 1])])
def test_single_tokens_and_heads_have_no_order(cv, tokens, heads, strides):
    """Strides of dimensions of one element say nothing; they are taken, and not used."""
    fake(cv, [tokens, heads, 16], BF16, "TWE", strides=strides)
