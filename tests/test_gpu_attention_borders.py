"""Attention at the borders of what its header allows: offsets that go back."""
import importlib

import pytest
import torch

from test_gpu_attention import BF16, F16, Call, numbers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [20, 90])  # (few to a sequence, and many)
@pytest.mark.parametrize("back", [lambda n: [0, n // 3, n // 4], lambda n: [n // 2, n // 9, n], lambda n: [n // 3, n, n // 2, n // 4],
                                  lambda n: [n // 2, n // 4, n // 3, 0, n // 8]],
                         ids=["last", "first", "two", "between"])
def test_pieces_of_sequences_whose_offsets_go_back(api, cv, back, rows, dtype):
    """A sequence whose end lies before its begin has no rows; the others' are the same as where it has its end at its begin, whether their
    keys are in one piece or in several."""
    offsets = back(rows)
    sequences = len(offsets) - 1
    call = Call([(rows, rows)] + [(0, 0)] * (sequences - 1), 4, 4, 64, dtype, rows, room=2100)
    call.k, call.v = (torch.where(t.isnan(), torch.ones_like(t), t) for t in (call.k, call.v))
    call.key_lengths = numbers([1100 + 300 * b for b in range(sequences)])
    assert cv.Attention.workspace(rows, call.keys, sequences, 4, 4, 64) > 0
    want, stats = torch.full(call.q.shape, 7.0, dtype=dtype, device="cuda"), torch.full((4, rows), 7.0, device="cuda")
    for b in range(sequences):
        if offsets[b] < offsets[b + 1]:
            call.offsets = numbers([offsets[b]] * (b + 1) + [offsets[b + 1]] * (sequences - b))
            alone, lse = call.run(api)
            at = slice(offsets[b], offsets[b + 1])
            want[at], stats[:, at] = alone[at], lse[:, at]
            assert (alone[at] != 7).any(-1).all() and (lse[:, at] != 7).all()
    call.offsets = numbers(offsets)
    out, lse = call.run(api)
    assert torch.equal(out, want) and torch.equal(lse, stats)


def test_small_gradients_beside_large_ones_in_f16(api):
    """A row's gradient of q, and that of keys which only rows of small gradients see, depend on no other row: bit for bit the same where those beside
    them have gradients larger by 2^28."""
    for d, heads, key_heads in ((64, 2, 2), (128, 4, 2)):
        call = Call([(150, 150)], heads, key_heads, d, F16, d)
        call.grad = (call.grad.float() * 2.0 ** -16).half()
        out, lse = call.run(api)
        small = call.gradients(api, out, lse)
        last, alone = slice(140, 150), slice(40, 43)
        large = call.grad.float() * 2.0 ** 28
        large[last], large[alone] = call.grad[last].float(), call.grad[alone].float()
        call.grad = large.half()
        assert call.grad.isfinite().all() and call.grad.abs().max() > 2.0 ** 13
        got = call.gradients(api, out, lse)
        for rows in (last, alone):
            assert torch.equal(got[0][rows], small[0][rows]) and (got[0][rows] != 0).any()
        for a, b in zip(got[1:], small[1:]):
            assert torch.equal(a[last], b[last]) and (a[last] != 0).any()


@pytest.mark.parametrize("rows", [1, 40])
def test_large_values_behind_growing_scores(api, rows):
    """Values of 1e37 at a key whose score lies above those of the keys before it, by less than makes the sums' reference follow."""
    for d in (64, 128):
        call = Call([(rows, 200)], 2, 2, d, BF16, 31, causal=False, room=200, scale=1.0)
        call.q.zero_(), call.k.zero_()
        call.q[..., 0] = 1
        call.k[:, :, 0] = torch.arange(200, device="cuda").div(50, rounding_mode="floor").mul(1.7).to(BF16)[:, None]
        for key in (49, 99, 120, 199):
            v = call.v.clone()
            call.v[key] = 1e37
            assert call.check(api)[0].abs().max() > 5e32  # (shares are e^-5.1 / 62 = 1e-4 at least)
            call.v = v
