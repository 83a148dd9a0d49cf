"""Infinities and NaN in attention's inputs reach the rows that see them, and what the gradient of those rows reaches, and nothing else: every
other row and key has the results of a call without them, within the bounds of those."""
import importlib
import math

import pytest
import torch

import head_reference as ref
from row_reference import close
from test_gpu_attention import BF16, F16, Call

pytestmark = pytest.mark.gpu
NAN, INF = math.nan, math.inf


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


CALLS = {  # lengths, heads, key heads, elements, room
    "short": ([(40, 40), (50, 50)], 2, 2, 64, None),
    "groups": ([(70, 70), (33, 33)], 6, 2, 40, None),
    "long": ([(300, 300), (131, 131)], 4, 1, 128, None),
    "tokens": ([(1, 100), (3, 90)], 4, 2, 128, 128),
    "few": ([(5, 500), (7, 300)], 2, 2, 64, 512),
    "pieces": ([(6, 4000)], 4, 4, 128, 4096),
    "many pieces": ([(200, 3001)], 2, 1, 64, 3001),
}
LONG = {  # rows in pieces, for the gradient alone
    "rows in pieces": ([(1200, 1200)], 2, 1, 64, None),
    "wide rows in pieces": ([(700, 900), (40, 60)], 3, 1, 128, 900),
}


def made(name, dtype, seed=0):
    lengths, heads, key_heads, d, room = {**CALLS, **LONG}[name]
    return Call(lengths, heads, key_heads, d, dtype, 21 + seed, room=room)


def check_rows(call, out, lse, some):
    """Rows `some` (truth values) against the definition, without the keys that they don't see."""
    for rows, keys in call.parts():
        n, m = rows.stop - rows.start, keys.stop - keys.start
        for i in range(n):
            if some[rows.start + i]:
                seen = slice(keys.start, keys.start + m - n + i + 1)
                for h in range(call.heads):
                    kh, at = h // (call.heads // call.key_heads), rows.start + i
                    want = ref.attention(call.q[at:at + 1, h].double(), call.k[seen, kh].double(), call.v[seen, kh].double(), call.scale, True, call.dtype)
                    close(out[at:at + 1, h], want[0], want[2], "row %d, head %d" % (at, h))
                    if want[1][0] > -INF:
                        close(lse[h, at:at + 1], want[1], want[3], "lse of row %d, head %d" % (at, h))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_hidden_values(api, name, value, dtype):
    """A value in the keys or values that some of the rows in its tile do not see."""
    call = made(name, dtype)
    clean, clean_lse = call.run(api)
    keep_k, keep_v = call.k.clone(), call.v.clone()
    for into in "vk":
        call.k, call.v = keep_k.clone(), keep_v.clone()
        meets = torch.zeros(call.rows, dtype=torch.bool, device="cuda")
        for (rows, keys), (n, _) in zip(call.parts(), call.lengths):
            last = min(n, 1 + n // 3)              # the key that the last rows see: these
            getattr(call, into)[keys.stop - last, :, 3] = value
            meets[rows.stop - last:rows.stop] = True
        out, lse = call.run(api)
        if into == "v":
            assert (out[meets][..., 3].isnan() if math.isnan(value) else out[meets][..., 3] == value).all()
            others = torch.arange(call.d, device="cuda") != 3
            assert out[meets][..., others].isfinite().all() and lse.isfinite().all()
        elif math.isnan(value):
            assert out[meets].isnan().all() and lse[:, meets].isnan().all()
        assert out[~meets].isfinite().all() and lse[:, ~meets].isfinite().all()
        check_rows(call, out, lse, ~meets)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", ["short", "groups", "long"])
def test_values_from_a_key_on(api, name, dtype):
    """All values from one key on are NaN: the row before is the last one without."""
    call = made(name, dtype, 1)
    keep = call.v.clone()
    for rows, keys in call.parts():
        for at in (keys.start + 1, keys.start + 2, keys.start + 31, keys.stop - 1):
            call.v = keep.clone()
            call.v[at:keys.stop] = NAN
            out, lse = call.run(api)
            meets = torch.zeros(call.rows, dtype=torch.bool, device="cuda")
            meets[at:rows.stop] = True
            assert out[meets].isnan().all() and out[~meets].isfinite().all() and lse.isfinite().all()
            some = torch.zeros_like(meets)
            some[max(rows.start, at - 4):at] = True
            check_rows(call, out, lse, some)


def gradients(call, out, lse):
    """(values, errors) of the gradients of q, k and v in 64 bits."""
    size = max(float(t[keep].double().norm(dim=-1).max()) for t, keep in ((call.grad, call.kept_grad), (call.v, call.kept_v)))
    bound = size * size
    want = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (call.q, call.k, call.v)]
    errors = [torch.zeros_like(t) for t in want]
    for rows, keys in call.parts():
        for h in range(call.heads):
            kh = h // (call.heads // call.key_heads)
            values, off = ref.attention_grad(call.grad[rows, h].double(), call.q[rows, h].double(), call.k[keys, kh].double(), call.v[keys, kh].double(),
                                             out[rows, h].double(), lse[h, rows].double(), call.scale, True, call.dtype, bound)
            for i, at in enumerate(((rows, h), (keys, kh), (keys, kh))):
                want[i][at] += values[i]
                errors[i][at] += off[i]
    return want, errors


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", list(CALLS) + list(LONG))
@pytest.mark.parametrize("into", ["q", "k", "v", "grad"])
def test_gradients_beside_what_is_not_finite(api, name, into, dtype):
    """With one row, or one key, of each sequence not finite in one input."""
    call = made(name, dtype, 2)
    out, lse = call.check(api)
    want, errors = gradients(call, out, lse)
    keep = getattr(call, into)
    for value in (NAN, INF):
        setattr(call, into, keep.clone())
        rows_met = torch.zeros(call.rows, dtype=torch.bool, device="cuda")
        keys_met, values_met = (torch.zeros(call.keys, dtype=torch.bool, device="cuda") for _ in range(2))
        for rows, keys in call.parts():
            n, m = rows.stop - rows.start, keys.stop - keys.start
            if into in "kv":
                back = min(n, 1 + n // 3)          # as many rows, the last ones, see the key
                at = keys.stop - back
                rows_met[rows.stop - back:rows.stop] = True
                keys_met[at] = True
                values_met[at] = into == "k"
            else:
                row = n // 2                        # it sees the keys up to this one
                at, last = rows.start + row, keys.start + m - n + row
                rows_met[at] = True
                keys_met[keys.start:last + 1] = values_met[keys.start:last + 1] = True
            getattr(call, into)[at] = value
        got = call.gradients(api, out, lse)
        setattr(call, into, keep)
        for what, a, b, e, kept, met in zip(("gradient of q", "of k", "of v"), got, want, errors, (call.kept_q, call.kept_k, call.kept_k),
                                            (rows_met, keys_met, values_met)):
            fine = kept & ~met
            close(a[fine], b[fine], e[fine], what)
            assert (a[~kept] == 7).all()
            if math.isnan(value):
                assert a[met].isnan().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("into", ["out", "lse"])
def test_gradients_of_results_that_are_not_finite(api, name, into, dtype):
    """A row's result, or its lse, is NaN: its gradient, and those of the keys that it sees, and no others."""
    call = made(name, dtype, 3)
    out, lse = call.check(api)
    want, errors = gradients(call, out, lse)
    rows_met = torch.zeros(call.rows, dtype=torch.bool, device="cuda")
    keys_met = torch.zeros(call.keys, dtype=torch.bool, device="cuda")
    for rows, keys in call.parts():
        n, m = rows.stop - rows.start, keys.stop - keys.start
        row = n // 2
        rows_met[rows.start + row] = True
        keys_met[keys.start:keys.start + m - n + row + 1] = True
    if into == "out":
        out = torch.where(rows_met[:, None, None], torch.full_like(out, NAN), out)
    else:
        lse = torch.where(rows_met, torch.full_like(lse, NAN), lse)
    values_met = keys_met if into == "lse" else torch.zeros_like(keys_met)
    got = call.gradients(api, out, lse)
    for what, a, b, e, kept, met in zip(("gradient of q", "of k", "of v"), got, want, errors, (call.kept_q, call.kept_k, call.kept_k),
                                        (rows_met, keys_met, values_met)):
        fine = kept & ~met
        close(a[fine], b[fine], e[fine], what)
        assert a[met].isnan().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_other_sequences_to_the_last_bit(api, causal, dtype):
    call = Call([(40, 40), (50, 50), (60, 60)], 4, 2, 64, dtype, 41, causal)
    clean, clean_lse = call.run(api)
    grads = call.gradients(api, clean, clean_lse)
    call.k[45], call.v[60], call.grad[50], call.q[70] = NAN, INF, NAN, -INF
    out, lse = call.run(api)
    got = call.gradients(api, out, lse)
    for rows in (slice(0, 40), slice(90, 150)):
        assert torch.equal(out[rows], clean[rows]) and torch.equal(lse[:, rows], clean_lse[:, rows])
        assert all(torch.equal(a[rows], b[rows]) for a, b in zip(got, grads))
