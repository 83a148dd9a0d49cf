"""The gradients' long sums, exactly: where every term is a whole number and no sum of them reaches 2^24, 32 bits hold each
partial sum as it is, in whatever order, and one term lost or added twice is seen. (The bounds of row_reference.py grow with the number
of terms; over tens of thousands of them a term is less than the bound.)"""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MOST = 1 << 24


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})  # (a wait for the default stream has the calls after it record events)


def whole(shape, most, dtype, seed):
    """Whole numbers from 1 on (none may be lost unseen), which `dtype` holds."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(1, min(most, 200) + 1, shape, generator=g, device="cuda", dtype=torch.int16).to(dtype)


# ---- embedding ---------------------------------------------------------------------------------------------------------
# tokens * columns on both sides of 2^24, where the pieces that are summed change from 8 tokens to 32; rows narrower than a lane's run
SIZES = [(65, 130), (2047, 130), (30000, 130), (70001, 3), (100003, 515), (60000, 1031), (2600000, 7)]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("in_type", [F32, F16, BF16])
@pytest.mark.parametrize("n,d", SIZES)
def test_one_token_over_all_pieces(api, n, d, in_type, accumulate):
    dy, wrap = whole((n, d), (MOST - 1) // (n + 1), in_type, n), api.as_tensor
    out = whole((3, d), (MOST - 1) // (n + 1), F32, 5)
    want = dy.sum(0, dtype=torch.float64)
    want = torch.stack([out[0].double(), out[1].double() + want, out[2].double()]) if accumulate else torch.stack([want * 0, want, want * 0])
    api.embedding_grad_into(wrap(out), wrap(dy), wrap(torch.ones(n, dtype=torch.int64, device="cuda")), accumulate=accumulate)
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("in_type", [F32, F16, BF16])
@pytest.mark.parametrize("n,d", SIZES)
def test_runs_of_all_lengths(api, n, d, in_type, accumulate):
    """Frequent tokens and rare ones: runs of equal tokens from one to a large part of all begin and end anywhere in a piece."""
    v, g = 1500, torch.Generator(device="cuda").manual_seed(n)
    tokens = (v ** torch.rand((n,), generator=g, device="cuda", dtype=torch.float64)).long() - 1
    dy, out, wrap = whole((n, d), (MOST - 1) // (n + 1), in_type, n), whole((v, d), (MOST - 1) // (n + 1), F32, 5), api.as_tensor
    before = torch.cat([torch.zeros((1, d), dtype=torch.float64, device="cuda"), dy[tokens.argsort()].double().cumsum(0)])
    counts = torch.bincount(tokens, minlength=v)
    want = before[counts.cumsum(0)] - before[counts.cumsum(0) - counts]
    want[2] = 0
    if accumulate:
        want += out
    api.embedding_grad_into(wrap(out), wrap(dy), wrap(tokens), padding=2, accumulate=accumulate)
    assert torch.equal(out.double(), want)


# ---- layer norm --------------------------------------------------------------------------------------------------------
# a width of each shape of a row (waves, elements to a lane, none) on both sides of what a launch of few rows takes, and with more rows than
# the most workgroups of four take in one turn
@pytest.mark.parametrize("rows", [1024, 1025, 6151, 13001])
@pytest.mark.parametrize("d", [1, 3, 24, 300, 768, 1500, 4096, 7003, 12288, 16391])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sums_over_rows(api, dtype, d, rows):
    most = int(((MOST - 1) // rows) ** 0.5)
    x, dy, wrap = whole((rows, d), most, dtype, 1), whole((rows, d), most, dtype, 2), api.as_tensor
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dx, dg, db = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    api.layer_norm_grad_into(*[wrap(t) for t in (dx, dg, db, dy, x)], None, wrap(mean), wrap(rstd))
    assert torch.equal(dg.double(), (x.float() * dy.float()).sum(0, dtype=torch.float64))
    assert torch.equal(db.double(), dy.sum(0, dtype=torch.float64))


def test_sums_over_more_than_four_gigabytes(api):
    rows, d, wrap = 540001, 2048, api.as_tensor
    x, dy = torch.full((rows, d), 2.0, device="cuda"), torch.full((rows, d), 1.0, device="cuda")
    assert x.numel() * 4 > 1 << 32
    x[::1001], dy[::997] = 3, 5
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dx, dg, db = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    api.layer_norm_grad_into(*[wrap(t) for t in (dx, dg, db, dy, x)], None, wrap(mean), wrap(rstd))
    assert (dg == float((x[:, 0].double() * dy[:, 0].double()).sum())).all() and (db == float(dy[:, 0].double().sum())).all()
