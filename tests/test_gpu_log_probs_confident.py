"""Log probabilities of rows in which one logit stands far above the others: what the others leave of it, 1 - p, is small, and the log
probability -log(p) and the entropy are known as well as it is, never above 0 and never below."""
import importlib
import math

import pytest
import torch

from row_reference import U32, close

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SLACK = 2.0  # how far a logit may lie above the one that its lane's exponentials are taken relative to


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


def reference(logits, tokens, scale):
    """(log probabilities, entropies) in 64 bits, and how far off 32 bits may be. With `far` from the row's first largest logit to another,
    that one's exponential is off by 4 * U32 for each of `far` and by 4 * U32, and so is each factor by which sums are rescaled on its way,
    3 of them for each SLACK of `far` (two are for the rounding of scale * logit) and 4 at the end; additions are one for each run of a lane (of
    16 bytes, 64 lanes at least) and some 32 for the lanes and waves. A largest logit that is in the sums itself is at most SLACK above another, so
    that 1 - p is at least 1 / (1 + e^SLACK), and its errors, and those of every addition, count times the inverse of that. Terms of the
    entropy are made of differences up to 2 * SLACK longer than `far`."""
    z = scale * logits
    rows, v = z.shape
    first = z == z.amax(1, keepdim=True)
    first &= first.cumsum(1) == 1
    far = (z.amax(1, keepdim=True) - z)
    e = torch.where(first, 0.0, torch.exp(-far))
    rest = e.sum(1, keepdim=True)
    p = e / (1 + rest)
    far = torch.where(p > 0, far, 0.0)                                # (-infinity has no share)
    less = p.sum(1)
    sums = torch.log1p(rest)[:, 0]
    there = (tokens >= 0) & (tokens < v)
    its = (z.amax(1, keepdim=True) - z).gather(1, tokens.long().clamp(0, v - 1)[:, None])[:, 0]
    logp = torch.where(there, -its - sums, 0.0)
    entropy = sums + (p * far).sum(1)
    n, worst = v / 256 + 32, 1 + math.exp(SLACK)
    rel = (4 + 3 * 4 / SLACK) * far + 4 + 4 * 4 + n                   # of each exponential and its way, in U32
    e_sums = U32 * ((p * rel).sum(1) + less * worst * (8 * SLACK + 24 + n) + 4 * sums)
    e_logp = torch.where(there, U32 * (3 * its + logp.abs()) + e_sums, 0.0) + 2.0 ** -100
    e_terms = U32 * ((p * (far + 2 * SLACK) * (rel + 4)).sum(1) + less * worst * 2 * SLACK * (8 * SLACK + 28 + n))
    e_entropy = e_sums + e_terms + (entropy - sums) * (e_sums + 4 * U32) + U32 * entropy + 2.0 ** -100
    return logp, entropy, e_logp, e_entropy


def check(api, logits, tokens, scale, top=0):
    n, v = logits.shape
    out, entropy, lse = (torch.full((n,), 7.0, device="cuda") for _ in range(3))
    wrap, more = api.as_tensor, {}
    if top:
        values, words = torch.full((n, top), 7.0, device="cuda"), torch.full((n, top), -7, dtype=torch.int32, device="cuda")
        more = {"top_values": wrap(values), "top_tokens": wrap(words)}
    api.log_probs_into(wrap(out), wrap(logits), wrap(tokens), scale, entropy=wrap(entropy), lse=wrap(lse), **more)
    exactly = float(torch.tensor(scale, dtype=F32))  # (the operator's scale has 32 bits)
    want = reference(logits.double(), tokens, exactly)
    assert (out <= 0).all() and (entropy >= 0).all()
    close(out, want[0], want[2], "log probability")
    close(entropy, want[1], want[3], "entropy")
    if top:
        assert (values <= 0).all() and (values.diff(dim=1) <= 0).all()
        for i in range(top):
            one = reference(logits.double(), words[:, i], exactly)
            close(values[:, i], one[0], one[2], "log probability of the first but %d" % i)
    return out


GAPS = [0.0, 0.5, 1.9, 2.1, 4.0, 7.9, 10.0, 13.0, 16.0, 19.9, 20.1, 26.0, 40.0, 70.0]


def rows_with_peaks(v, dtype, seed, scale, copies=1):
    """For each gap some rows of which one logit stands that much, times the scale, above the largest other one: anywhere, in the row's first
    logits, and in its last."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = 3 * len(GAPS) * copies
    x = (torch.randn((n, v), generator=g, device="cuda") * 2).to(dtype)
    at = torch.randint(0, v, (n,), generator=g, device="cuda")
    at[1::3] = torch.randint(0, min(v, 8), (len(at[1::3]),), generator=g, device="cuda")
    at[2::3] = v - 1 - torch.randint(0, min(v, 8), (len(at[2::3]),), generator=g, device="cuda")
    gap = torch.tensor(GAPS, device="cuda").repeat_interleave(3).repeat(copies)
    row = torch.arange(n, device="cuda")
    x[row, at] = -math.inf
    x[row, at] = (x.amax(1).float() + gap / scale).to(dtype)
    tokens = torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, at, torch.randint(0, v, (n,), generator=g, device="cuda"))
    return x, tokens


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [1.0, 0.8, 1.7])
@pytest.mark.parametrize("v", [3, 9, 500, 1001, 4000, 32000, 130001])
def test_rows_with_a_peak(api, v, scale, dtype):
    x, tokens = rows_with_peaks(v, dtype, v, scale)
    check(api, x, tokens, scale, min(v, 5))
    if v <= 4000:  # (rows that fill the card: fewer waves to a row)
        x, tokens = rows_with_peaks(v, dtype, v + 1, scale, 100)
        check(api, x, tokens, scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_peaks_of_equal_logits_and_above_far_ones(api, dtype):
    x, tokens = rows_with_peaks(2000, dtype, 5, 1.0)
    x[:, 700] = x[torch.arange(len(x)), tokens]      # another one of that logit
    check(api, x, tokens, 1.0, 8)
    x, tokens = rows_with_peaks(2000, dtype, 6, 1.0)
    x[:, ::2] = torch.where(x[:, ::2] == x.amax(1, keepdim=True), x[:, ::2], torch.full_like(x[:, ::2], -1e4))
    x[:, 1::50] = torch.where(x[:, 1::50] == x.amax(1, keepdim=True), x[:, 1::50], torch.full_like(x[:, 1::50], -math.inf))
    check(api, x, tokens, 1.0, 8)
    # one logit that is not -infinity
    x = torch.full((6, 3000), -math.inf, device="cuda").to(dtype)
    tokens = torch.tensor([0, 1, 63, 64, 2047, 2999], device="cuda")
    x[torch.arange(6), tokens] = torch.tensor([-3e4, -1.5, 0.0, 0.3, 100.0, 3e4], device="cuda").to(dtype)
    for scale in (1.0, 0.3):
        out, entropy = torch.full((6,), 7.0, device="cuda"), torch.full((6,), 7.0, device="cuda")
        api.log_probs_into(api.as_tensor(out), api.as_tensor(x), api.as_tensor(tokens), scale, entropy=api.as_tensor(entropy))
        assert (out == 0).all() and (entropy == 0).all()


def test_near_certain_tokens_keep_their_digits(api):
    """One token of 1 - p down to 1e-20: a log probability of two or three right digits at least, where 32 bits hold no 1 - 1e-20."""
    v = 32000
    x = torch.zeros((40, v), device="cuda")
    tokens = torch.arange(40, device="cuda") * 799 + 5
    peaks = torch.linspace(12, 56, 40, device="cuda")
    x[torch.arange(40), tokens] = peaks
    out = check(api, x, tokens, 1.0)
    rest = (v - 1) * torch.exp(-peaks.double())
    assert ((out.double() + torch.log1p(rest)).abs() <= 2e-3 * torch.log1p(rest)).all() and (out < 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_at_both_ends_of_the_type(api, dtype):
    """Of logits that lie further apart than the type reaches, scaled down: log probabilities are finite."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.full((3, 1000), low, device="cuda").to(dtype)
    x[0, 5], x[1, 900], x[2, 0] = high, high, 1.0
    tokens = torch.tensor([7, 900, 999], device="cuda")
    out = check(api, x, tokens, 0.25, 3)
    assert out.isfinite().all() and out[0] < -1e38 and out[1] == 0
