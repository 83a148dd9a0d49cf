"""cvcudaxLogProbsSubmit and its gradient against their definition in 64 bits (head_reference.py derives the bounds)."""
import importlib
import math

import numpy as np
import pytest
import torch

import head_reference as ref
from row_reference import close

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


def random(shape, dtype, seed, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def words(n, v, seed, dtype=torch.int64):
    """Tokens, some of them padding."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    made = torch.randint(0, v, (n,), generator=g, device="cuda").to(dtype)
    made[::5] = -1
    made[3::7] = v
    return made


def run(api, x, tokens, scale=1.0, top=0, stats=True, stream=None):
    n = x.shape[0]
    made = [torch.full((n,), 7.0, device="cuda") for _ in range(3)]
    more, wrap = {}, api.as_tensor
    if stats:
        more = {"entropy": wrap(made[1]), "lse": wrap(made[2])}
    if top:
        made += [torch.full((n, top), 7.0, device="cuda"), torch.full((n, top), 7, dtype=torch.int32, device="cuda")]
        more.update(top_values=wrap(made[3]), top_tokens=wrap(made[4]))
    api.log_probs_into(wrap(made[0]), api.as_tensor(x, "NW"), wrap(tokens), scale, stream=stream, **more)
    return made


def first_of_the_largest(x, top):
    """The columns of the `top` largest of each row, of equal ones the first, a NaN before all numbers."""
    key = torch.where(x.isnan(), torch.full_like(x, INF).double(), x.double() + 0.0)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    nan = x.isnan().gather(1, order)
    order = order.gather(1, torch.sort(nan.int(), dim=1, descending=True, stable=True).indices)
    return order[:, :top].int()


def check(api, x, tokens, scale=1.0, top=0):
    got = run(api, x, tokens, scale, top)
    want, errors = ref.log_probs(x.double(), tokens, scale)
    for name, a, b, e in zip(("log probabilities", "entropy", "lse"), got, want, errors):
        same = b == -INF
        assert (a[same] == -INF).all()
        close(a[~same], b[~same], e[~same], name)
    if top:
        at = first_of_the_largest(x, top)
        assert torch.equal(got[4], at)
        for k in range(top):
            b, e = ref.log_probs(x.double(), at[:, k], scale)
            same = b[0] == -INF
            assert (got[3][:, k][same] == -INF).all()
            close(got[3][:, k][~same], b[0][~same], e[0][~same], "top value %d" % k)
    return got


SIZES = [(1, 1), (3, 2), (5, 7), (4, 63), (2, 64), (3, 65), (9, 511), (7, 515), (40, 1000), (5, 2048), (3, 2049), (4, 5001), (2, 16384), (3, 16385),
         (5, 30011), (1, 128000), (600, 16500), (2, 150001)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,v", SIZES)
def test_rows(api, n, v, dtype):
    x = random((n, v), dtype, n + v)
    check(api, x, words(n, v, 1), 1.0, min(5, v))
    check(api, x, words(n, v, 2, torch.int32), 0.7, min(32, v))
    assert torch.equal(run(api, x, words(n, v, 1), stats=False)[0], run(api, x, words(n, v, 1), top=1)[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [5, 64, 1000, 3001, 20000, 40001])
def test_equal_logits(api, v, dtype):
    """All the same, two values, a few levels, zeros of both signs, more candidates than room for them."""
    x = torch.zeros((6, v), dtype=dtype, device="cuda")
    x[1, v // 2:] = 1
    x[2] = random((v,), dtype, 1).round()
    x[3, ::2] = -0.0
    x[4, -3:] = 2.5
    x[5] = -1
    check(api, x, words(6, v, 1), 1.0, min(32, v))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [5, 700, 5000, 20000])
def test_masked_logits(api, v, dtype):
    """Logits of -infinity, all but one, all but a few, all of them; of the type's lowest value."""
    x = random((7, v), dtype, 1)
    x[0, 1:] = -INF
    x[1, :-1] = -INF
    x[2, 3:] = -INF
    x[3] = -INF
    x[4, : v // 2] = -INF
    x[5, 2:] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).min
    tokens = torch.tensor([0, v - 1, 4, 1, 0, 2, 3], device="cuda")
    got = check(api, x, tokens, 1.0, min(5, v))
    assert got[2][3] == -INF and got[0][3] == -INF and got[1][3] == 0 and got[0][2] == -INF and got[1][0] == 0


@pytest.mark.parametrize("v", [300, 3000, 30000])
def test_what_is_not_finite_stays_in_its_row(api, v):
    x = random((6, v), F32, 3)
    tokens = torch.tensor([1, 2, 3, -1, 4, 5], device="cuda")
    clean = run(api, x, tokens, top=4)
    x[1, 7], x[3, 9], x[3, 200], x[4, 5] = NAN, NAN, -NAN, INF
    got = run(api, x, tokens, top=4)
    for r in range(6):
        for a, b in zip(got, clean):
            assert r in (1, 3, 4) or torch.equal(a[r], b[r])
    assert got[0][1].isnan() and got[0][3] == 0 and got[0][4].isnan() and got[2][[1, 3, 4]].isnan().all()
    assert torch.equal(got[4], first_of_the_largest(x, 4)) and got[3][[1, 3, 4]].isnan().all()


def test_large_and_small_logits(api):
    tokens = torch.tensor([0, 1, 2], device="cuda")
    for size in (1e-3, 50.0, 1e4):
        check(api, random((3, 9000), F32, 4, size), tokens, 1.0, 8)
    check(api, random((3, 9000), F32, 4, 1e4) + 1e6, tokens, 1e-4, 8)
    x = random((3, 5000), F32, 5, 3e37)  # differences that 32 bits do not hold
    got = run(api, x, tokens, top=1)
    assert (got[1] == 0).all() and (got[3] == 0).all() and torch.equal(got[4][:, 0], x.argmax(1).int())


def test_rows_with_gaps(api):
    for dtype in (F32, BF16):
        wide = random((20, 3010), dtype, 6)
        x = wide[:, 1:3002]  # rows that begin between 4-byte words
        got = check(api, x, words(20, 3001, 1), 1.0, 5)
        assert all(torch.equal(a, b) for a, b in zip(got, run(api, x.contiguous(), words(20, 3001, 1), 1.0, 5)))


def test_more_than_four_gigabytes(api):
    n, v = 17000, 128000
    x = torch.zeros((n, v), dtype=BF16, device="cuda")
    assert x.numel() > 1 << 31
    x[-20:] = random((20, v), BF16, 7)
    tokens = words(n, v, 8)
    got = run(api, x, tokens, 1.0, 3)
    want, errors = ref.log_probs(x[-20:].double(), tokens[-20:], 1.0)
    for a, b, e in zip(got, want, errors):
        close(a[-20:], b, e)
    assert torch.equal(got[4][-20:], first_of_the_largest(x[-20:], 3)) and torch.equal(got[4][0].cpu(), torch.arange(3, dtype=torch.int32))
    grad = torch.ones(n, device="cuda")
    made = gradient(api, x, tokens, got[2], grad, out=x)
    b, e = ref.log_probs_grad(random((20, v), BF16, 7).double(), tokens[-20:], got[2][-20:].double(), grad[-20:].double(), 1.0)
    close(made[-20:], b, e)


# ---- gradient ----------------------------------------------------------------------------------------------------------
def gradient(api, x, tokens, lse, grad, scale=1.0, entropy=None, grad_entropy=None, out=None):
    out = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") if out is None else out
    wrap = lambda t: None if t is None else api.as_tensor(t)
    api.log_probs_grad_into(api.as_tensor(out, "NW"), api.as_tensor(x, "NW"), wrap(tokens), wrap(lse), wrap(grad), scale, entropy=wrap(entropy),
                            grad_entropy=wrap(grad_entropy))
    return out


def check_gradient(api, x, tokens, scale=1.0, out=None, size=1.0):
    _, entropy, lse = run(api, x, tokens, scale)
    n = x.shape[0]
    g, h = random((n,), F32, 11, size), random((n,), F32, 12, size)
    xd = x.double()
    got = gradient(api, x, tokens, lse, g, scale)
    want = ref.log_probs_grad(xd, tokens, lse.double(), g.double(), scale)
    close(got, *want)
    both = gradient(api, x, tokens, lse, g, scale, entropy, h, out=out)
    want = ref.log_probs_grad(xd, tokens, lse.double(), g.double(), scale, entropy.double(), h.double())
    close(both, *want)
    return got, both, (lse, g, entropy, h)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,v", SIZES)
def test_gradient(api, n, v, dtype):
    x = random((n, v), dtype, n + v)
    check_gradient(api, x, words(n, v, 1))
    check_gradient(api, x, words(n, v, 2, torch.int32), 1.6)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [3, 1000, 8195, 20001])
def test_gradient_of_rows_with_gaps_and_in_place(api, v, dtype):
    wide, tokens = random((9, v + 5), dtype, 1), words(9, v, 1)
    x, out = wide[:, 3:v + 3], torch.full((9, v + 4), 9.0, dtype=dtype, device="cuda")
    got, both, (lse, g, entropy, h) = check_gradient(api, x, tokens, out=out[:, 1:v + 1])
    assert (out[:, 0] == 9).all() and (out[:, v + 1:] == 9).all()
    keep = wide.clone()
    gradient(api, x, tokens, lse, g, 1.0, entropy, h, out=x)
    assert torch.equal(x, both) and torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, v + 3:], keep[:, v + 3:])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradient_of_masked_logits(api, dtype):
    x = random((5, 700), dtype, 2)
    x[0, 1:], x[1], x[2, :350], x[3, 1:] = -INF, -INF, -INF, torch.finfo(dtype).min
    tokens = torch.tensor([0, 5, 3, 0, -1], device="cuda")
    got, both, _ = check_gradient(api, x, tokens)
    assert (got[1] == 0).all() and (both[1] == 0).all() and (got[4] == 0).all() and got.isfinite().all() and both.isfinite().all()
    assert (got[2, :3] == 0).all()


def test_gradient_of_what_is_not_finite(api):
    x = random((3, 900), F32, 3)
    tokens = torch.tensor([1, 2, 3], device="cuda")
    x[1, 4] = NAN
    _, _, lse = run(api, x, tokens)
    got = gradient(api, x, tokens, lse, torch.ones(3, device="cuda"))
    assert got[1].isnan().all() and got[[0, 2]].isfinite().all()


def test_whole_interface(api):
    """New tensors, another stream, and a graph of both directions that is replayed with other logits."""
    x, tokens = random((300, 5000), BF16, 4), words(300, 5000, 5)
    g = random((300,), F32, 6)
    want = run(api, x, tokens)
    grads = gradient(api, x, tokens, want[2], g)
    wrap, side = api.as_tensor, api.Stream()
    lse = api.Tensor((300,), np.float32)
    logp = api.log_probs(wrap(x), wrap(tokens), lse=lse)
    with side:
        made = api.log_probs_grad(wrap(x), wrap(tokens), lse, wrap(g))
    torch.cuda.synchronize()
    assert torch.equal(logp.torch(), want[0]) and torch.equal(made.torch(), grads)
    out, stats, to = torch.empty(300, device="cuda"), torch.empty(300, device="cuda"), torch.empty_like(x)
    graph, t = torch.cuda.CUDAGraph(), [wrap(a) for a in (out, stats, to, x, tokens, g)]
    with torch.cuda.graph(graph):
        s = api.as_stream(torch.cuda.current_stream())
        api.log_probs_into(t[0], t[3], t[4], lse=t[1], stream=s)
        api.log_probs_grad_into(t[2], t[3], t[4], t[1], t[5], stream=s)
    for turn in range(3):
        x.copy_(random((300, 5000), BF16, 40 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), stats.clone(), to.clone()
        want = run(api, x, tokens)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2]) and torch.equal(got[2], gradient(api, x, tokens, want[2], g))


@pytest.mark.parametrize("dtype,n", [(F32, 1100), (F16, 2200), (BF16, 2200)])
def test_many_rows_of_an_odd_width(api, dtype, n):
    """More logits than the card keeps near its memory; rows begin at odd addresses and end within a run."""
    v = 32003
    x = random((n, v), dtype, 13, 3.0)
    assert x.numel() * x.element_size() > 128 << 20
    check(api, x, words(n, v, 14), 0.9, 5)
    tokens = words(n, v, 15)
    got, both, (lse, g, entropy, h) = check_gradient(api, x, tokens)
    assert torch.equal(gradient(api, x, tokens, lse, g, 1.0, entropy, h, out=x), both)
