"""cvcudaxLayerNormSubmit and its gradient against their definition in 64 bits (row_reference.py derives the bounds)."""
import importlib

import numpy as np
import pytest
import torch

import row_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)]
EPS = 1e-5


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})  # (a wait for the default stream has the calls after it record events)


def rows_of(shape, dtype, seed, offset=0.3, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + offset).to(dtype)


def weights_of(d, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype), (0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype)


def layout_of(t):
    """A layout that lets rows have gaps."""
    return "ABDEFGW"[-t.ndim:]


def forward(api, x, gamma, beta, eps=EPS, out=None, stats=True, stream=None):
    wrap = lambda t: None if t is None else api.as_tensor(t, layout_of(t))
    out = torch.empty(x.shape, dtype=x.dtype, device="cuda") if out is None else out
    rows = x.shape[:-1] or (1,)
    mean, rstd = (torch.full(rows, 7.0, device="cuda") for _ in range(2)) if stats else (None, None)
    api.layer_norm_into(wrap(out), wrap(x), wrap(gamma), wrap(beta), eps, mean=wrap(mean), rstd=wrap(rstd), stream=stream)
    return out, mean, rstd


def check_forward(api, x, gamma, beta, eps=EPS, **kw):
    xd = x.double()
    gd, bd = (torch.ones(1, device="cuda").double() if gamma is None else gamma.double(),
              torch.zeros(1, device="cuda").double() if beta is None else beta.double())
    want = ref.layer_norm(xd, gd, bd, eps)
    errors = ref.layer_norm_errors(xd, gd, bd, want[1], want[2], eps)
    got = forward(api, x, gamma, beta, eps, **kw)
    for name, a, b, e in zip(("out", "mean", "rstd"), got, want, errors):
        if a is not None:
            ref.close(a.view(b.shape), b, e, name)
    return got


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 1), (1, 2), (5, 7), (2, 63), (3, 64), (4, 65), (1, 127), (7, 255), (2, 256), (5, 257),
                                    (3, 511), (66, 515), (130, 768), (33, 1000), (1, 4096), (1, 4095), (9, 4096), (700, 1023),
                                    (5, 5001), (3, 8192), (4, 12288), (2, 16385), (3, 20000), (1, 40001), (2, 70003)])
@pytest.mark.parametrize("dtype,weights", TYPES)
def test_forward(api, rows, d, dtype, weights):
    gamma, beta = weights_of(d, weights, 2)
    check_forward(api, rows_of((rows, d), dtype, rows * 7 + d), gamma, beta)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_forward_without_weights_and_statistics(api, dtype):
    x = rows_of((37, 200), dtype, 5)
    gamma, beta = weights_of(200, dtype, 6)
    for g, b in ((None, None), (gamma, None), (None, beta)):
        whole, _, _ = check_forward(api, x, g, b)
        alone, _, _ = forward(api, x, g, b, stats=False)
        assert torch.equal(whole, alone)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [24, 515, 768, 4096, 9001])
def test_rows_with_gaps_and_in_place(api, dtype, d):
    gamma, beta = weights_of(d, F32, 3)
    wide = rows_of((4, 6, d + 3), dtype, 8)
    x = wide[:, 1:, 1:d + 1]  # two distances, and rows that begin between 4-byte words
    keep = wide.clone()
    out = torch.full((4, 5, d + 5), 9.0, dtype=dtype, device="cuda")
    got, _, _ = check_forward(api, x, gamma, beta, out=out[:, :, 2:d + 2])
    assert torch.equal(wide, keep) and (out[:, :, :2] == 9).all() and (out[:, :, d + 2:] == 9).all()
    dense, _, _ = forward(api, x.contiguous(), gamma, beta)
    assert torch.equal(dense, got)
    forward(api, x, gamma, beta, out=x)
    assert torch.equal(dense, x)


def test_rows_far_from_zero_and_of_equal_values(api):
    d = 1024
    gamma, beta = weights_of(d, F32, 3)
    check_forward(api, rows_of((20, d), F32, 1, offset=3000.0), gamma, beta)   # the variance is 1e-7 of the squares
    check_forward(api, rows_of((20, d), F32, 1, offset=0.0, scale=1e-6), gamma, beta)
    check_forward(api, rows_of((20, d), F32, 1, scale=1e15), gamma, beta)
    out, mean, rstd = forward(api, torch.full((3, d), 2.5, device="cuda"), gamma, beta)
    assert torch.equal(out, beta.expand(3, d)) and (mean == 2.5).all()
    ref.close(rstd, torch.full((3,), EPS ** -0.5, dtype=torch.float64, device="cuda"), 8 * ref.U32 * EPS ** -0.5)


@pytest.mark.parametrize("d", [100, 768, 4096, 9000, 40000])
def test_what_is_not_finite_stays_in_its_row(api, d):
    gamma, beta = weights_of(d, F32, 3)
    x = rows_of((9, d), F32, 4)
    clean, _, _ = forward(api, x, gamma, beta)
    y = x.clone()
    y[2, d // 2], y[5, 0], y[7, d - 1] = float("nan"), float("inf"), float("-inf")
    got, _, _ = forward(api, y, gamma, beta)
    for r in range(9):
        assert got[r].isnan().all() if r in (2, 5, 7) else torch.equal(got[r], clean[r])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [8200, 16383, 24000])
def test_many_wide_rows(api, dtype, d):
    """More rows than workgroups that hold one: some go through one row, some through two, some through three."""
    gamma, beta = weights_of(d, dtype, 12)
    x = rows_of((600, d), dtype, 13)
    got, _, _ = check_forward(api, x, gamma, beta)
    forward(api, x, gamma, beta, out=x)
    assert torch.equal(x, got)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [2, 33001, 40003])
def test_rows_read_more_than_once_in_place(api, dtype, d):
    """Rows that do not fit the registers, their ends within a run: what is stored must not be read again."""
    gamma, beta = weights_of(d, F32, 3)
    x, dy = rows_of((5, d), dtype, 8), rows_of((5, d), dtype, 9)
    got, mean, rstd = check_forward(api, x, gamma, beta)
    dx = check_gradients(api, dy, x, gamma, mean, rstd)[0]
    for over in (dy, x):
        before = over.clone()
        made = [torch.empty(d, device="cuda") for _ in range(2)]
        api.layer_norm_grad_into(*[api.as_tensor(t) for t in (over, *made, dy, x, gamma, mean, rstd)])
        assert torch.equal(over, dx)
        over.copy_(before)
    forward(api, x, gamma, beta, out=x)
    assert torch.equal(x, got)


def test_more_than_four_gigabytes(api):
    rows, d = 1100000, 2048
    x = torch.empty((rows, d), dtype=F16, device="cuda")
    out = torch.empty_like(x)
    assert x.numel() * 2 > 1 << 32
    x[:1000].copy_(rows_of((1000, d), F16, 1))
    x[1000:-1000] = 0
    x[-1000:].copy_(rows_of((1000, d), F16, 2))
    gamma, beta = weights_of(d, F16, 3)
    forward(api, x, gamma, beta, out=out)
    for part in (slice(0, 1000), slice(rows - 1000, rows)):
        want = ref.layer_norm(x[part].double(), gamma.double(), beta.double(), EPS)
        e = ref.layer_norm_errors(x[part].double(), gamma.double(), beta.double(), want[1], want[2], EPS)
        ref.close(out[part], want[0], e[0])


def test_no_rows_and_no_elements(cv, api):
    op, grad = cv.LayerNorm(), cv.LayerNormGrad()
    none, out = cv.Tensor.alloc([0, 8], np.float32, "NW"), cv.Tensor.alloc([0, 8], np.float32, "NW")
    op(None, none, None, None, out)
    sums = [cv.Tensor.from_numpy(np.full(8, 5, np.float32), "W") for _ in range(2)]
    stats = cv.Tensor.alloc([0], np.float32, "W")
    grad(None, none, none, None, stats, stats, out, sums[0], sums[1], cv.Tensor.alloc([64], np.uint8, "W"))
    torch.cuda.synchronize()
    assert all((s.numpy() == 0).all() for s in sums)
    op(None, cv.Tensor.alloc([3, 0], np.float32, "NW"), None, None, cv.Tensor.alloc([3, 0], np.float32, "NW"))


# ---- gradient ----------------------------------------------------------------------------------------------------------
def gradients(api, dy, x, gamma, mean, rstd, out=None, weights=F32, stream=None):
    wrap = lambda t: None if t is None else api.as_tensor(t, layout_of(t))
    d = x.shape[-1]
    out = torch.empty(x.shape, dtype=x.dtype, device="cuda") if out is None else out
    sums = [torch.full((d,), 3.0, dtype=weights, device="cuda") for _ in range(2)]
    api.layer_norm_grad_into(wrap(out), wrap(sums[0]), wrap(sums[1]), wrap(dy), wrap(x), wrap(gamma), wrap(mean), wrap(rstd),
                             stream=stream)
    return out, sums[0], sums[1]


def check_gradients(api, dy, x, gamma, mean, rstd, weights=F32, **kw):
    args = (dy.double(), x.double(), torch.ones(1, device="cuda").double() if gamma is None else gamma.double(), mean.double(),
            rstd.double())
    got = gradients(api, dy, x, gamma, mean, rstd, weights=weights, **kw)
    for name, a, b, e in zip(("dx", "dgamma", "dbeta"), got, ref.layer_norm_grad(*args), ref.layer_norm_grad_errors(*args)):
        ref.close(a, b, e, name)
    return got


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 1), (1, 2), (5, 7), (2, 63), (300, 64), (4, 65), (1, 127), (7, 255), (2000, 256),
                                    (5, 257), (3, 511), (661, 515), (1300, 768), (33, 1000), (1, 4096), (1, 4095), (257, 4096),
                                    (700, 1023), (5, 5001), (3, 8192), (40, 12288), (2, 16385), (3, 20000), (1, 40001), (2, 70003),
                                    (10000, 24), (5000, 3)])
@pytest.mark.parametrize("dtype,weights", TYPES)
def test_gradient(api, rows, d, dtype, weights):
    gamma, beta = weights_of(d, weights, 2)
    x, dy = rows_of((rows, d), dtype, rows + d), rows_of((rows, d), dtype, rows * 3 + d, offset=0.01, scale=0.1)
    _, mean, rstd = forward(api, x, gamma, beta)
    check_gradients(api, dy, x, gamma, mean, rstd, weights)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [24, 515, 768, 4096, 9001])
def test_gradient_of_rows_with_gaps_and_in_place(api, dtype, d):
    gamma, beta = weights_of(d, F32, 3)
    wide, wide_dy = rows_of((4, 6, d + 3), dtype, 8), rows_of((4, 5, d + 1), dtype, 9)
    x, dy = wide[:, 1:, 1:d + 1], wide_dy[..., :d]
    _, mean, rstd = forward(api, x, gamma, beta)
    got = check_gradients(api, dy, x, gamma, mean, rstd)
    for over in (dy, x):
        before = over.clone()
        again = gradients(api, dy, x, gamma, mean, rstd, out=over)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
        over.copy_(before)


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 255, 256, 257, 1024, 1025])
@pytest.mark.parametrize("d", [4, 31, 32, 33, 765, 1025, 4099, 8201])
def test_gradient_of_few_rows(api, rows, d):
    """One launch or two, whole and ragged tiles of columns and rows; over its inputs, and with NaN in one row."""
    gamma, beta = weights_of(d, F32, 2)
    x, dy = rows_of((rows, d), BF16, rows + d), rows_of((rows, d), BF16, rows * 3 + d, offset=0.01, scale=0.1)
    _, mean, rstd = forward(api, x, gamma, beta)
    got = check_gradients(api, dy, x, gamma, mean, rstd)
    before = dy.clone()
    again = gradients(api, dy, x, gamma, mean, rstd, out=dy)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    before[rows - 1, d - 1] = float("nan")
    dx, dg, db = gradients(api, before, x, gamma, mean, rstd)
    assert torch.equal(dx[:-1], got[0][:-1]) and dx[-1].isnan().all()
    assert torch.equal(dg[:-1], got[1][:-1]) and torch.equal(db[:-1], got[2][:-1]) and dg[-1].isnan() and db[-1].isnan()


def test_gradient_without_some_of_them(api):
    x, dy = rows_of((50, 300), BF16, 1), rows_of((50, 300), BF16, 2)
    gamma, beta = weights_of(300, BF16, 3)
    _, mean, rstd = forward(api, x, gamma, beta)
    whole = gradients(api, dy, x, gamma, mean, rstd, weights=BF16)
    wrap = api.as_tensor
    for g, b in ((True, False), (False, True), (False, False)):
        out, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
        api.layer_norm_grad_into(wrap(out), wrap(dg) if g else None, wrap(db) if b else None, wrap(dy), wrap(x), wrap(gamma), wrap(mean),
                                 wrap(rstd))
        assert torch.equal(out, whole[0])
        assert (not g or torch.equal(dg, whole[1])) and (not b or torch.equal(db, whole[2]))
    check_gradients(api, dy, x, None, mean, rstd)


def test_gradient_against_differences():
    # the formula itself, in 64 bits on the CPU, against central differences of the definition (steps of 1e-5: 1e-9 or less
    # of third derivatives, 1e-10 of roundings)
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn((3, 11), generator=g, dtype=torch.float64) for _ in range(2))
    gamma, beta = (torch.randn(11, generator=g, dtype=torch.float64) for _ in range(2))
    _, mean, rstd = ref.layer_norm(x, gamma, beta, EPS)
    want = ref.layer_norm_grad(dy, x, gamma, mean, rstd)
    for t, grad in zip((x, gamma, beta), want):
        for i in range(t.numel()):
            ends = []
            for h in (1e-5, -1e-5):
                t.view(-1)[i] += h
                ends.append(float((ref.layer_norm(x, gamma, beta, EPS)[0] * dy).sum()))
                t.view(-1)[i] -= h
            assert abs((ends[0] - ends[1]) / 2e-5 - float(grad.view(-1)[i])) < 1e-7


def test_gradient_is_the_same_in_every_call(api):
    x, dy = rows_of((5000, 768), F16, 1), rows_of((5000, 768), F16, 2)
    gamma, beta = weights_of(768, F32, 3)
    _, mean, rstd = forward(api, x, gamma, beta)
    first = gradients(api, dy, x, gamma, mean, rstd)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, gradients(api, dy, x, gamma, mean, rstd)))


def test_gradient_of_what_is_not_finite(api):
    x, dy = rows_of((40, 600), F32, 1), rows_of((40, 600), F32, 2)
    gamma, beta = weights_of(600, F32, 3)
    _, mean, rstd = forward(api, x, gamma, beta)
    clean = gradients(api, dy, x, gamma, mean, rstd)
    dy[7, 11] = float("inf")
    got = gradients(api, dy, x, gamma, mean, rstd)
    others = [r for r in range(40) if r != 7]
    columns = [c for c in range(600) if c != 11]
    assert torch.equal(got[0][others], clean[0][others]) and not got[0][7].isfinite().any()
    for k in (1, 2):
        assert torch.equal(got[k][columns], clean[k][columns]) and not got[k][11].isfinite()


def test_gradient_of_more_than_four_gigabytes(api):
    rows, d = 540000, 2048
    x, dy = (torch.zeros((rows, d), device="cuda") for _ in range(2))
    assert x.numel() * 4 > 1 << 32
    x[-500:], dy[-500:] = rows_of((500, d), F32, 1), rows_of((500, d), F32, 2)
    gamma, _ = weights_of(d, F32, 3)
    _, mean, rstd = ref.layer_norm(x[-500:].double(), gamma.double(), gamma.double(), EPS)
    stats = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    stats[0][-500:], stats[1][-500:] = mean, rstd
    got = gradients(api, dy, x, gamma, *stats)
    args = (dy[-500:].double(), x[-500:].double(), gamma.double(), stats[0][-500:].double(), stats[1][-500:].double())
    for a, b, e in zip((got[0][-500:], got[1], got[2]), ref.layer_norm_grad(*args), ref.layer_norm_grad_errors(*args)):
        ref.close(a, b, e)
    assert (got[0][:-500] == 0).all()


def test_another_stream(api):
    # work given to a stream of its own waits for what another stream is still writing
    x, dy = rows_of((4096, 1000), F32, 1), rows_of((4096, 1000), F32, 2)
    gamma, beta = weights_of(1000, F32, 3)
    want, mean, rstd = forward(api, x, gamma, beta)
    grads = gradients(api, dy, x, gamma, mean, rstd)
    torch.cuda.synchronize()
    side = api.Stream()
    tx, out = api.as_tensor(x), api.Tensor((4096, 1000), np.float32)
    middle = api.layer_norm(tx, api.as_tensor(gamma), api.as_tensor(beta), EPS)
    api.layer_norm_into(out, middle, api.as_tensor(gamma), api.as_tensor(beta), EPS, stream=side)
    again = api.layer_norm(middle, api.as_tensor(gamma), api.as_tensor(beta), EPS)
    with side:
        other = api.layer_norm_grad(api.as_tensor(dy), tx, api.as_tensor(gamma), api.as_tensor(mean), api.as_tensor(rstd))
    torch.cuda.synchronize()
    assert torch.equal(middle.torch(), want) and torch.equal(out.torch(), again.torch())
    assert all(torch.equal(a.torch(), b) for a, b in zip(other, grads))


def test_in_a_graph(api):
    x, dy = rows_of((300, 768), F16, 1), rows_of((300, 768), F16, 2)
    gamma, beta = weights_of(768, F32, 3)
    out, (mean, rstd) = torch.empty_like(x), (torch.empty(300, device="cuda") for _ in range(2))
    dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    room = torch.empty(api.LayerNormGrad.workspace(300, 768), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    t = {k: api.as_tensor(v) for k, v in dict(x=x, dy=dy, gamma=gamma, beta=beta, out=out, mean=mean, rstd=rstd, dx=dx, dg=dg, db=db,
                                               room=room).items()}
    with torch.cuda.graph(graph):
        s = api.as_stream(torch.cuda.current_stream())
        api.layer_norm_into(t["out"], t["x"], t["gamma"], t["beta"], EPS, mean=t["mean"], rstd=t["rstd"], stream=s)
        api.layer_norm_grad_into(t["dx"], t["dg"], t["db"], t["dy"], t["x"], t["gamma"], t["mean"], t["rstd"], workspace=t["room"], stream=s)
    for k in range(4):
        x.copy_(rows_of((300, 768), F16, 10 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (out, mean, rstd, dx, dg, db)]
        want = check_forward(api, x, gamma, beta)
        want += check_gradients(api, dy, x, gamma, want[1], want[2])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
