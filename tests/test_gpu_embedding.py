"""cvcudaxEmbeddingSubmit and its gradient against their definition in 64 bits. A lookup is one product and one rounding; a
row's gradient a sum of as many terms as its token occurs, in any order: that many roundings of their magnitudes (and one for the
scale, one for what it is added to)."""
import importlib
import math

import numpy as np
import pytest
import torch

import row_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16)]


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})  # (a wait for the default stream has the calls after it record events)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


def words(n, v, seed, dtype=torch.int64):
    """The k-th word about 1/k as often as the first."""
    u = torch.rand((n,), generator=gen(seed), device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1).to(dtype)


def layout_of(t):
    return "ABDEFGW"[-t.ndim:]


def wrap(api, t):
    return None if t is None else api.as_tensor(t, layout_of(t))


@pytest.mark.parametrize("table_type,out_type", PAIRS + [(F32, F16), (F32, BF16)])
@pytest.mark.parametrize("tokens_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 9, 4096), (3, 5, 7), (8, 1000, 64), (17, 100, 515), (1000, 77, 768), (5, 300, 9001),
                                   (20000, 50, 24)])
def test_lookup(api, n, v, d, table_type, out_type, tokens_type):
    table, tokens = normal((v, d), table_type, d), words(n, v, n, tokens_type)
    out = torch.full((n, d), 5.0, dtype=out_type, device="cuda")
    scale = math.sqrt(d)
    api.embedding_into(wrap(api, out), wrap(api, table), wrap(api, tokens), scale)
    want = table.double()[tokens.long()] * float(np.float32(scale))
    ref.close(out, want, ref.U32 * want.abs())
    whole = api.embedding(wrap(api, table), wrap(api, tokens), scale, dtype=out_type).torch()
    assert whole.dtype == out_type and torch.equal(whole, out)


def test_lookup_of_unknown_tokens_and_shapes(api):
    table = normal((10, 33), F32, 1)
    tokens = torch.tensor([[3, -1, 10], [9, 0, 1 << 40], [-(1 << 40), (1 << 32) + 3, 5]], device="cuda")
    out = api.embedding(api.as_tensor(table), api.as_tensor(tokens)).torch()
    known = (tokens >= 0) & (tokens < 10)
    assert out.shape == (3, 3, 33) and torch.equal(out[known], table[tokens[known]]) and (out[~known] == 0).all()
    small = torch.tensor([-1, 10, -(1 << 31), (1 << 31) - 1, 4], dtype=torch.int32, device="cuda")
    out = api.embedding(api.as_tensor(table), api.as_tensor(small)).torch()
    assert (out[:4] == 0).all() and torch.equal(out[4], table[4])
    # an unknown token's row is zeros also where the table's first row is not finite
    table[0] = float("nan")
    assert (api.embedding(api.as_tensor(table), api.as_tensor(small)).torch()[:4] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [24, 515, 1024])
def test_lookup_between_rows_with_gaps(api, dtype, d):
    wide = normal((20, d + 3), dtype, 1)
    tokens = words(12, 20, 2).view(3, 4)
    out = torch.full((3, 5, d + 5), 9.0, dtype=dtype, device="cuda")
    api.embedding_into(wrap(api, out[:, 1:, 1:d + 1]), wrap(api, wide[:, 1:d + 1]), wrap(api, tokens.contiguous()))
    assert torch.equal(out[:, 1:, 1:d + 1], wide[tokens][..., 1:d + 1])
    assert (out[:, 0] == 9).all() and (out[..., 0] == 9).all() and (out[..., d + 1:] == 9).all()


def test_lookup_beyond_four_gigabytes(api):
    v, d = 600000, 2048
    table = torch.empty((v, d), device="cuda")
    assert table.numel() * 4 > 1 << 32
    table[-100:], table[:100] = normal((100, d), F32, 1), normal((100, d), F32, 2)
    tokens = torch.tensor([v - 1, v - 100, 0, 99, v - 50], device="cuda")
    out = api.embedding(api.as_tensor(table), api.as_tensor(tokens)).torch()
    assert torch.equal(out, table[tokens])
    # as many rows of the result: the last tokens' places
    n = 1100000
    many = torch.zeros(n, dtype=torch.int32, device="cuda")
    many[-1000:] = torch.arange(1000, device="cuda") % 100
    out = torch.empty((n, d), dtype=BF16, device="cuda")
    api.embedding_into(api.as_tensor(out), api.as_tensor(table), api.as_tensor(many))
    assert torch.equal(out[-1000:], table[:100].bfloat16().repeat(10, 1))
    assert torch.equal(out[n // 2], table[0].bfloat16())


# ---- gradient ----------------------------------------------------------------------------------------------------------
def check_gradient(api, dy, tokens, v, out_type, scale=1.0, padding=None, accumulate=False, out=None):
    d = dy.shape[-1]
    flat, rows = tokens.reshape(-1).long(), dy.reshape(-1, d).double()
    keep = (flat >= 0) & (flat < v) & (flat != (-1 if padding is None else padding))
    total, size = torch.zeros((v, d), dtype=torch.float64, device="cuda"), torch.zeros((v, d), dtype=torch.float64, device="cuda")
    total.index_put_((flat[keep],), rows[keep], accumulate=True)
    size.index_put_((flat[keep],), rows[keep].abs(), accumulate=True)
    count = torch.bincount(flat[keep], minlength=v)[:, None]
    scale32 = float(np.float32(scale))
    if out is None:
        out = torch.full((v, d), 3.0, dtype=out_type, device="cuda")
    before = out.clone()
    want, error = total * scale32, (count + 2) * ref.U32 * size * abs(scale32)
    if accumulate:
        want = want + before.double()
        error = error + ref.U32 * want.abs()
    api.embedding_grad_into(wrap(api, out), wrap(api, dy), wrap(api, tokens), scale, padding=padding, accumulate=accumulate)
    absent = (count == 0)[:, 0]
    assert torch.equal(out[absent], before[absent]) if accumulate else (out[absent] == 0).all()
    ref.close(out[~absent], want[~absent], error[~absent])
    return out


@pytest.mark.parametrize("in_type,out_type", PAIRS + [(F16, F32), (BF16, F32)])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 9, 4096), (3, 5, 7), (64, 1000, 64), (255, 100, 515), (1003, 300, 515), (5000, 77, 768),
                                   (2049, 40000, 260), (4097, 3, 24), (9000, 1000, 33), (70001, 120000, 16), (20000, 130, 1030)])
def test_gradient(api, n, v, d, in_type, out_type):
    tokens = words(n, v, n)
    dy = normal((n, d), in_type, d, 0.1)
    check_gradient(api, dy, tokens, v, out_type, math.sqrt(d))
    check_gradient(api, dy, tokens.int(), v, out_type, padding=0)
    check_gradient(api, dy, tokens, v, out_type, 0.5, accumulate=True, out=normal((v, d), out_type, 3))


@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 127, 1000, 4096, 30000])
def test_gradient_of_one_token_and_of_different_ones(api, n):
    d = 130
    dy = normal((n, d), F32, n)
    one = torch.full((n,), 41, device="cuda")
    check_gradient(api, dy, one, 50, F32)
    assert (check_gradient(api, dy, one, 50, F32, padding=41) == 0).all()
    order = torch.randperm(n, generator=gen(n), device="cuda")
    got = check_gradient(api, dy, order, n, F32)
    assert torch.equal(got[order], dy)  # each a sum of one


@pytest.mark.parametrize("n,v", [(4096, 700), (4097, 700), (65536, 1 << 20), (65537, 3), (200000, 260000), (524289, 50000), (700000, 1 << 19)])
def test_gradient_of_many_tokens(api, n, v):
    # every size of the sort, one to three passes of it
    tokens, dy = words(n, v, n), normal((n, 8), F32, n)
    check_gradient(api, dy, tokens, v, F32, padding=1)
    check_gradient(api, dy[:, :3], (v - 1 - tokens).int(), v, F32)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 64, 65, 100])
@pytest.mark.parametrize("in_type,out_type", [(F32, F32), (F16, F32), (BF16, BF16)])
def test_gradient_of_few_tokens(api, n, in_type, out_type):
    for v, d in ((1, 2), (30, 3), (40, 515), (1000, 4096), (70, 20000)):
        tokens, dy = words(n, v + 3, n) - 1, normal((n, d), in_type, 5)  # (some are unknown)
        got = check_gradient(api, dy, tokens, v, out_type, 3.0)
        assert torch.equal(got, check_gradient(api, dy, tokens.int(), v, out_type, 3.0))
        check_gradient(api, dy, tokens, v, out_type, 0.5, padding=0, accumulate=True, out=normal((v, d), out_type, 3))
        check_gradient(api, dy, tokens, v, out_type, padding=v - 1)
    dy = normal((n, 170001), in_type, 6)  # one group of large pieces, from 99 tokens on
    check_gradient(api, dy, words(n, 5, n), 5, out_type)


@pytest.mark.parametrize("gap", [0, 4])
def test_gradient_of_few_tokens_into_a_large_table(api, gap):
    v, d = 140000, 1024
    table = torch.full((v, d + gap), 9.0, device="cuda")
    tokens, dy = torch.tensor([v - 1, 5, v, 0, 5, 70000], device="cuda"), normal((6, d), F32, 7)
    api.embedding_grad_into(wrap(api, table[:, :d]), wrap(api, dy), wrap(api, tokens), padding=0)
    assert torch.equal(table[[v - 1, 5, 70000], :d], torch.stack([dy[0], dy[1] + dy[4], dy[5]]))
    table[[v - 1, 5, 70000], :d] = 0
    assert not table[:, :d].any() and (table[:, d:] == 9).all()


def test_gradient_of_unknown_tokens(api):
    dy = normal((12, 40), F32, 1)
    tokens = torch.tensor([3, -1, 10, 9, 0, 1 << 40, -(1 << 40), (1 << 32) + 3, 5, 3, 1 << 31, 3], device="cuda")
    check_gradient(api, dy, tokens, 10, F32)
    check_gradient(api, dy, tokens, 10, F32, accumulate=True)
    small = torch.tensor([3, -1, 10, 9, 0, (1 << 31) - 1, -(1 << 31), 3, 5, 3, 11, 3], dtype=torch.int32, device="cuda")
    check_gradient(api, dy, small, 10, F32, padding=5)
    check_gradient(api, dy, small, 10, F32, padding=1 << 40)
    dy[1] = float("nan")  # an unknown token's gradient has no part in anything
    assert check_gradient(api, dy.nan_to_num(), small, 10, F32).equal(
        api.embedding_grad(api.as_tensor(dy), api.as_tensor(small), 10).torch())


@pytest.mark.parametrize("in_type,out_type", [(F32, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("d", [24, 515, 1024])
def test_gradient_between_rows_with_gaps(api, in_type, out_type, d):
    tokens = words(300, 40, 2).view(3, 100)
    wide = normal((3, 101, d + 3), in_type, 1)
    dy = wide[:, 1:, 1:d + 1]
    out = torch.full((40, d + 5), 9.0, dtype=out_type, device="cuda")
    check_gradient(api, dy, tokens, 40, out_type, out=out[:, 2:d + 2])
    assert (out[:, :2] == 9).all() and (out[:, d + 2:] == 9).all()
    dense = api.embedding_grad(wrap(api, dy.contiguous()), wrap(api, tokens.contiguous()), 40, dtype=out_type).torch()
    assert torch.equal(dense, out[:, 2:d + 2])


@pytest.mark.parametrize("n", [40, 3000, 30000])
def test_gradient_into_rows_at_two_distances(api, n):
    # a table of three parts with gaps between them: what is cleared ends where a part does
    for rows, d in ((50, 64), (7, 515), (2000, 32)):
        whole = torch.full((3, rows + 2, d), 9.0, device="cuda")
        table = whole[:, 1:rows + 1]
        tokens, dy = words(n, 3 * rows, n), normal((n, d), F32, 4)
        api.embedding_grad_into(wrap(api, table), wrap(api, dy), wrap(api, tokens))
        dense = api.embedding_grad(wrap(api, dy), wrap(api, tokens), 3 * rows).torch()
        assert torch.equal(table.reshape(3 * rows, d), dense) and (whole[:, 0] == 9).all() and (whole[:, -1] == 9).all()
        assert torch.equal(api.embedding(wrap(api, table), wrap(api, tokens)).torch(), dense[tokens])


@pytest.mark.parametrize("n", [1, 300, 5000])
def test_gradient_of_few_tokens_in_a_large_table(api, n):
    check_gradient(api, normal((n, 48), F32, n), words(n, 40000, n), 40000, F32)
    check_gradient(api, normal((n, 6), BF16, n), 39999 - words(n, 40000, n), 40000, BF16)


def test_gradient_of_what_is_not_finite(api):
    tokens = words(2000, 60, 2)
    dy = normal((2000, 48), F32, 1)
    clean = check_gradient(api, dy, tokens, 60, F32)
    at = int((tokens == 7).nonzero()[0, 0])
    dy[at, 5] = float("inf")
    got = api.embedding_grad(api.as_tensor(dy), api.as_tensor(tokens), 60).torch()
    assert got[7, 5] == float("inf")
    got[7, 5] = clean[7, 5]
    assert torch.equal(got, clean)


def test_gradient_is_the_same_in_every_call(api):
    tokens = words(30000, 5000, 2)
    dy = normal((30000, 100), BF16, 1)
    first = api.embedding_grad(api.as_tensor(dy), api.as_tensor(tokens), 5000, dtype=np.float32).torch().clone()
    for _ in range(3):
        assert torch.equal(first, api.embedding_grad(api.as_tensor(dy), api.as_tensor(tokens), 5000, dtype=np.float32).torch())


def test_gradient_beyond_four_gigabytes(api):
    v, d = 600000, 2048
    dy = normal((400, d), F32, 1)
    tokens = torch.cat([torch.arange(v - 100, v, device="cuda"), torch.arange(100, device="cuda")]).repeat(2)
    out = torch.full((v, d), 3.0, device="cuda")
    assert out.numel() * 4 > 1 << 32
    api.embedding_grad_into(api.as_tensor(out), api.as_tensor(dy), api.as_tensor(tokens))
    want = dy[:200] + dy[200:]
    assert torch.equal(out[-100:], want[:100]) and torch.equal(out[:100], want[100:])
    assert not out[100:-100].any()
    # and as many rows of the result's gradient
    del out
    n = 1100000
    many = torch.full((n,), 5, dtype=torch.int32, device="cuda")
    many[:-1000] = 1
    dy = torch.zeros((n, d), dtype=BF16, device="cuda")
    dy[-1000:] = normal((1000, d), BF16, 3)
    got = api.embedding_grad(api.as_tensor(dy), api.as_tensor(many), 6, dtype=np.float32).torch()
    ref.close(got[5], dy[-1000:].double().sum(0), 1002 * ref.U32 * dy[-1000:].double().abs().sum(0))
    assert not got[1].any()


def test_no_tokens(cv, api):
    table, none = cv.Tensor.from_numpy(np.ones((4, 8), np.float32), "NW"), cv.Tensor.alloc([0], np.int64, "W")
    rows = cv.Tensor.alloc([0, 8], np.float32, "NW")
    cv.Embedding()(None, table, none, rows)
    room = cv.Tensor.alloc([max(1, cv.EmbeddingGrad.workspace(0, 4, 8))], np.uint8, "W")
    cv.EmbeddingGrad()(None, rows, none, table, room, accumulate=True)
    torch.cuda.synchronize()
    assert (table.numpy() == 1).all()
    cv.EmbeddingGrad()(None, rows, none, table, room)
    torch.cuda.synchronize()
    assert (table.numpy() == 0).all()
    # a table without rows knows no token
    out = cv.Tensor.from_numpy(np.ones((3, 8), np.float32), "NW")
    cv.Embedding()(None, cv.Tensor.alloc([0, 8], np.float32, "NW"), cv.Tensor.from_numpy(np.zeros(3, np.int32), "W"), out)
    torch.cuda.synchronize()
    assert (out.numpy() == 0).all()


def test_gradient_against_differences(api):
    # L = sum(embedding(table) * r): linear in the table, so central differences are exact up to their roundings
    v, d, tokens = 7, 5, torch.tensor([3, 0, 3, 6, 3, 1], device="cuda")
    table, r = normal((v, d), F32, 1), normal((6, d), F32, 2)
    grad = api.embedding_grad(api.as_tensor(r), api.as_tensor(tokens), v, 1.5).torch()
    for i in range(v):
        for j in range(d):
            ends = []
            for h in (0.25, -0.25):
                moved = table.clone()
                moved[i, j] += h
                ends.append((api.embedding(api.as_tensor(moved), api.as_tensor(tokens), 1.5).torch().double() * r.double()).sum())
            # table + h and the lookup round: 4 * 2^-24 of values below 8, times three terms below 4 each
            assert abs(float((ends[0] - ends[1]) / 0.5 - grad[i, j])) < 4 * ref.U32 * 8 * 12 / 0.5


def test_another_stream_and_a_graph(api):
    tokens, dy = words(3000, 400, 1), normal((3000, 200), F32, 2)
    want = check_gradient(api, dy, tokens, 400, F32, 2.0, padding=3).clone()
    table = normal((400, 200), F32, 5)
    side = api.Stream()
    torch.cuda.synchronize()
    t_dy, t_tokens = api.as_tensor(dy), api.as_tensor(tokens)
    with side:
        got = api.embedding_grad(t_dy, t_tokens, 400, 2.0, padding=3)
        back = api.embedding(got, t_tokens)
    again = api.embedding(got, t_tokens)  # waits for the side stream
    torch.cuda.synchronize()
    assert torch.equal(got.torch(), want) and torch.equal(back.torch(), want[tokens]) and torch.equal(again.torch(), want[tokens])
    out, grad = torch.empty((3000, 200), device="cuda"), torch.empty((400, 200), device="cuda")
    size = api.EmbeddingGrad.workspace(3000, 400, 200)
    room = api.as_tensor(torch.empty(size, dtype=torch.uint8, device="cuda")) if size else None
    t = [api.as_tensor(x) for x in (out, table, grad)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = api.as_stream(torch.cuda.current_stream())
        api.embedding_into(t[0], t[1], t_tokens, stream=s)
        api.embedding_grad_into(t[2], t[0], t_tokens, 2.0, padding=3, workspace=room, stream=s)
    for k in range(4):
        tokens.copy_(words(3000, 400, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, table[tokens])
        assert torch.equal(grad, check_gradient(api, out, tokens, 400, F32, 2.0, padding=3))
