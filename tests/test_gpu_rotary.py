"""cvcudaxRotarySubmit against its definition in 64 bits (head_reference.py derives the bounds)."""
import importlib

import numpy as np
import pytest
import torch

import head_reference as ref
from row_reference import close

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LONG = dict(factor=8.0, original=8192.0, low=1.0, high=4.0, magnitude=1.1)


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


def random(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def places(n, seed, dtype=torch.int64, most=131072):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, most, (n,), generator=g, device="cuda").to(dtype)


def run(api, x, positions, dims, out=None, scaling=None, **how):
    out = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") if out is None else out
    scaling = None if scaling is None else api.RotaryScaling(**scaling)
    api.rotary_into(api.as_tensor(out, "TWE"), api.as_tensor(x, "TWE"), api.as_tensor(positions), dims, scaling=scaling, **how)
    return out


def check(api, x, positions, dims, scaling=None, out=None, **how):
    got = run(api, x, positions, dims, scaling=scaling, out=out, **how)
    want, error = ref.rotary(x.double(), positions, dims, **dict(scaling or {}, **how))
    close(got[..., :dims], want[..., :dims], error[..., :dims])
    assert torch.equal(got[..., dims:], x[..., dims:])
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,dims", [(2, 2), (3, 2), (6, 6), (7, 4), (16, 16), (50, 50), (64, 24), (64, 64), (80, 80), (96, 32), (100, 36), (128, 128),
                                    (129, 128), (256, 256), (300, 256)])
def test_heads(api, d, dims, interleaved, dtype):
    for n, heads in ((1, 1), (5, 3), (33, 40)):
        x, positions = random((n, heads, d), dtype, d + n), places(n, n)
        check(api, x, positions, dims, interleaved=interleaved)
        check(api, x, positions.int(), dims, interleaved=interleaved, inverse=True, scaling=LONG)


@pytest.mark.parametrize("interleaved", [True, False])
def test_far_and_negative_positions(api, interleaved):
    """Nothing of an angle is lost with whole turns, in 32 bits either."""
    positions = torch.tensor([0, 1, -1, 2, 4095, 65537, 1000003, -1000003, (1 << 24) + 1, (1 << 31) - 1], device="cuda")
    x = random((10, 2, 64), F32, 1)
    for base in (10000.0, 500000.0, 1.5):
        check(api, x, positions, 64, interleaved=interleaved, base=base)
        check(api, x, positions.int(), 64, interleaved=interleaved, base=base, scaling=dict(factor=4.0))
    out = run(api, x[:1], positions[:1], 64)
    assert torch.equal(out, x[:1])  # position 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_heads_with_gaps_and_in_place(api, interleaved, dtype):
    wide = random((20, 7, 75), dtype, 2)
    positions = places(20, 3)
    x = wide[:, 1:5, 3:67]  # queries of one projection's result, rows that begin between 4-byte words
    keep, out = wide.clone(), torch.full((20, 6, 70), 9.0, dtype=dtype, device="cuda")
    got = check(api, x, positions, 40, interleaved=interleaved, out=out[:, 2:, 1:65])
    assert torch.equal(wide, keep) and (out[:, :2] == 9).all() and (out[..., :1] == 9).all() and (out[..., 65:] == 9).all()
    run(api, x, positions, 40, out=x, interleaved=interleaved)
    assert torch.equal(x, got)
    x.copy_(keep[:, 1:5, 3:67])
    assert torch.equal(wide, keep)


@pytest.mark.parametrize("interleaved", [True, False])
def test_turned_back(api, interleaved):
    """The gradient: what was turned and is turned back is what it was, to four roundings of 32 bits in each element of a pair."""
    x, positions = random((200, 8, 128), F32, 4), places(200, 5)
    there = run(api, x, positions, 128, interleaved=interleaved)
    back = run(api, there, positions, 128, interleaved=interleaved, inverse=True)
    assert ((back - x).abs() <= 32 * ref.U32 * x.abs().amax()).all()


def test_more_than_four_gigabytes(api):
    x = torch.zeros((140000, 64, 256), dtype=BF16, device="cuda")
    assert x.numel() > 1 << 31
    positions = places(140000, 6)
    x[-50:] = random((50, 64, 256), BF16, 7)
    out = run(api, x, positions, 256)
    want, error = ref.rotary(x[-50:].double(), positions[-50:], 256)
    close(out[-50:], want, error)
    assert (out[:-50] == 0).all()


def test_what_is_not_finite_stays_in_its_pair(api):
    x, positions = random((3, 2, 64), F32, 8), places(3, 9)
    clean = run(api, x, positions, 64)
    x[1, 1, 5] = float("nan")
    got = run(api, x, positions, 64)
    others = torch.ones_like(x, dtype=torch.bool)
    others[1, 1, 5] = others[1, 1, 37] = False
    assert torch.equal(got[others], clean[others]) and got[1, 1, 5].isnan() and got[1, 1, 37].isnan()


def test_another_stream_and_a_graph(api):
    x, positions = random((500, 8, 64), F16, 10), places(500, 11)
    want, back = run(api, x, positions, 64), run(api, x, positions, 64, inverse=True)
    side, tx, tp = api.Stream(), api.as_tensor(x), api.as_tensor(positions)
    first = api.rotary(tx, tp)
    with side:
        second = api.rotary(first, tp, inverse=True)
    torch.cuda.synchronize()
    assert torch.equal(first.torch(), want) and torch.equal(second.torch(), run(api, want, positions, 64, inverse=True))
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(x)
    to = api.as_tensor(out)
    with torch.cuda.graph(graph):
        api.rotary_into(to, tx, tp, inverse=True, stream=api.as_stream(torch.cuda.current_stream()))
    for turn in range(3):
        positions.copy_(places(500, 20 + turn))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.clone(), run(api, x, positions, 64, inverse=True))
    assert back.isfinite().all()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,n,d,dims", [(F32, 9000, 129, 128), (BF16, 12000, 100, 36), (F16, 12000, 128, 128), (F32, 9000, 66, 62)])
def test_many_tokens(api, dtype, n, d, dims, interleaved):
    """More than the card keeps near its memory."""
    x, positions = random((n, 32, d), dtype, 16), places(n, 17)
    assert 2 * x.numel() * x.element_size() > 128 << 20
    got = check(api, x, positions, dims, interleaved=interleaved)
    assert torch.equal(run(api, x, positions, dims, out=x, interleaved=interleaved), got)
