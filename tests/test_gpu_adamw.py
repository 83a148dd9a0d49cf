"""cvcudaxAdamWSubmit: 32-bit states against the definition in 64 bits, and the bits of the documented order of operations
against numpy on the host, where each of them is rounded by itself (elementary float32 arithmetic and square roots)."""
import importlib
import math

import numpy as np
import pytest
import torch

import row_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
BLOCK = 256
HYPER = dict(lr=3e-3, betas=(0.9, 0.97), epsilon=1e-8, weight_decay=0.05)


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})  # (a wait for the default stream has the calls after it record events)


# ---- the same steps on the host ----------------------------------------------------------------------------------------
f = np.float32


def decode_moment(q, scale):
    t = q.astype(f) * f(1 / 127)
    return t * np.abs(t) * np.repeat(scale, BLOCK)[:q.size]


def decode_variance(q, scale):
    t = q.astype(f) * f(1 / 255)
    t = t * t
    return t * t * np.repeat(scale, BLOCK)[:q.size]


def blocks(x):
    out = np.zeros((-(-x.size // BLOCK), BLOCK), f)
    out.reshape(-1)[:x.size] = x
    return out


def share(b, scale):
    with np.errstate(all="ignore"):
        return np.where(scale[:, None] > 0, b / scale[:, None], f(0)).astype(f)


def encode_moment(m):
    b = blocks(m)
    scale = np.abs(b).max(1)
    q = np.rint(np.sqrt(share(np.abs(b), scale)) * f(127)) * np.sign(b)
    return q.astype(np.int8).reshape(-1)[:m.size], scale


def encode_variance(v):
    b = blocks(v)
    scale = b.max(1)
    q = np.maximum(np.rint(np.sqrt(np.sqrt(share(b, scale))) * f(255)), (b > 0).astype(f))
    return q.astype(np.uint8).reshape(-1)[:v.size], scale


def host_step(p, m, v, g, t, lr, betas, epsilon, weight_decay):
    b1, b2 = betas
    m = f(b1) * m + g * f(1 - b1)
    v = f(b2) * v + g * f(1 - b2) * g
    root = np.sqrt(v) * f(1 / math.sqrt(1 - b2 ** t)) + f(epsilon)
    return p * f(1 - lr * weight_decay) - m / root * f(lr / (1 - b1 ** t)), m, v


# ---- tensors -----------------------------------------------------------------------------------------------------------
def made(n, seed, scale):
    return (np.random.default_rng(seed).standard_normal(n) * scale).astype(f)


def device(x, dtype=F32):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(dtype)


def step(api, p, m, v, g, t, copies=None, scales=None, grad_scale=None, stream=None, **hyper):
    wrap = lambda part: None if part is None else [None if x is None else api.as_tensor(x) for x in part]
    api.adamw_into(wrap(p), wrap(m), wrap(v), wrap(g), t, copies=wrap(copies), moment_scales=wrap(scales[0]) if scales else None,
                   variance_scales=wrap(scales[1]) if scales else None, grad_scale=None if grad_scale is None else api.as_tensor(grad_scale),
                   stream=stream, **{**HYPER, **hyper})


SIZES = [1, 2, 255, 256, 257, 1000, 4096, 5001, 1 << 16, 3, 100003]


@pytest.mark.parametrize("param,grad,copy", [(F32, F32, None), (F32, BF16, BF16), (F32, F16, F16), (BF16, BF16, None), (F16, F32, BF16)])
def test_states_of_32_bits(api, param, grad, copy):
    p = [device(made(n, k, 0.1), param) for k, n in enumerate(SIZES)]
    g = [device(made(n, 50 + k, 1e-3), grad) for k, n in enumerate(SIZES)]
    m, v = [torch.zeros(n, device="cuda") for n in SIZES], [torch.zeros(n, device="cuda") for n in SIZES]
    copies = [torch.zeros(n, dtype=copy, device="cuda") for n in SIZES] if copy else None
    for t in (1, 2, 3):
        before = [(a.double(), b.double(), c.double(), d.double()) for a, b, c, d in zip(p, m, v, g)]
        host = [host_step(*(x.float().cpu().numpy() for x in part), t, **HYPER) for part in zip(p, m, v, g)]
        step(api, p, m, v, g, t, copies)
        b1, b2 = HYPER["betas"]
        for k, (pd, md, vd, gd) in enumerate(before):
            assert np.array_equal(m[k].cpu().numpy(), host[k][1]) and np.array_equal(v[k].cpu().numpy(), host[k][2])
            assert torch.equal(p[k].cpu(), torch.from_numpy(host[k][0]).to(param))
            if copy:
                assert torch.equal(copies[k].cpu(), torch.from_numpy(host[k][0]).to(copy))
            # against the definition: 4 roundings in m and v, 8 in the step
            em, ev = b1 * md + (1 - b1) * gd, b2 * vd + (1 - b2) * gd * gd
            ref.close(m[k], em, 4 * ref.U32 * (b1 * md.abs() + (1 - b1) * gd.abs()))
            ref.close(v[k], ev, 6 * ref.U32 * ev + ref.STEP[F32] * 4)
            change = HYPER["lr"] * (em / (1 - b1 ** t)) / ((ev / (1 - b2 ** t)).sqrt() + HYPER["epsilon"])
            e_change = HYPER["lr"] / (1 - b1 ** t) * 4 * ref.U32 * (b1 * md.abs() + (1 - b1) * gd.abs()) / ((ev / (1 - b2 ** t)).sqrt() + HYPER["epsilon"])
            ref.close(p[k], pd * (1 - HYPER["lr"] * HYPER["weight_decay"]) - change, 3 * ref.U32 * pd.abs() + 12 * ref.U32 * change.abs() + e_change)


@pytest.mark.parametrize("param,grad", [(F32, F32), (F32, BF16), (F16, F16)])
def test_states_of_8_bits(api, param, grad):
    p = [device(made(n, k, 0.1), param) for k, n in enumerate(SIZES)]
    m, v = [torch.zeros(n, dtype=torch.int8, device="cuda") for n in SIZES], [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in SIZES]
    scales = [[torch.zeros(-(-n // BLOCK), device="cuda") for n in SIZES] for _ in range(2)]
    for t in (1, 2, 3):
        g = [device(made(n, 50 * t + k, 1e-3), grad) for k, n in enumerate(SIZES)]
        before = [tuple(x.cpu().numpy() for x in part) for part in zip(m, v, scales[0], scales[1])]
        host = [host_step(a.float().cpu().numpy(), decode_moment(q, s), decode_variance(u, r), d.float().cpu().numpy(), t, **HYPER)
                for (q, u, s, r), a, d in zip(before, p, g)]
        step(api, p, m, v, g, t, scales=scales)
        for k, (hp, hm, hv) in enumerate(host):
            assert torch.equal(p[k].cpu(), torch.from_numpy(hp).to(param))
            for state, scale, (codes, largest) in ((m, scales[0], encode_moment(hm)), (v, scales[1], encode_variance(hv))):
                assert np.array_equal(scale[k].cpu().numpy(), largest) and np.array_equal(state[k].cpu().numpy(), codes)
            # what the codes stand for is near what they were made from: half a step of the root at q
            hm64, top = hm.astype(np.float64), np.repeat(scales[0][k].cpu().numpy().astype(np.float64), BLOCK)[:hm.size]
            root = np.sqrt(np.abs(hm64) / np.maximum(top, 1e-300))
            got = decode_moment(m[k].cpu().numpy(), scales[0][k].cpu().numpy())
            assert (np.abs(got - hm64) <= top * ((root + 0.5 / 127) ** 2 - root ** 2) * (1 + 1e-5)).all()
            assert ((v[k].cpu().numpy() > 0) == (hv > 0)).all()
    for state, scale, decode in ((m, scales[0], decode_moment), (v, scales[1], decode_variance)):
        out = [torch.full((n,), 3.0, device="cuda") for n in SIZES]
        api.adamw_unpack_into([api.as_tensor(x) for x in out], [api.as_tensor(x) for x in state], [api.as_tensor(x) for x in scale])
        for o, q, s in zip(out, state, scale):
            assert np.array_equal(o.cpu().numpy(), decode(q.cpu().numpy(), s.cpu().numpy()))


@pytest.mark.parametrize("small", [False, True])
def test_more_tensors_than_a_launch_takes(api, small):
    sizes = [1 + (k * 37) % 700 for k in range(400)]
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    p, g = device(made(offsets[-1], 1, 0.1)), device(made(offsets[-1], 2, 1e-3), BF16)
    cut = lambda x: [x[a:b] for a, b in zip(offsets[:-1], offsets[1:])]  # tensors that follow one another, at any alignment
    want = p.cpu().numpy().copy()
    m, v = (torch.zeros(offsets[-1], dtype=d, device="cuda") for d in ((torch.int8, torch.uint8) if small else (F32, F32)))
    scales = [[torch.zeros(-(-n // BLOCK), device="cuda") for n in sizes] for _ in range(2)] if small else None
    step(api, cut(p), cut(m), cut(v), cut(g), 1, scales=scales)
    hp, hm, hv = host_step(want, np.zeros_like(want), np.zeros_like(want), g.float().cpu().numpy(), 1, **HYPER)
    assert np.array_equal(p.cpu().numpy(), hp)
    if small:
        assert all(np.array_equal(x.cpu().numpy(), encode_moment(y)[0]) for x, y in zip(cut(m), cut(hm)))
        assert all(np.array_equal(x.cpu().numpy(), encode_variance(y)[0]) for x, y in zip(cut(v), cut(hv)))
    else:
        assert np.array_equal(m.cpu().numpy(), hm) and np.array_equal(v.cpu().numpy(), hv)


@pytest.mark.parametrize("small", [False, True])
def test_scaled_gradients_and_copies_of_some(api, small):
    sizes = [300, 1000, 77]
    p, g = [device(made(n, k, 0.1)) for k, n in enumerate(sizes)], [device(made(n, 9 + k, 1e-3), d) for k, (n, d) in enumerate(zip(sizes, (F32, BF16, F16)))]
    host_p, factor = [x.cpu().numpy() for x in p], f(0.37)
    m, v = ([torch.zeros(n, dtype=d, device="cuda") for n in sizes] for d in ((torch.int8, torch.uint8) if small else (F32, F32)))
    scales = [[torch.zeros(-(-n // BLOCK), device="cuda") for n in sizes] for _ in range(2)] if small else None
    copies = [torch.zeros(300, dtype=BF16, device="cuda"), None, torch.zeros(77, dtype=F16, device="cuda")]
    step(api, p, m, v, g, 4, copies, scales, torch.tensor([0.37], device="cuda"))
    for k, n in enumerate(sizes):
        hp, _, _ = host_step(host_p[k], np.zeros(n, f), np.zeros(n, f), g[k].float().cpu().numpy() * factor, 4, **HYPER)
        assert np.array_equal(p[k].cpu().numpy(), hp)
        if copies[k] is not None:
            assert torch.equal(copies[k].cpu(), torch.from_numpy(hp).to(copies[k].dtype))


def test_blocks_of_zeros_and_what_is_not_finite(api):
    n = 5 * BLOCK + 10
    g = made(n, 1, 1e-3)
    g[BLOCK:2 * BLOCK] = 0
    g[2 * BLOCK + 3], g[3 * BLOCK + 200] = np.nan, np.inf
    g[4 * BLOCK] = 1e-22  # its square is below every float
    p, m, v = device(made(n, 2, 0.1)), torch.zeros(n, dtype=torch.int8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    scales = [[torch.zeros(6, device="cuda")] for _ in range(2)]
    before = p.cpu().numpy()
    step(api, [p], [m], [v], [device(g)], 1, scales=scales)
    with np.errstate(all="ignore"):
        hp, hm, hv = host_step(before, np.zeros(n, f), np.zeros(n, f), g, 1, **HYPER)
    got = p.cpu().numpy()
    assert np.array_equal(got, hp, equal_nan=True) and np.isnan(got).sum() == 2
    assert np.array_equal(got[BLOCK:2 * BLOCK], before[BLOCK:2 * BLOCK] * f(1 - HYPER["lr"] * HYPER["weight_decay"]))
    assert not m[BLOCK:2 * BLOCK].any() and not v[BLOCK:2 * BLOCK].any()
    values = [torch.zeros(n, device="cuda") for _ in range(2)]
    for out, q, s in ((values[0], m, scales[0]), (values[1], v, scales[1])):
        api.adamw_unpack_into([api.as_tensor(out)], [api.as_tensor(q)], [api.as_tensor(s[0])])
        for b in range(6):
            part = out[b * BLOCK:(b + 1) * BLOCK]
            assert part.isnan().all() if b in (2, 3) else part.isfinite().all()


def test_no_tensors_and_empty_ones(cv, api):
    api.adamw_into([], [], [], [], 1)
    api.adamw_unpack_into([], [], [])
    empty = [cv.Tensor.alloc([0], np.float32, "W") for _ in range(4)]
    one = [cv.Tensor.from_numpy(np.full(3, 0.5, np.float32), "W") for _ in range(4)]
    cv.AdamW()(None, *[[a, b, a] for a, b in zip(empty, one)], None, None, None, None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)
    torch.cuda.synchronize()
    hp, _, _ = host_step(*(np.full(3, 0.5, f) for _ in range(4)), 1, 1e-3, (0.9, 0.999), 1e-8, 0.01)
    assert np.array_equal(one[0].numpy(), hp)


def test_a_tensor_beyond_four_gigabytes(api):
    n = (1 << 30) + 1000
    p, m, v, g = (torch.zeros(n, device="cuda") for _ in range(4))
    p[-1000:], g[-1000:] = device(made(1000, 1, 0.1)), device(made(1000, 2, 1e-3))
    before = p[-1000:].cpu().numpy()
    step(api, [p], [m], [v], [g], 1)
    hp, hm, hv = host_step(before, np.zeros(1000, f), np.zeros(1000, f), g[-1000:].cpu().numpy(), 1, **HYPER)
    assert np.array_equal(p[-1000:].cpu().numpy(), hp) and np.array_equal(m[-1000:].cpu().numpy(), hm)
    assert np.array_equal(v[-1000:].cpu().numpy(), hv) and not p[:-1000].any()


def test_another_stream_and_a_graph(api):
    n = 200000
    p, g = device(made(n, 1, 0.1)), device(made(n, 2, 1e-3))
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    want = p.cpu().numpy(), np.zeros(n, f), np.zeros(n, f)
    side, t = api.Stream(), [api.as_tensor(x) for x in (p, m, v, g)]
    torch.cuda.synchronize()
    for k in range(1, 5):  # in turn on two streams, each waits for the other
        api.adamw_into([t[0]], [t[1]], [t[2]], [t[3]], k, stream=side if k % 2 else None, **HYPER)
        want = host_step(*want, g.cpu().numpy(), k, **HYPER)
    torch.cuda.synchronize()
    assert np.array_equal(p.cpu().numpy(), want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.adamw_into([t[0]], [t[1]], [t[2]], [t[3]], 9, stream=api.as_stream(torch.cuda.current_stream()), **HYPER)
    for k in range(4):
        g.copy_(device(made(n, 30 + k, 1e-3)))
        graph.replay()
        torch.cuda.synchronize()
        want = host_step(*want, g.cpu().numpy(), 9, **HYPER)
        assert np.array_equal(p.cpu().numpy(), want[0]) and np.array_equal(m.cpu().numpy(), want[1])
