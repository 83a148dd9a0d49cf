"""The row operators' calls by native code do what pyapi._submit does, and torch tensors wrapped by native code are what
Python makes of them."""
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


def calls(api):
    """(call, its results) of every form, on fresh tensors."""
    g = torch.Generator(device="cuda").manual_seed(1)

    def t(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    wrap = api.as_tensor
    x, dy, gamma, beta = wrap(t(7, 40)), wrap(t(7, 40)), wrap(t(40)), wrap(t(40))
    out, mean, rstd, dx, dg, db = (wrap(t(*s)) for s in ((7, 40), (7,), (7,), (7, 40), (40,), (40,)))
    table, tokens, rows, grad = wrap(t(9, 40)), wrap(torch.arange(7, device="cuda") % 3), wrap(t(7, 40)), wrap(t(9, 40))
    stats = wrap(t(7)), wrap(t(7))
    many = lambda *sizes, **kw: [wrap(t(n, **kw)) for n in sizes]
    p, m, v, q = many(300, 5), many(300, 5), [wrap(t(n).abs()) for n in (300, 5)], many(300, 5, dtype=torch.bfloat16)
    copies = [wrap(t(300, dtype=torch.float16)), None]
    codes = [wrap(torch.randint(-127, 128, (n,), generator=g, device="cuda").to(torch.int8)) for n in (300, 5)]
    squares = [wrap(torch.randint(0, 256, (n,), generator=g, device="cuda").to(torch.uint8)) for n in (300, 5)]
    scales = [[wrap(t(n).abs()) for n in (2, 1)] for _ in range(2)]
    p2, factor, values = many(300, 5), wrap(t(1)), many(300, 5)
    return [
        (lambda: api.layer_norm_into(out, x, gamma, beta, mean=mean, rstd=rstd), [out, mean, rstd]),
        (lambda: api.layer_norm_into(out, x), [out]),
        (lambda: api.layer_norm_grad_into(dx, dg, db, dy, x, gamma, *stats), [dx, dg, db]),
        (lambda: api.layer_norm_grad_into(dx, None, None, dy, x, None, *stats), [dx]),
        (lambda: api.embedding_into(rows, table, tokens, 2.0), [rows]),
        (lambda: api.embedding_grad_into(grad, dy, tokens, 2.0, padding=1, accumulate=True), [grad]),
        (lambda: api.embedding_grad_into(grad, dy, tokens), [grad]),
        (lambda: api.adamw_into(p, m, v, q, 3, copies=copies), p + m + v + copies[:1]),
        (lambda: api.adamw_into(p2, codes, squares, q, 3, moment_scales=scales[0], variance_scales=scales[1], grad_scale=factor),
         p2 + codes + squares + scales[0] + scales[1]),
        (lambda: api.adamw_unpack_into(values, codes, scales[0]), values),
    ]


def test_native_calls_do_what_submit_does(api, monkeypatch):
    python = _Python(api)
    for (native, got), (other, want) in zip(calls(api), calls(api)):
        handed_on = []
        monkeypatch.setattr(api, "_submit", lambda *a: handed_on.append(a))
        native()
        monkeypatch.undo()
        assert not handed_on
        assert all(t._wrote == (0, None) and t._read == {} for t in got)
        monkeypatch.setattr(api, "_run", python)
        other()
        monkeypatch.undo()
        torch.cuda.synchronize()
        assert all(torch.equal(a.torch(), b.torch()) for a, b in zip(got, want))
    assert python.calls == 10


def test_marks_that_stand_and_others(api):
    x, out, other = (api.as_tensor(torch.randn(64, 512, device="cuda")) for _ in range(3))
    for _ in range(3):  # the second time the first one's marks stand
        api.layer_norm_into(out, x)
        assert out._wrote == (0, None) and out._read == {} and x._read == {0: None}
    api.layer_norm_into(other, out)
    assert out._wrote == (0, None) and out._read == {0: None}
    api.layer_norm_into(out, x)  # a read of what is written: the marks do not stand
    assert out._wrote == (0, None) and out._read == {} and x._read == {0: None}
    s = api.Stream()
    api.layer_norm_into(out, other, stream=s)
    assert out._wrote[0] == s.handle != 0 and set(other._read) == {s.handle}
    api.layer_norm_into(other, out)  # waits for that
    assert other._wrote[0] == 0 and other._read == {} and set(out._read) == {0}
    torch.cuda.synchronize()
    want = torch.nn.functional.layer_norm(x.torch(), (512,))
    assert (out.torch() - torch.nn.functional.layer_norm(want, (512,))).abs().max() < 1e-4


class _Python:
    def __init__(self, api):
        self.submit, self.calls = api._submit, 0

    def __call__(self, *args):
        self.calls += 1
        self.submit(*args)


def test_what_native_calls_raise(api, cv):
    x, y = api.as_tensor(torch.zeros(4, 8, device="cuda")), api.as_tensor(torch.zeros(4, 9, device="cuda"))
    for call in (lambda: api.layer_norm_into(y, x), lambda: api.embedding_into(y, x, x), lambda: api.adamw_into([x], [x], [x], [y], 1),
                 lambda: api.adamw_into([x], [x], [x], [x], 0), lambda: api.adamw_into([x], [x], [x], [x], 1, copies=[y])):
        with pytest.raises(cv.Error) as e:
            call()
        assert e.value.status == 2


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.float16, torch.bfloat16,
                                   torch.float32, torch.float64, torch.complex64])
def test_wrapped_torch_tensors(api, cv, dtype):
    x = torch.arange(60, device="cuda").reshape(3, 4, 5).to(dtype)
    for t, layout in ((x, None), (x[:, 1:], "HWC"), (x[0], "NW"), (torch.nn.Parameter(x, requires_grad=False), None)):
        a, b = api.as_tensor(t, layout), api.Tensor(_wrap=cv.Tensor.from_torch(t, layout or ""))
        assert a.shape == b.shape == tuple(t.shape) and a.dtype == b.dtype and a.layout == b.layout == layout and a._t.strides == b._t.strides
        assert a._t.dtype == b._t.dtype and a._t._keep == [t]
        assert torch.equal(a.torch(), t) and torch.equal(b.torch(), t) and a.torch().dtype == dtype and a.torch().data_ptr() == t.data_ptr()
        handle = a._t
        assert handle.refcount() == 1
        del a
        handle.close()


def test_wrapped_tensors_go(api, cv):
    import weakref
    x = torch.zeros(4, 8, device="cuda")
    kept, a, b = weakref.ref(x), api.as_tensor(x), api.as_tensor(x)
    raw = a._t
    del x, a
    assert raw.refcount() == 1 and kept() is not None
    raw.close()  # once; as it goes there is nothing left to give back
    assert raw.handle is None
    del raw
    assert kept() is not None
    del b
    assert kept() is None


def test_results_come_back(api):
    made = api.layer_norm(api.as_tensor(torch.ones(4, 8, device="cuda")))
    raw = made._t
    del made
    again = api.layer_norm(api.as_tensor(torch.ones(4, 8, device="cuda")))
    assert again._t is raw
    again.torch()  # seen: it does not come back
    del again
    assert api.layer_norm(api.as_tensor(torch.ones(4, 8, device="cuda")))._t is not raw


def test_what_cannot_be_wrapped(api, cv):
    with pytest.raises(cv.Error) as e:
        api.as_tensor(torch.zeros(4, 8, device="cuda").t())  # its rows' elements do not follow one another
    assert e.value.status == 2
    with pytest.raises(cv.Error):
        api.as_tensor(torch.zeros(0, 8, device="cuda"))
    with pytest.raises(cv.Error):
        api.as_tensor(torch.zeros(4, 8, device="cuda"), "NHWC")
    with pytest.raises(TypeError):
        api.as_tensor(torch.zeros(4, dtype=torch.bfloat16, device="cuda")).cuda()  # the array interface has no name for it


def test_captured_gradients(api, cv):
    """With a workspace of the caller's, which the calls take that make their results too; refused without one, and the capture goes on."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, d, v = 4096, 96, 500
    x, dy = (torch.randn((rows, d), generator=g, device="cuda") for _ in range(2))
    mean, rstd, gamma = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda"), torch.ones(d, device="cuda")
    tokens = torch.randint(0, v, (rows,), generator=g, device="cuda")
    wrap = api.as_tensor
    made = [torch.empty(s, device="cuda") for s in ((rows, d), (d,), (d,), (v, d), (v, d))]
    sizes = api.LayerNormGrad.workspace(rows, d), api.EmbeddingGrad.workspace(rows, v, d)
    rooms, others = ([wrap(torch.empty(n, dtype=torch.uint8, device="cuda")) for n in sizes] for _ in range(2))
    dx, dg, db, table, few = map(wrap, made)
    tx, tdy, tgamma, tmean, trstd, ttokens, tfew, ttfew = map(wrap, (x, dy, gamma, mean, rstd, tokens, dy[:64], tokens[:64]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: api.layer_norm_grad_into(dx, dg, db, tdy, tx, tgamma, tmean, trstd), lambda: api.layer_norm_grad(tdy, tx, tgamma, tmean, trstd),
                     lambda: api.embedding_grad_into(table, tdy, ttokens), lambda: api.embedding_grad(tdy, ttokens, v)):
            with pytest.raises(cv.Error) as e:
                call()
            assert e.value.status == 4
        api.layer_norm_grad_into(dx, dg, db, tdy, tx, tgamma, tmean, trstd, workspace=rooms[0])
        api.embedding_grad_into(table, tdy, ttokens, workspace=rooms[1])
        api.embedding_grad_into(few, tfew, ttfew)  # needs none
    for _ in range(4):
        dy.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in made]
        want = [*api.layer_norm_grad(tdy, tx, tgamma, tmean, trstd, workspace=others[0]), api.embedding_grad(tdy, ttokens, v, workspace=others[1]),
                api.embedding_grad(tfew, ttfew, v)]
        assert all(torch.equal(a, b.torch()) for a, b in zip(got, want))


def test_gradients_of_few_rows_make_no_workspace(api, monkeypatch):
    """On any stream, and captured: the least workspace, which is not touched, is one tensor for all calls and carries no marks."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, d = 256, 768
    x, dy = (torch.randn((rows, d), generator=g, device="cuda") for _ in range(2))
    mean, rstd, gamma = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda"), torch.ones(d, device="cuda")
    made = [torch.empty(s, device="cuda") for s in ((rows, d), (d,), (d,))]
    wrap = lambda: [api.as_tensor(t) for t in (*made, dy, x, gamma, mean, rstd)]

    def none(*args):
        raise AssertionError("a result of %s" % (args,))

    monkeypatch.setattr(api, "_result", none)
    results = []
    api.layer_norm_grad_into(*wrap())
    room = api._untouched_workspace()
    results.append([t.clone() for t in made])
    torch.cuda.synchronize()
    api.layer_norm_grad_into(*wrap(), stream=api.Stream())
    torch.cuda.synchronize()
    results.append([t.clone() for t in made])
    graph, captured = torch.cuda.CUDAGraph(), wrap()
    with torch.cuda.graph(graph):
        api.layer_norm_grad_into(*captured)
    for _ in range(3):
        for t in made:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        results.append([t.clone() for t in made])
    assert all(torch.equal(a, b) for got in results for a, b in zip(got, results[0]))
    assert api._untouched_workspace() is room and not hasattr(room, "_wrote") and not hasattr(room, "_read")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_results_of_every_type_come_back(api, monkeypatch, dtype):
    made, new = [], api._new_result
    monkeypatch.setattr(api, "_new_result", lambda *args: made.append(args) or new(*args))
    x, stats, gamma = (api.as_tensor(torch.ones(s, dtype=t, device="cuda")) for s, t in (((40, 24), dtype), (40, torch.float32), (24, dtype)))
    tokens = api.as_tensor(torch.arange(40, device="cuda") % 7)
    for _ in range(50):
        api.layer_norm(api.layer_norm(x))
        api.embedding(x, tokens)
        api.layer_norm_grad(x, x, gamma, stats, stats)
        api.embedding_grad(x, tokens, 9)
    # (40, 24) twice at a time, two of (24,), one of (9, 24)
    assert sorted(tuple(m[0]) for m in made) == [(9, 24), (24,), (24,), (40, 24), (40, 24)]
    torch.cuda.synchronize()


class _Between:
    """The marks' lock; once, when it is given back the first time, another call runs: where another thread's may, after a call
    has looked at the marks it found and before it is submitted."""

    def __init__(self, lock, call):
        self.lock, self.call = lock, call

    def acquire(self, blocking=True):
        return self.lock.acquire(blocking)

    def release(self):
        self.lock.release()
        if self.call is not None:
            call, self.call = self.call, None
            call()

    def __enter__(self):
        self.acquire()

    def __exit__(self, *exc):
        self.release()


def test_marks_that_another_call_sets_meanwhile(api, monkeypatch):
    """A call whose marks stood when it looked leaves its own behind another's that came between: what follows on that one's stream
    waits for it. (The other call's operator does nothing, so that nothing is written twice at a time.)"""
    x, out = (api.as_tensor(torch.randn(64, 512, device="cuda")) for _ in range(2))
    s = api.Stream()
    for reads, writes in (([], [out]), ([], [x])):
        for _ in range(2):
            api.layer_norm_into(out, x)
        monkeypatch.setattr(api, "_followed", {})
        lock = _Between(api._events_lock, lambda: api._submit(s, reads, writes, lambda *args: None))
        monkeypatch.setattr(api, "_events_lock", lock)
        api.layer_norm_into(out, x)
        monkeypatch.undo()
        assert lock.call is None
        assert out._wrote == (0, None) and out._read == {} and x._read[0] is None
        monkeypatch.setattr(api, "_followed", {})
        torch.cuda.synchronize()
        x, out = api.as_tensor(x.torch()), api.as_tensor(out.torch())


def test_what_is_captured(api):
    """Streams that are captured, however they are given, and others beside them."""
    side, other = api.Stream(), torch.cuda.Stream()
    assert not any(api._capturing(s) for s in (None, side, other, api.Stream.default, api.as_stream(other.cuda_stream)))
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=other):
        x.add_(1)
        got = [api._capturing(s) for s in (None, other, api.as_stream(other), api.as_stream(other.cuda_stream), side)]
        with side:
            got.append(api._capturing(None))
        with api.as_stream(other):
            got.append(api._capturing(None))
    assert got == [True, True, True, True, False, False, True] and not api._capturing(other)
