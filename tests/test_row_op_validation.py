"""What the operators on rows of values (cvcuda/LayerNorm.h, Embedding.h, AdamW.h) refuse, on the CPU: tensors wrap a made-up
device address, every case is rejected on the host before any launch."""
import ctypes as C
import importlib

import numpy as np
import pytest
import torch

INVALID_ARGUMENT, NOT_COMPATIBLE = 2, 9
FAKE = 0x7F0000000000
F32, F16, BF16 = np.float32, np.float16, torch.bfloat16


def fake(cv, shape, dtype=F32, layout="", strides=None, at=FAKE):
    """Tensor over a made-up address; strides in elements (packed ones when not given)."""
    es = 2 if dtype is BF16 else np.dtype(dtype).itemsize
    if strides is None:
        strides, acc = [], 1
        for s in reversed(shape):
            strides.insert(0, acc)
            acc *= s
    return cv.Tensor.wrap(at, shape, [s * es for s in strides], dtype, layout)


def refused(cv, fn, *args, status=INVALID_ARGUMENT, **kw):
    with pytest.raises(cv.Error) as e:
        fn(*args, **kw)
    assert e.value.status == status, str(e.value)
    st, msg = cv.last_error()
    assert st == status and msg


def test_bfloat16_is_a_type_of_its_own(cv, K):
    t = fake(cv, [4, 8], BF16)
    assert t.dtype == K.DATA_TYPE_BF16 and t.strides == [16, 2]
    n, name = C.c_int32(), cv.capi.nvcv.nvcvDataTypeGetName(C.c_uint64(K.DATA_TYPE_BF16))
    assert name == b"NVCVX_DATA_TYPE_BF16"
    assert cv.capi.nvcv.nvcvDataTypeGetStrideBytes(C.c_uint64(K.DATA_TYPE_BF16), C.byref(n)) == 0 and n.value == 2
    # the operators on images refuse it
    img, out = fake(cv, [1, 8, 8, 3], BF16, "NHWC"), fake(cv, [1, 3, 8, 8], BF16, "NCHW")
    refused(cv, cv.Reformat(), 0, img, out)
    refused(cv, cv.Resize(), 0, img, fake(cv, [1, 4, 4, 3], BF16, "NHWC"), 1)


def test_layer_norm_refusals(cv):
    op = cv.LayerNorm()
    x, y, w = fake(cv, [6, 10]), fake(cv, [6, 10]), fake(cv, [10])
    refused(cv, op, 0, None, w, w, y)
    refused(cv, op, 0, x, w, w, None)
    refused(cv, op, 0, fake(cv, [6, 10], np.float64), w, w, fake(cv, [6, 10], np.float64))
    refused(cv, op, 0, fake(cv, [6, 10], np.uint8), w, w, fake(cv, [6, 10], np.uint8))
    refused(cv, op, 0, x, w, w, fake(cv, [6, 10], F16))              # type
    refused(cv, op, 0, x, w, w, fake(cv, [5, 10]))                   # rows
    refused(cv, op, 0, x, w, w, fake(cv, [6, 11]))                   # row elements
    refused(cv, op, 0, x, fake(cv, [9]), w, y)
    refused(cv, op, 0, x, w, fake(cv, [11]), y)
    refused(cv, op, 0, x, fake(cv, [10], F16), None, y)              # 16-bit weights of 32-bit rows
    refused(cv, op, 0, fake(cv, [6, 10], BF16), fake(cv, [10], BF16), w, fake(cv, [6, 10], BF16))  # gamma and beta differ
    refused(cv, op, 0, fake(cv, [6, 10], BF16), fake(cv, [10], F16), None, fake(cv, [6, 10], BF16))
    refused(cv, op, 0, x, w, w, y, fake(cv, [5]))
    refused(cv, op, 0, x, w, w, y, None, fake(cv, [6], F16))
    for eps in (-1e-5, float("nan"), float("inf")):
        refused(cv, op, 0, x, w, w, y, epsilon=eps)
    refused(cv, op, 0, fake(cv, [6, 10], at=FAKE + 2), w, w, y)      # between elements
    # rows at distances of three kinds
    refused(cv, op, 0, fake(cv, [3, 4, 5, 10], layout="ABDW", strides=[10000, 1100, 20, 1]), w, w, fake(cv, [3, 4, 5, 10]))
    assert cv._cv.cvcudaxLayerNormCreate(None) == INVALID_ARGUMENT
    cv.last_error()
    refused(cv, lambda: cv.check(cv._cv.cvcudaxLayerNormSubmit(cv.Reformat().handle, 0, x.handle, None, None, y.handle, None, None, 1e-5)),
            status=NOT_COMPATIBLE)


def test_layer_norm_gradient_refusals(cv):
    op = cv.LayerNormGrad()
    x, dy, dx, w, s = fake(cv, [6, 10]), fake(cv, [6, 10]), fake(cv, [6, 10]), fake(cv, [10]), fake(cv, [6])
    need = cv.LayerNormGrad.workspace(6, 10)
    room = fake(cv, [max(need, 1)], np.uint8)
    assert need > 0
    refused(cv, op, 0, None, x, w, s, s, dx, w, w, room)
    refused(cv, op, 0, dy, x, w, None, s, dx, w, w, room)
    refused(cv, op, 0, dy, x, w, s, None, dx, w, w, room)
    refused(cv, op, 0, dy, x, w, s, s, None, w, w, room)
    refused(cv, op, 0, fake(cv, [6, 10], F16), x, w, s, s, dx, w, w, room)
    refused(cv, op, 0, dy, x, w, s, s, fake(cv, [7, 10]), w, w, room)
    refused(cv, op, 0, dy, x, w, fake(cv, [5]), s, dx, w, w, room)
    refused(cv, op, 0, dy, x, w, s, s, dx, fake(cv, [11]), w, room)
    refused(cv, op, 0, dy, x, w, s, s, dx, w, fake(cv, [10], F16), room)
    refused(cv, op, 0, dy, x, w, s, s, dx, w, w, None)
    refused(cv, op, 0, dy, x, w, s, s, dx, w, w, fake(cv, [need - 1], np.uint8))
    refused(cv, op, 0, dy, x, w, s, s, dx, w, w, fake(cv, [need], F32))
    refused(cv, op, 0, dy, x, w, s, s, dx, w, w, fake(cv, [need], np.uint8, at=FAKE + 8))
    refused(cv, cv.LayerNormGrad.workspace, -1, 4)
    refused(cv, cv.LayerNormGrad.workspace, 4, 1 << 31)


def test_embedding_refusals(cv):
    op = cv.Embedding()
    table, tokens, out = fake(cv, [50, 10]), fake(cv, [6], np.int64), fake(cv, [6, 10])
    refused(cv, op, 0, None, tokens, out)
    refused(cv, op, 0, table, None, out)
    refused(cv, op, 0, table, fake(cv, [6], np.uint32), out)
    refused(cv, op, 0, table, fake(cv, [6], F32), out)
    refused(cv, op, 0, table, fake(cv, [7], np.int32), out)
    refused(cv, op, 0, table, tokens, fake(cv, [6, 11]))
    refused(cv, op, 0, fake(cv, [50, 10], F16), tokens, out)
    refused(cv, op, 0, fake(cv, [50, 10], F16), tokens, fake(cv, [6, 10], BF16))
    refused(cv, op, 0, table, fake(cv, [6], np.int32, "W", strides=[1], at=FAKE + 1), out)
    refused(cv, op, 0, table, fake(cv, [2, 3], np.int32, "NW", strides=[4, 1]), out)  # tokens with gaps
    refused(cv, op, 0, table, tokens, out, float("nan"))


def test_embedding_gradient_refusals(cv):
    op = cv.EmbeddingGrad()
    table, tokens, dy = fake(cv, [50, 10]), fake(cv, [6], np.int64), fake(cv, [6, 10])
    need = cv.EmbeddingGrad.workspace(6, 50, 10)
    room = fake(cv, [need], np.uint8) if need else None
    refused(cv, op, 0, None, tokens, table, room)
    refused(cv, op, 0, dy, None, table, room)
    refused(cv, op, 0, dy, tokens, None, room)
    refused(cv, op, 0, dy, fake(cv, [5], np.int64), table, room)
    refused(cv, op, 0, fake(cv, [6, 9]), tokens, table, room)
    refused(cv, op, 0, dy, tokens, fake(cv, [50, 10], F16), room)
    refused(cv, op, 0, fake(cv, [6, 10], F16), tokens, fake(cv, [50, 10], BF16), room)
    refused(cv, op, 0, dy, tokens, table, room, float("inf"))
    refused(cv, op, 0, dy, tokens, table, room, 1.0, -2)
    if need:
        refused(cv, op, 0, dy, tokens, table, None)
        refused(cv, op, 0, dy, tokens, table, fake(cv, [need - 1], np.uint8))
    refused(cv, cv.EmbeddingGrad.workspace, 1 << 31, 4, 4)
    refused(cv, cv.EmbeddingGrad.workspace, 4, -1, 4)
    api = importlib.import_module("cvcuda_amd.pyapi")
    with pytest.raises(ValueError):
        api.embedding_grad_into(None, None, None, padding=-1)


HYPER = (1, 1e-3, 0.9, 0.999, 1e-8, 0.01)


def test_adamw_refusals(cv):
    op = cv.AdamW()
    p, m, v, g = ([fake(cv, [600])] for _ in range(4))

    def step(p=p, m=m, v=v, g=g, copies=None, ms=None, vs=None, scale=None, hyper=HYPER):
        op(0, p, m, v, g, copies, ms, vs, scale, *hyper)

    refused(cv, step, p=[None])
    refused(cv, step, p=[fake(cv, [600], np.float64)])
    refused(cv, step, g=[fake(cv, [599])])
    refused(cv, step, g=[fake(cv, [600], np.int32)])
    refused(cv, step, m=[fake(cv, [600], F16)])
    refused(cv, step, v=[fake(cv, [601])])
    refused(cv, step, p=[fake(cv, [20, 30], layout="NW", strides=[40, 1])])    # not dense
    refused(cv, step, copies=[fake(cv, [600])])                                # a copy of 32 bits
    refused(cv, step, copies=[fake(cv, [60], F16)])
    refused(cv, step, scale=fake(cv, [2]))
    refused(cv, step, scale=fake(cv, [1], F16))
    q, u, s = [fake(cv, [600], np.int8)], [fake(cv, [600], np.uint8)], [fake(cv, [3])]
    refused(cv, step, ms=s, vs=s)                                              # scales of 32-bit states
    refused(cv, step, m=q, v=u, ms=s)                                          # one state's scales only
    refused(cv, step, m=q, v=u, ms=[fake(cv, [2])], vs=s)
    refused(cv, step, m=q, v=u, ms=s, vs=[fake(cv, [3], F16)])
    refused(cv, step, m=u, v=u, ms=s, vs=s)
    for k, bad in ((0, 0), (1, float("nan")), (2, 1.0), (2, -0.1), (3, 1.0), (3, float("nan")), (4, -1e-8), (4, float("inf")),
                   (5, float("inf"))):
        hyper = list(HYPER)
        hyper[k] = bad
        refused(cv, step, hyper=hyper)
    # what is wrong with a later tensor is found before the first is changed (its address is made up)
    refused(cv, step, p=p + p, m=m + m, v=v + v, g=g + [fake(cv, [599])])
    assert cv._cv.cvcudaxAdamWSubmit(op.handle, 0, -1, None, None, None, None, None, None, None, None, None) == INVALID_ARGUMENT
    cv.last_error()
    assert cv._cv.cvcudaxAdamWSubmit(op.handle, 0, 1, None, None, None, None, None, None, None, None,
                                     C.byref(cv.capi.AdamWArgs(1e-3, .9, .9, 1e-8, 0, 1))) == INVALID_ARGUMENT
    cv.last_error()
    unpack = cv.AdamWUnpack()
    refused(cv, unpack, 0, [fake(cv, [600])], s, p)
    refused(cv, unpack, 0, q, [fake(cv, [2])], p)
    refused(cv, unpack, 0, q, s, [fake(cv, [600], F16)])
    refused(cv, unpack, 0, q, s, [fake(cv, [599])])


def test_lists_of_different_lengths(cv):
    api = importlib.import_module("cvcuda_amd.pyapi")
    t = api.Tensor(_wrap=fake(cv, [8]))
    with pytest.raises(ValueError):
        api.adamw_into([t, t], [t], [t, t], [t, t], 1)
    with pytest.raises(ValueError):
        api.adamw_unpack_into([t], [t], [t, t])
    with pytest.raises(ValueError):
        cv.AdamW()(0, [t._t], [], [t._t], [t._t], None, None, None, None, *HYPER)


@pytest.mark.parametrize("columns", [16385, 20000, 40000, 70003, 1 << 20, 3000001, 1 << 30])
def test_workspace_of_wide_rows(cv, columns):
    """Rows that no workgroup holds ask for no more than the widest that one does, beyond the two sums of one part."""
    most = max(cv.LayerNormGrad.workspace(6144, 16384), 2 * 4 * columns)
    for rows in (1, 5, 1000, 6144, 100000, (1 << 31) - 1):
        assert 2 * 4 * columns <= cv.LayerNormGrad.workspace(rows, columns) <= most
    # little beside the input itself
    assert cv.LayerNormGrad.workspace(6144, columns) <= 6144 * columns * 2 // 16


def test_workspace_of_few_rows(cv):
    """A gradient of one launch makes its sums from the rows: it asks for the least, and nothing that is touched is as small."""
    for columns in (4, 64, 1000, 8192, 16384):
        for rows in (1, 6, 300, 1024):
            assert cv.LayerNormGrad.workspace(rows, columns) == 16
        assert cv.LayerNormGrad.workspace(1025, columns) >= 2 * 4 * columns
    for rows, columns in ((1, 1), (4, 2), (3, 3), (1, 16385), (1025, 4)):
        assert cv.LayerNormGrad.workspace(rows, columns) > 16
    assert cv.LayerNormGrad.workspace(0, 100) == cv.LayerNormGrad.workspace(100, 0) == 0


def test_a_captured_gradient_needs_a_workspace(cv, monkeypatch):
    """Memory that only the call holds goes back to the allocator with it; a graph would write there in every replay."""
    api = importlib.import_module("cvcuda_amd.pyapi")
    calls, capturing = [], True
    monkeypatch.setattr(api, "_default_stream_key", lambda stream: None)
    monkeypatch.setattr(api, "_native_stream_key", lambda: None)
    monkeypatch.setattr(api, "_capturing", lambda stream: capturing)
    monkeypatch.setattr(api, "_run", lambda stream, reads, writes, op, *args: calls.append(writes))
    monkeypatch.setattr(api, "_result", lambda shape, *args: api.Tensor(_wrap=fake(cv, shape, np.uint8)))
    monkeypatch.setattr(api, "_like", lambda *args: api._result((1,)))
    wrap = lambda *args, **kw: api.Tensor(_wrap=fake(cv, *args, **kw))
    x, w, s, table, tokens = wrap([4096, 10]), wrap([10]), wrap([4096]), wrap([50, 10]), wrap([4096], np.int64)
    norm, embedding = cv.LayerNormGrad.workspace(4096, 10), cv.EmbeddingGrad.workspace(4096, 50, 10)
    assert norm > 0 and embedding > 0
    forms = [(lambda **kw: api.layer_norm_grad_into(x, w, w, x, x, w, s, s, **kw), norm), (lambda **kw: api.layer_norm_grad(x, x, w, s, s, **kw), norm),
             (lambda **kw: api.embedding_grad_into(table, x, tokens, **kw), embedding), (lambda **kw: api.embedding_grad(x, tokens, 50, **kw), embedding)]
    for call, need in forms:
        for stream in (None, "side"):
            with pytest.raises(cv.Error) as e:
                call(stream=stream)
            assert e.value.status == 4 and "workspace=" in str(e.value) and str(need) in str(e.value) and not calls
        room = wrap([need], np.uint8)
        call(workspace=room)
        assert calls.pop()[-1] is room
    # what needs none is captured without one
    api.layer_norm_grad_into(x, None, None, x, x, w, s, s)
    api.embedding_grad_into(table, wrap([64, 10]), wrap([64], np.int64))
    assert [len(writes) for writes in calls] == [1, 1]
    capturing = False
    forms[0][0]()
    assert calls[-1][-1].shape == (norm,)


def test_results_of_bfloat16_are_handed_out_again(cv, monkeypatch):
    """As those of every other type (no GPU: the library's tensors are stand-ins)."""
    api, made = importlib.import_module("cvcuda_amd.pyapi"), []

    def new(shape, dtype, layout):
        made.append((shape, dtype))
        return fake(cv, list(shape), dtype)

    monkeypatch.setattr(api, "_new_result", new)
    monkeypatch.setattr(api.torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(api, "_native_stream_key", lambda: 0)
    monkeypatch.setattr(api, "_outputs", api._Outputs())
    for dtype in (BF16, np.dtype(F16), np.dtype(np.int16)):
        result = api._result((4, 8), dtype, None, None)
        raw = result._t
        assert result.dtype == dtype and result.shape == (4, 8)
        result._wrote = (0, None)
        del result
        again, other = api._result((4, 8), dtype, None, None), api._result((4, 8), dtype, None, None)
        assert again._t is raw and other._t is not raw
    assert made == [((4, 8), t) for t in (BF16, F16, np.int16) for _ in range(2)]
    with pytest.raises(TypeError):
        api._outputs.get((4, 8), torch.float32, None)  # (numpy's types stand for the others)
