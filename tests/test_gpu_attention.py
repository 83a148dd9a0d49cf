"""cvcudaxAttentionSubmit and its gradient against their definition in 64 bits (head_reference.py derives the bounds)."""
import importlib
import math

import numpy as np
import pytest
import torch

import head_reference as ref
from row_reference import close

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})  # (a wait for the default stream has the calls after it record events)


def random(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def numbers(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Call:
    """Sequences of (rows, keys), with `before` rows of none before them and `behind` behind; their keys packed as the rows (room None) or in
    places of `room` each. What lies in no sequence is NaN."""

    def __init__(self, lengths, heads, key_heads, d, dtype, seed, causal=True, room=None, before=0, behind=0, scale=None, size=1.0):
        self.lengths, self.heads, self.key_heads, self.d, self.dtype, self.causal = lengths, heads, key_heads, d, dtype, causal
        self.scale = d ** -0.5 if scale is None else scale
        starts = [before]
        for n, _ in lengths:
            starts.append(starts[-1] + n)
        self.rows = starts[-1] + behind
        self.offsets, self.starts = numbers(starts), starts
        self.key_offsets = self.key_lengths = None
        if room is None:
            assert all(a == b for a, b in lengths)
            self.key_starts, self.keys = starts, self.rows
        else:
            self.key_starts = [before + room * i for i in range(len(lengths) + 1)]
            self.keys = self.key_starts[-1] + behind
            self.key_offsets, self.key_lengths = numbers(self.key_starts), numbers([b for _, b in lengths])
        made = {"q": (self.rows, heads), "k": (self.keys, key_heads), "v": (self.keys, key_heads), "grad": (self.rows, heads)}
        for i, (name, shape) in enumerate(made.items()):
            t = random(shape + (d,), dtype, seed * 10 + i, size)
            keep = torch.zeros(shape[0], dtype=torch.bool, device="cuda")
            for b, (rows, keys) in enumerate(lengths):
                at = self.key_starts[b] if name in "kv" else starts[b]
                keep[at:at + (keys if name in "kv" else rows)] = True
            t[~keep] = float("nan")
            setattr(self, name, t)
            setattr(self, "kept_" + name, keep)

    def parts(self):
        """(rows, keys) of each sequence."""
        for b, (rows, keys) in enumerate(self.lengths):
            yield slice(self.starts[b], self.starts[b] + rows), slice(self.key_starts[b], self.key_starts[b] + keys)

    def more(self, api):
        made = {"causal": self.causal, "scale": self.scale}
        if self.key_offsets is not None:
            made.update(key_offsets=api.as_tensor(self.key_offsets), key_lengths=api.as_tensor(self.key_lengths))
        return made

    def run(self, api, out=None, stats=True, **how):
        out = torch.full(self.q.shape, 7.0, dtype=self.dtype, device="cuda") if out is None else out
        lse = torch.full((self.heads, self.rows), 7.0, device="cuda") if stats else None
        wrap = lambda t: api.as_tensor(t, "TWE")
        api.attention_into(wrap(out), wrap(self.q), wrap(self.k), wrap(self.v), api.as_tensor(self.offsets),
                           lse=api.as_tensor(lse) if stats else None, **self.more(api), **how)
        return out, lse

    def gradients(self, api, out, lse, made=None, **how):
        made = [torch.full(t.shape, 7.0, dtype=self.dtype, device="cuda") for t in (self.q, self.k, self.v)] if made is None else made
        wrap = lambda t: api.as_tensor(t, "TWE")
        api.attention_grad_into(*map(wrap, made), wrap(self.grad), wrap(self.q), wrap(self.k), wrap(self.v), wrap(out), api.as_tensor(lse),
                                api.as_tensor(self.offsets), **self.more(api), **how)
        return made

    def check(self, api, **how):
        out, lse = self.run(api, **how)
        for rows, keys in self.parts():
            for h in range(self.heads):
                kh = h // (self.heads // self.key_heads)
                want = ref.attention(self.q[rows, h].double(), self.k[keys, kh].double(), self.v[keys, kh].double(), self.scale, self.causal, self.dtype)
                close(out[rows, h], want[0], want[2], "out of head %d of rows %s" % (h, rows))
                none = want[1] == -math.inf
                assert (lse[h, rows][none] == -math.inf).all() and (out[rows, h][none] == 0).all()
                close(lse[h, rows][~none], want[1][~none], want[3][~none], "lse of head %d of rows %s" % (h, rows))
        outside = ~self.kept_q
        assert (out[outside] == 7).all() and (lse[:, outside] == 7).all()
        return out, lse

    def check_gradients(self, api, out, lse, **how):
        got = self.gradients(api, out, lse, **how)
        norm = lambda t, keep: float(t[keep].double().norm(dim=-1).max()) if keep.any() else 0.0
        bound = norm(self.grad, self.kept_grad) * norm(self.v, self.kept_v)
        want = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (self.q, self.k, self.v)]
        errors = [torch.zeros_like(t) for t in want]
        for rows, keys in self.parts():
            for h in range(self.heads):
                kh = h // (self.heads // self.key_heads)
                values, off = ref.attention_grad(self.grad[rows, h].double(), self.q[rows, h].double(), self.k[keys, kh].double(),
                                                 self.v[keys, kh].double(), out[rows, h].double(), lse[h, rows].double(), self.scale, self.causal,
                                                 self.dtype, bound)
                for i, at in enumerate(((rows, h), (keys, kh), (keys, kh))):
                    want[i][at] += values[i]
                    errors[i][at] += off[i]
        for name, a, b, e, keep in zip(("gradient of q", "of k", "of v"), got, want, errors, (self.kept_q, self.kept_k, self.kept_k)):
            # (F16 ends at 65504: what is beyond that and half a step is infinite)
            over = keep[:, None, None] & a.isinf() & (b.abs() + e >= 65520) & (a.sign() == b.sign())
            fine = keep[:, None, None] & ~over
            close(a[fine], b[fine], e[fine], name)
            assert (a[~keep] == 7).all()
        return got


MIXED = [(31, 31), (32, 32), (0, 0), (33, 33), (1, 1), (65, 65), (130, 130)]
HEADS = [(1, 1), (4, 4), (6, 2), (8, 1)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 128])
def test_packed_sequences(api, d, causal, dtype):
    for seed, (heads, key_heads) in enumerate(HEADS):
        Call(MIXED, heads, key_heads, d, dtype, seed, causal, before=3, behind=5).check(api)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 128])
def test_gradients_of_packed_sequences(api, d, causal, dtype):
    for seed, (heads, key_heads) in enumerate(HEADS):
        call = Call(MIXED, heads, key_heads, d, dtype, seed, causal, before=3, behind=5)
        out, lse = call.check(api)
        call.check_gradients(api, out, lse)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,keys", [(1, 1), (1, 31), (1, 33), (1, 129), (1, 700), (1, 5000), (3, 1000), (17, 64), (40, 2000), (128, 129),
                                       (129, 640), (200, 3001)])
def test_few_and_many_rows_before_a_cache(api, rows, keys, dtype):
    """One sequence and some of other lengths: the keys are split where there are few rows."""
    for d, heads, key_heads in ((64, 4, 4), (128, 8, 2)):
        for causal in (True, False):
            lengths = [(rows, keys), (min(rows, 2), max(keys // 3, min(rows, 2))), (rows, keys)]
            Call(lengths[:1], heads, key_heads, d, dtype, rows + keys, causal, room=keys + 3, behind=2).check(api)
            Call(lengths, heads, key_heads, d, dtype, rows + keys, causal, room=keys + 3, before=1).check(api)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_of_keys_of_their_own(api, causal, dtype):
    for d, heads, key_heads in ((40, 3, 3), (128, 4, 2)):
        call = Call([(5, 90), (0, 30), (33, 33), (70, 200), (1, 1)], heads, key_heads, d, dtype, d, causal, room=210, before=2, behind=3)
        out, lse = call.check(api)
        got = call.check_gradients(api, out, lse)
        # (keys that no row sees have gradients of 0)
        assert (got[1][212:242] == 0).all() and (got[2][212:242] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_that_see_nothing(api, dtype):
    """More rows than keys, and no keys at all: zeros, -infinity, gradients of 0."""
    for lengths in ([(40, 7), (5, 0), (3, 3), (300, 100)], [(2, 0)], [(1, 0), (2, 1)]):
        for causal in (True, False):
            call = Call(lengths, 4, 2, 64, dtype, 3, causal, room=128)
            out, lse = call.check(api)
            call.check_gradients(api, out, lse)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_more_sequences_than_lanes(api, dtype):
    g = torch.Generator().manual_seed(1)
    lengths = [(int(n), int(n)) for n in torch.randint(0, 9, (200,), generator=g)]
    call = Call(lengths, 2, 1, 32, dtype, 4)
    out, lse = call.check(api)
    call.check_gradients(api, out, lse)
    lengths = [(int(n), int(n) + 30) for n in torch.randint(0, 2, (150,), generator=g)]
    Call(lengths, 2, 1, 32, dtype, 4, room=33).check(api)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_scores_and_equal_ones(api, dtype):
    """Softmaxes of one key, of keys that grow along the sequence, and of equal ones."""
    call = Call([(70, 70), (200, 200)], 2, 2, 64, dtype, 5, size=6.0)   # scores of some hundreds
    out, lse = call.check(api)
    call.check_gradients(api, out, lse)
    call = Call([(1, 900)], 2, 2, 64, dtype, 5, room=900)
    call.k[:, :] = call.k[:1] * torch.linspace(0.1, 4, 900, device="cuda")[:, None, None].to(dtype)
    call.q[:] = call.k[-1:]
    call.check(api)
    call.k[:] = call.k[:1]
    call.check(api)


def test_small_and_large_gradients_in_16_bits(api):
    """Gradients far below what F16 holds of their products with shares, and values far above 1."""
    for size in (2.0 ** -12, 1.0, 2.0 ** 10):
        call = Call([(300, 300)], 2, 2, 64, F16, 6, causal=False)
        call.v *= 2.0 ** 7
        call.grad *= size
        out, lse = call.check(api)
        call.check_gradients(api, out, lse)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_parts_of_one_tensor(api, dtype):
    """Queries, keys and values side by side, results in the same places of others."""
    call = Call([(50, 50), (70, 70)], 4, 2, 64, dtype, 7)
    out, lse = call.check(api)
    want = call.check_gradients(api, out, lse)
    whole = random((120, 9, 64), dtype, 1)
    parts = whole.split([4, 2, 2, 1], 1)
    for part, t in zip(parts, (call.q, call.k, call.v)):
        part.copy_(t)
    call.q, call.k, call.v = parts[:3]
    made = torch.full((120, 6, 72), 9.0, dtype=dtype, device="cuda")
    again, _ = call.run(api, out=made[:, 1:5, :64])
    assert torch.equal(again, out) and (made[:, 0] == 9).all() and (made[:, 5] == 9).all() and (made[..., 64:] == 9).all()
    grads = torch.full((120, 9, 64), 9.0, dtype=dtype, device="cuda")
    got = call.gradients(api, out, lse, made=list(grads.split([4, 2, 2, 1], 1)[:3]))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (grads[:, 8] == 9).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_what_is_not_finite_stays_in_its_sequence(api, dtype):
    call = Call([(40, 40), (50, 50), (60, 60)], 2, 1, 64, dtype, 8)
    clean, lse = call.check(api)
    grads = call.check_gradients(api, clean, lse)
    call.k[45], call.v[60], call.grad[50] = float("nan"), float("inf"), float("nan")
    out, lse = call.run(api)
    got = call.gradients(api, out, lse)
    assert out[45:90].isnan().all()  # (the rows that see the key)
    for rows in (slice(0, 40), slice(90, 150)):
        assert torch.equal(out[rows], clean[rows])
        for a, b in zip(got, grads):
            # (F16: rounded relative to the longest rows of the call, which may be others now)
            assert torch.equal(a[rows], b[rows]) if dtype is BF16 else ((a[rows] - b[rows]).abs() <= 2.0 ** -9 * b[rows].abs().max()).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_the_same_in_every_call(api, dtype):
    call = Call([(700, 700), (90, 90)], 8, 2, 128, dtype, 9)
    out, lse = call.run(api)
    grads = call.gradients(api, out, lse)
    token = Call([(1, 4000)], 8, 2, 128, dtype, 9, room=4000)
    one = token.run(api)
    for _ in range(3):
        again = call.run(api)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        assert all(torch.equal(a, b) for a, b in zip(call.gradients(api, out, lse), grads))
        assert all(torch.equal(a, b) for a, b in zip(token.run(api), one))
        assert torch.equal(call.run(api, stats=False)[0], out)


def test_more_than_four_gigabytes(api):
    """A cache whose last places lie beyond 32 bits, of bytes and of elements."""
    places, heads, d = 5000000, 4, 128
    k, v = (torch.zeros((places, heads, d), dtype=BF16, device="cuda") for _ in range(2))
    assert k.numel() > 1 << 31
    call = Call([(3, 500), (40, 600)], 8, heads, d, BF16, 10, room=600)
    few = call.k, call.v, call.key_offsets
    k[-1200:], v[-1200:] = call.k, call.v
    far = [places - 1200, places - 600, places]
    call.k, call.v, call.key_offsets, call.key_starts = k, v, numbers(far), far
    out, lse = call.check(api)
    call.k, call.v, call.key_offsets = few
    grads = call.gradients(api, out, lse)
    call.k, call.v, call.key_offsets = k, v, numbers(far)
    made = [torch.empty_like(call.q), torch.zeros_like(k), torch.zeros_like(v)]
    call.gradients(api, out, lse, made=made)
    assert torch.equal(made[0], grads[0])
    for a, b in zip(made[1:], grads[1:]):
        for at, n in ((0, 500), (600, 600)):
            assert torch.equal(a[places - 1200 + at:places - 1200 + at + n], b[at:at + n])
        assert (a[:places - 1200] == 0).all()


def test_offsets_beyond_the_tensors(api):
    """They count as the border: what is there is computed, nothing else is touched."""
    call = Call([(30, 30), (50, 50)], 2, 2, 64, BF16, 11)
    want, lse = call.run(api)
    whole = torch.equal
    call.offsets = numbers([-5, 30, 1000])
    out, _ = call.run(api)
    assert whole(out, want)
    call.offsets = numbers([0, 30, 20])  # the second has nothing
    out, _ = call.run(api)
    assert whole(out[:30], want[:30]) and (out[30:] == 7).all()
    call.offsets, call.key_offsets, call.key_lengths = numbers([0, 30, 80]), numbers([0, 30, 200]), numbers([500, 50])
    out, _ = call.run(api)
    assert whole(out, want)
    grads = call.gradients(api, out, lse)
    call.key_lengths = numbers([-3, 50])
    out, lse = call.run(api)
    assert (out[:30] == 0).all() and whole(out[30:], want[30:]) and (lse[:, :30] == -math.inf).all()
    assert (call.gradients(api, out, lse)[0][:30] == 0).all() and grads[0].isfinite().all()


def test_no_sequences(api):
    call = Call([(4, 4)], 2, 2, 64, BF16, 12)
    call.offsets = numbers([0])
    out, lse = call.run(api)
    grads = call.gradients(api, out, lse)
    assert all((t == 7).all() for t in (out, lse, *grads))


def test_another_stream(api):
    call = Call([(700, 700), (300, 300)], 4, 4, 64, F16, 13)
    out, lse = call.run(api)
    grads = call.gradients(api, out, lse)
    torch.cuda.synchronize()
    side, wrap = api.Stream(), api.as_tensor
    q, k, v, offsets = wrap(call.q), wrap(call.k), wrap(call.v), wrap(call.offsets)
    stats = wrap(torch.empty_like(lse))
    first = api.attention(q, k, v, offsets, lse=stats)
    with side:
        got = api.attention_grad(wrap(call.grad), q, k, v, first, stats, offsets)
    again = api.attention_grad(wrap(call.grad), q, k, v, first, stats, offsets)
    torch.cuda.synchronize()
    assert torch.equal(first.torch(), out)
    assert all(torch.equal(a.torch(), b) and torch.equal(c.torch(), b) for a, b, c in zip(got, grads, again))


def test_in_a_graph(api):
    """Prompts and single tokens, the latter with a workspace of their own."""
    call = Call([(100, 100), (60, 60)], 4, 2, 64, F16, 14)
    token = Call([(1, 3000)], 4, 2, 64, F16, 15, room=3000)
    need = api.Attention.workspace(1, 3000, 1, 4, 2, 64)
    assert need > 0 and api.Attention.workspace(160, 160, 2, 4, 2, 64) == 0
    rooms = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (need, api.AttentionGrad.workspace(160, 160, 2, 4, 2, 64))]
    out, one = torch.empty_like(call.q), torch.empty_like(token.q)
    lse, ones = torch.empty((4, 160), device="cuda"), torch.empty((4, 1), device="cuda")
    made = [torch.empty_like(t) for t in (call.q, call.k, call.v)]
    graph, wrap = torch.cuda.CUDAGraph(), api.as_tensor
    t = {name: wrap(getattr(call, name)) for name in ("q", "k", "v", "grad", "offsets")}
    u = {name: wrap(getattr(token, name)) for name in ("q", "k", "v", "offsets", "key_offsets", "key_lengths")}
    wrapped = [wrap(x) for x in (out, lse, one, ones, *made, *rooms)]
    with torch.cuda.graph(graph):
        s = api.as_stream(torch.cuda.current_stream())
        api.attention_into(wrapped[0], t["q"], t["k"], t["v"], t["offsets"], lse=wrapped[1], stream=s)
        api.attention_grad_into(*wrapped[4:7], t["grad"], t["q"], t["k"], t["v"], wrapped[0], wrapped[1], t["offsets"], workspace=wrapped[8], stream=s)
        with pytest.raises(api.Error):
            api.attention_into(wrapped[2], u["q"], u["k"], u["v"], u["offsets"], key_offsets=u["key_offsets"], key_lengths=u["key_lengths"], stream=s)
        api.attention_into(wrapped[2], u["q"], u["k"], u["v"], u["offsets"], key_offsets=u["key_offsets"], key_lengths=u["key_lengths"],
                           lse=wrapped[3], workspace=wrapped[7], stream=s)
    for turn in range(4):
        call.q.copy_(random(call.q.shape, F16, 100 + turn))
        token.q.copy_(random(token.q.shape, F16, 200 + turn))
        token.key_lengths.copy_(numbers([3000 - 700 * turn]))  # a cache's lengths change between replays
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, lse, one, ones, *made)]
        want = call.run(api)
        token.lengths = [(1, 3000 - 700 * turn)]
        want += token.check(api)
        want += tuple(call.gradients(api, want[0], want[1]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once(api):
    """Threads that call at the same time, each with its own tensors."""
    import threading
    calls = [Call([(1, 2000 + 100 * i)], 8, 2, 64, BF16, 20 + i, room=2000 + 100 * i) for i in range(4)]
    want = [c.check(api) for c in calls]
    wrong = []

    def work(c, w):
        for _ in range(20):
            got = c.run(api)
            torch.cuda.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, w)):
                wrong.append(c)

    threads = [threading.Thread(target=work, args=x) for x in zip(calls, want)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_gradients_of_one_row_in_a_graph_and_beside_others(api):
    """What the smallest call works with is its own: it needs a workspace when it is captured, and changes nobody else's."""
    calls = [Call([(1, 1)], 1, 1, 8, BF16, 30 + i) for i in range(2)]
    made = [c.run(api) for c in calls]
    assert api.AttentionGrad.workspace(1, 1, 1, 1, 1, 8) > 0
    api.layer_norm_grad(*[api.as_tensor(t) for t in (random((4, 8), BF16, 1), random((4, 8), BF16, 2))], None,
                        *[api.as_tensor(torch.ones(4, device="cuda")) for _ in range(2)])
    torch.cuda.synchronize()
    before = {d: t.torch().clone() for d, t in api._untouched.items()}
    for c, m in zip(calls, made):
        c.check_gradients(api, *m)
    torch.cuda.synchronize()
    assert all(torch.equal(api._untouched[d].torch(), t) for d, t in before.items())
    graph = torch.cuda.CUDAGraph()
    t = {n: api.as_tensor(getattr(calls[0], n)) for n in ("q", "k", "v", "grad", "offsets")}
    outs, lse = [api.as_tensor(torch.empty_like(calls[0].q)) for _ in range(4)], api.as_tensor(torch.empty((1, 1), device="cuda"))
    with torch.cuda.graph(graph):
        s = api.as_stream(torch.cuda.current_stream())
        api.attention_into(outs[3], t["q"], t["k"], t["v"], t["offsets"], lse=lse, stream=s)
        with pytest.raises(api.Error):
            api.attention_grad_into(*outs[:3], t["grad"], t["q"], t["k"], t["v"], outs[3], lse, t["offsets"], stream=s)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,heads,key_heads", [(40, 2, 2), (128, 6, 2), (64, 8, 1)])
def test_gradients_of_few_rows_and_of_few_keys(api, d, heads, key_heads, causal, dtype):
    """Where the work of a kernel is split: long caches of few rows, and few keys that many rows see; some sequences have far fewer than others."""
    few_rows = Call([(5, 3000), (0, 10), (1, 1), (130, 1500), (3, 0)], heads, key_heads, d, dtype, 40, causal, room=3000, before=2, behind=3)
    few_keys = Call([(1500, 40), (0, 0), (700, 1), (2, 130)], heads, key_heads, d, dtype, 41, causal, room=140, before=1, behind=2)
    for call in (few_rows, few_keys):
        for _ in range(2):
            again = call.check_gradients(api, *call.run(api))
        first = call.gradients(api, *call.run(api))
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(first, again))
    # (more than the rows' sums: both are split)
    sums = lambda rows: (2 * rows * heads + 3) // 4 * 16
    assert api.AttentionGrad.workspace(few_rows.rows, few_rows.keys, 5, heads, key_heads, d) > sums(few_rows.rows)
    assert api.AttentionGrad.workspace(few_keys.rows, few_keys.keys, 4, heads, key_heads, d) > sums(few_keys.rows)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys", [(0, 5), (3, 0), (200, 0)])
def test_no_rows_or_no_keys_at_all(api, rows, keys, causal):
    call = Call([(rows, keys)], 4, 2, 64, F16, 50, causal, room=keys, before=2)
    out, lse = call.check(api)
    for t in call.check_gradients(api, out, lse):
        assert (t[2:] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_tensor_in_three_places(api, dtype):
    """Keys that are values and queries as well: what is read twice counts for both."""
    call = Call([(70, 70), (9, 9)], 4, 4, 64, dtype, 51)
    call.k = call.v = call.q
    out, lse = call.check(api)
    grads = call.check_gradients(api, out, lse)
    x, g, o, s, seq = (api.as_tensor(t) for t in (call.q, call.grad, out, lse, call.offsets))
    again = api.attention(x, x, x, seq, causal=True, scale=call.scale)
    made = api.attention_grad(g, x, x, x, o, s, seq, causal=True, scale=call.scale)
    torch.cuda.synchronize()
    assert torch.equal(again.torch(), out) and all(torch.equal(a.torch(), b) for a, b in zip(made, grads))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,key_heads,d,room", [(8, 8, 128, 20000), (12, 4, 40, 60000), (4, 4, 64, 80000)])
def test_single_tokens_before_large_caches(api, heads, key_heads, d, room, dtype):
    """Caches that are larger than what the card keeps near its memory, filled to different lengths; NaN in all other places."""
    assert 2 * 4 * room * key_heads * d * 2 > 128 << 20
    Call([(1, 1), (1, 3000), (0, 40), (2, 777)], heads, key_heads, d, dtype, 60, True, room=room).check(api)
    Call([(1, room), (1, 0), (3, 33), (1, 1025)], heads, key_heads, d, dtype, 61, False, room=room, before=1, behind=1).check(api)
