"""Rotary positions, attention and log probabilities as a model uses them: a training step's two directions, and answers token by token from a
cache, in a graph. The parts by themselves are held to their definitions in their own files."""
import importlib
import math

import pytest
import torch

import head_reference as ref
from row_reference import STEP, U, close

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def api(cv, gpu):
    return importlib.import_module("cvcuda_amd.pyapi")


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(api, monkeypatch):
    monkeypatch.setattr(api, "_followed", {})


def random(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def rounded(value, error, dtype):
    return error + U[dtype] * (value.abs() + error) + STEP[dtype]


def there_and_back(qkv, lengths, positions, tokens, g, h, heads, key_heads, scale, temper, dtype):
    """(log probabilities, entropies, gradient of qkv) of a step in 64 bits, by automatic differentiation, and how far off the results of the
    operators in a row may be. Every operator is off by its own error (twice that, since it meets values that are off by less than their own
    size), and hands on that of what it takes: scores off by e make shares off by a factor of exp(2 e) at most."""
    d = qkv.shape[2]
    x = qkv.double().detach().requires_grad_()
    starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    parts = [slice(a, b) for a, b in zip(starts, starts[1:])]
    of = lambda head: head // (heads // key_heads)
    q, k, v = x[:, :heads], x[:, heads:heads + key_heads], x[:, heads + key_heads:]
    (q, e_q), (k, e_k) = ref.rotary(q, positions, d), ref.rotary(k, positions, d)
    e_q, e_k = (rounded(t.detach(), e.detach(), dtype) for t, e in ((q, e_q), (k, e_k)))
    out, e_out = torch.empty_like(q), torch.empty_like(e_q)
    saved = {}
    for p in parts:
        for n in range(heads):
            m = of(n)
            o, lse, e, _ = ref.attention(q[p, n], k[p, m], v[p, m], scale, True, dtype)
            out[p, n] = o
            s = scale * (q[p, n] @ k[p, m].t()).detach()
            seen = ref.sees(len(s), len(s), True, s.device)
            share = torch.where(seen, torch.exp(s - lse.detach()[:, None]), 0.0)
            e_s = scale * ((q[p, n].detach().abs() + e_q[p, n]) @ e_k[p, m].t() + e_q[p, n] @ k[p, m].detach().abs().t())
            r = torch.expm1(2 * torch.where(seen, e_s, 0.0).amax(1))
            saved[p.start, n] = lse.detach(), share, r
            e_out[p, n] = rounded(o.detach(), 2 * e.detach() + r[:, None] * (share @ v[p, m].detach().abs()), dtype)
    logits = out.reshape(len(out), -1)
    (logp, entropy, lse), (e_logp, e_entropy, _) = ref.log_probs(logits, tokens, temper)
    ((logp * g.double()).sum() + (entropy * h.double()).sum()).backward()
    with torch.no_grad():
        e_x = e_out.reshape(len(out), -1)
        most = 2 * temper * e_x.amax(1, keepdim=True)
        r = torch.expm1(most)
        every = temper * logits - lse[:, None]
        share = every.exp()
        part = (every + entropy[:, None]).abs()
        e_h = 2 * e_entropy[:, None] + (1 + r) ** 2 * (share * part * temper * e_x).sum(1, keepdim=True)
        e_logp = 2 * e_logp + most[:, 0]
        grad, e = ref.log_probs_grad(logits, tokens, lse, g.double(), temper, entropy, h.double())
        e = 2 * e + temper * (g.double().abs()[:, None] * r * share + h.double().abs()[:, None] * share * (r * part + (1 + r) * (most + e_h)))
        e_grad = rounded(grad, e, dtype).reshape(out.shape)
        grad = grad.reshape(out.shape)
        made = [torch.zeros_like(t) for t in (q, k, v)]
        error = [torch.zeros_like(t) for t in (q, k, v)]
        bound = float((grad.abs() + e_grad).norm(dim=-1).max() * v.detach().norm(dim=-1).max())
        for p in parts:
            for n in range(heads):
                m = of(n)
                its = q[p, n], k[p, m], v[p, m], out[p, n]
                lse_n, share, r = saved[p.start, n]
                values, own = ref.attention_grad(grad[p, n], *its, lse_n, scale, True, dtype, bound)
                dp, delta = grad[p, n] @ v[p, m].t(), (grad[p, n] * out[p, n]).sum(1, keepdim=True)
                t = (share * (dp - delta)).abs()
                e_dp = e_grad[p, n] @ v[p, m].abs().t()
                e_delta = (e_grad[p, n] * (out[p, n].abs() + e_out[p, n]) + grad[p, n].abs() * e_out[p, n]).sum(1, keepdim=True)
                e_t = r[:, None] * t + (1 + r[:, None]) * share * (e_dp + e_delta)
                off = (scale * (e_t @ k[p, m].abs() + (t + e_t) @ e_k[p, m]), scale * (e_t.t() @ q[p, n].abs() + (t + e_t).t() @ e_q[p, n]),
                       (r[:, None] * share).t() @ (grad[p, n].abs() + e_grad[p, n]) + share.t() @ e_grad[p, n])
                for i, at in enumerate(((p, n), (p, m), (p, m))):
                    made[i][at] += values[i]
                    error[i][at] += 2 * own[i] + off[i]
        error = [rounded(a, b, dtype) for a, b in zip(made, error)]
        for i in (0, 1):  # turned back: each element is off by its own part of both of its pair
            _, own = ref.rotary(made[i], positions, d, inverse=True)
            half = error[i].roll(d // 2, -1)
            error[i] = 2 * own + error[i] + half
        return logp, entropy, x.grad, e_logp, e_h[:, 0], torch.cat(error, 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_step_and_its_gradient(api, dtype):
    """Queries, keys and values are parts of one tensor, and their gradients of another."""
    lengths, heads, key_heads, d, scale, temper = [50, 1, 33], 4, 2, 32, 0.1, 2.0
    rows, every = sum(lengths), heads + 2 * key_heads
    qkv, back = random((rows, every, d), 1, dtype), torch.full((rows, every, d), 7.0, dtype=dtype, device="cuda")
    positions = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    offsets = torch.tensor([0, 50, 51, 84], dtype=torch.int32, device="cuda")
    tokens = torch.randint(-2, heads * d, (rows,), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    g, h = random((rows,), 3, torch.float32), random((rows,), 4, torch.float32)
    wrap = api.as_tensor
    part = lambda t, at, n: wrap(t[:, at:at + n], "TWE")
    q, k = (wrap(torch.empty((rows, n, d), dtype=dtype, device="cuda"), "TWE") for n in (heads, key_heads))
    v = part(qkv, heads + key_heads, key_heads)
    lse, stats, entropy = (torch.empty(s, device="cuda") for s in ((heads, rows), (rows,), (rows,)))
    out = torch.empty((rows, heads, d), dtype=dtype, device="cuda")
    at, seq, o = wrap(positions), wrap(offsets), wrap(out, "TWE")
    api.rotary_into(q, part(qkv, 0, heads), at)
    api.rotary_into(k, part(qkv, heads, key_heads), at)
    api.attention_into(o, q, k, v, seq, scale=scale, lse=wrap(lse))
    logits = wrap(out.view(rows, heads * d))
    logp = api.log_probs(logits, wrap(tokens), temper, lse=wrap(stats), entropy=wrap(entropy))
    grad = torch.empty_like(out)
    api.log_probs_grad_into(wrap(grad.view(rows, heads * d)), logits, wrap(tokens), wrap(stats), wrap(g), temper, entropy=wrap(entropy), grad_entropy=wrap(h))
    grads = part(back, 0, heads), part(back, heads, key_heads), part(back, heads + key_heads, key_heads)
    api.attention_grad_into(*grads, wrap(grad, "TWE"), q, k, v, o, wrap(lse), seq, scale=scale)
    api.rotary_into(grads[0], grads[0], at, inverse=True)
    api.rotary_into(grads[1], grads[1], at, inverse=True)
    torch.cuda.synchronize()
    want = there_and_back(qkv, lengths, positions, tokens, g, h, heads, key_heads, scale, temper, dtype)
    close(logp.torch(), want[0].detach(), want[3], "log probabilities")
    close(entropy, want[1].detach(), want[4], "entropies")
    close(back, want[2], want[5], "gradient")


HEADS, KEY_HEADS, D, ROOM = 4, 2, 16, 64
SCALING = dict(factor=4.0, original=32.0, low=1.0, high=4.0)


class Answers:
    """A model of one layer that answers: a token's row of a table is its query, keys and values, what attention gives are the next one's
    logits. Keys and values go into a cache of ROOM places to a sequence."""

    def __init__(self, api, prompts, dtype):
        self.api, self.dtype, self.n = api, dtype, len(prompts)
        self.table = random((HEADS * D, HEADS + 2 * KEY_HEADS, D), 7, dtype)
        whole = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.cache = torch.full((2, self.n * ROOM, KEY_HEADS, D), float("nan"), dtype=dtype, device="cuda")
        self.key_offsets = torch.arange(0, self.n * ROOM + 1, ROOM, dtype=torch.int32, device="cuda")
        self.lengths, self.positions, self.tokens = whole(self.n), whole(self.n), whole(self.n)
        self.offsets = torch.arange(self.n + 1, dtype=torch.int32, device="cuda")
        self.out = torch.empty((self.n, HEADS, D), dtype=dtype, device="cuda")
        self.logp, self.top_values, self.top = torch.empty(self.n, device="cuda"), torch.empty((self.n, 3), device="cuda"), whole(self.n, 3)
        self.room = torch.empty(max(api.Attention.workspace(self.n, self.n * ROOM, self.n, HEADS, KEY_HEADS, D), 1), dtype=torch.uint8, device="cuda")
        # the prompts, all at once
        lens = [len(p) for p in prompts]
        words = torch.tensor(sum(prompts, []), device="cuda")
        at = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in lens])
        slots = torch.cat([torch.arange(n, device="cuda") + ROOM * i for i, n in enumerate(lens)])
        ends = torch.tensor([sum(lens[:i]) for i in range(self.n + 1)], dtype=torch.int32, device="cuda")
        out = torch.empty((len(words), HEADS, D), dtype=dtype, device="cuda")
        self.lengths.copy_(torch.tensor(lens))
        self.attend(words, at, slots, ends, out, None)
        last = ends[1:].long() - 1
        self.out.copy_(out[last])
        self.choose(None)
        self.positions.copy_(self.lengths)
        torch.cuda.synchronize()

    def attend(self, words, positions, slots, offsets, out, stream):
        api, wrap = self.api, self.api.as_tensor
        rows = self.table.index_select(0, words)
        q, k = torch.empty_like(rows[:, :HEADS]), torch.empty_like(rows[:, HEADS:HEADS + KEY_HEADS])
        how, at = dict(scaling=api.RotaryScaling(**SCALING), stream=stream), wrap(positions)
        api.rotary_into(wrap(q, "TWE"), wrap(rows[:, :HEADS], "TWE"), at, **how)
        api.rotary_into(wrap(k, "TWE"), wrap(rows[:, HEADS:HEADS + KEY_HEADS], "TWE"), at, **how)
        self.cache[0].index_copy_(0, slots, k)
        self.cache[1].index_copy_(0, slots, rows[:, HEADS + KEY_HEADS:])
        api.attention_into(wrap(out, "TWE"), wrap(q, "TWE"), wrap(self.cache[0], "TWE"), wrap(self.cache[1], "TWE"), wrap(offsets),
                           key_offsets=wrap(self.key_offsets), key_lengths=wrap(self.lengths), workspace=wrap(self.room), stream=stream)
        return rows, q, k

    def choose(self, stream):
        wrap = self.api.as_tensor
        self.api.log_probs_into(wrap(self.logp), wrap(self.out.view(self.n, HEADS * D)), wrap(self.tokens), top_values=wrap(self.top_values),
                                top_tokens=wrap(self.top), stream=stream)
        self.tokens.copy_(self.top[:, 0])

    def step(self, stream=None):
        slots = self.key_offsets[:-1].long() + self.positions.long()
        self.lengths += 1
        kept = self.attend(self.tokens.long(), self.positions, slots, self.offsets, self.out, stream)
        self.choose(stream)
        self.positions += 1
        return kept  # (what a captured step works on lives as long as this)

    def state(self):
        return [t.clone() for t in (self.out, self.top, self.top_values, self.tokens, self.lengths, self.positions)]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_answers_from_a_cache(api, dtype):
    """Captured steps against eager ones, bit by bit, and all that was answered against the definition of whole sequences."""
    prompts = [[3, 60, 17, 17, 2], [5], [9, 8, 7, 6, 5, 4, 3, 2, 1, 0, 63]]
    eager, replayed = Answers(api, prompts, dtype), Answers(api, prompts, dtype)
    graph = torch.cuda.CUDAGraph()
    first = eager.tokens.clone()
    with torch.cuda.graph(graph):
        kept = replayed.step(api.as_stream(torch.cuda.current_stream()))
    words, outs = [p + [int(t)] for p, t in zip(prompts, first)], []
    for _ in range(12):
        graph.replay()
        torch.cuda.synchronize()
        got = replayed.state()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager.state()))
        logits = got[0].view(len(prompts), -1).double()
        assert torch.equal(got[1].long(), logits.sort(dim=1, descending=True, stable=True)[1][:, :3])
        outs.append(got[0])
        for p, t in zip(words, got[3]):
            p.append(int(t))
    assert kept is not None
    # sequence by sequence, at the places of its tokens
    for b, (p, w) in enumerate(zip(prompts, words)):
        w = w[:-1]
        rows = replayed.table[torch.tensor(w, device="cuda")]
        assert int(replayed.lengths[b]) == len(w)
        keys, values = (c[ROOM * b:ROOM * b + len(w)] for c in replayed.cache)
        turned, e = ref.rotary(rows[:, HEADS:HEADS + KEY_HEADS].double(), torch.arange(len(w), device="cuda"), D, **SCALING)
        close(keys, turned, e, "cached keys")
        assert torch.equal(values, rows[:, HEADS + KEY_HEADS:])
        assert torch.isnan(replayed.cache[:, ROOM * b + len(w):ROOM * (b + 1)]).all()
        q = torch.empty((len(w), HEADS, D), dtype=dtype, device="cuda")
        api.rotary_into(api.as_tensor(q, "TWE"), api.as_tensor(rows[:, :HEADS].contiguous(), "TWE"),
                        api.as_tensor(torch.arange(len(w), device="cuda")), scaling=api.RotaryScaling(**SCALING))
        torch.cuda.synchronize()
        for n in range(HEADS):
            m = n // (HEADS // KEY_HEADS)
            want = ref.attention(q[:, n].double(), keys[:, m].double(), values[:, m].double(), D ** -0.5, True, dtype)
            got = torch.stack([o[b, n] for o in outs])
            close(got, want[0][len(p):], want[2][len(p):], "answers of sequence %d" % b)
    assert math.isfinite(float(replayed.top_values.sum()))
