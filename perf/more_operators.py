"""Between the embedding and the weight update of a model that trains on the image batches or answers from them: rotary
positions, attention over packed sequences and the log probabilities of tokens, as cases that can be timed and compared.

`listed()` names the smallest calls, ordinary ones and the largest of five operators (rotary, attention, its gradient, log
probabilities, their gradient); `draw()` gives further cases of the same ranges; `prepare()` makes what a program has in
hand before the call and `run()` is one pass: in plain torch operations in 32 bits, or, where `own` is true, by the calls of
this package. `work()` counts what a pass cannot do without. `exact()` is the definition in 64 bits.
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}
BASE = 10000.0     # of the rotary frequencies
SCALING = {"factor": 8.0, "original": 8192.0, "low": 1.0, "high": 4.0, "magnitude": 1.1}  # for contexts longer than those trained on
FARTHEST = 131072  # positions of the rotary cases
MOST_BYTES = 1.2e9  # of a drawn case: what a pass reads and writes (the largest listed one: 2.1 GB)
MOST_SCORES = 1.5e9  # of a drawn case: queries * keys * heads, with every sequence as long as the longest (listed: 4.3e9)


def listed():
    return [
        # queries and keys of the next token of eight conversations, far into long contexts: latency alone
        {"name": "token_rotary", "kind": "rotary", "n": 8, "heads": 40, "d": 128, "dims": 128, "type": "bf16", "positions": "i64",
         "interleaved": False, "scaled": True, "inverse": False},
        # queries and keys of long prompts, packed
        {"name": "prompt_rotary", "kind": "rotary", "n": 16384, "heads": 40, "d": 128, "dims": 128, "type": "bf16", "positions": "i64",
         "interleaved": False, "scaled": False, "inverse": False},
        # the next token of one conversation: its keys lie in a cache with room
        {"name": "token_attention", "kind": "attention", "b": 1, "longest": 1, "cache": 700, "heads": 32, "key_heads": 8, "d": 128,
         "type": "bf16", "causal": True, "stats": False, "of": 1},
        # the next tokens of sixteen conversations of up to 8192 tokens
        {"name": "tokens_attention", "kind": "attention", "b": 16, "longest": 1, "cache": 8191, "heads": 32, "key_heads": 8, "d": 128,
         "type": "bf16", "causal": True, "stats": False, "of": 2},
        # 196 patches and a caption of up to 77 tokens, for each of 64 images: every token sees its whole pair
        {"name": "pairs_attention", "kind": "attention", "b": 64, "longest": 273, "cache": 0, "heads": 12, "key_heads": 12, "d": 64,
         "type": "f16", "causal": False, "stats": True, "of": 3},
        # long prompts of different lengths, packed
        {"name": "prompts_attention", "kind": "attention", "b": 8, "longest": 4096, "cache": 0, "heads": 32, "key_heads": 8, "d": 128,
         "type": "bf16", "causal": True, "stats": True, "of": 4},
        # the pairs' backward pass
        {"name": "pairs_attention_grad", "kind": "attention_grad", "b": 64, "longest": 273, "cache": 0, "heads": 12, "key_heads": 12,
         "d": 64, "type": "f16", "causal": False, "of": 3},
        # and that of long sequences
        {"name": "long_attention_grad", "kind": "attention_grad", "b": 8, "longest": 2048, "cache": 0, "heads": 32, "key_heads": 8,
         "d": 128, "type": "bf16", "causal": True, "of": 5},
        # what a server reports with the next token of eight conversations
        {"name": "token_log_probs", "kind": "log_probs", "n": 8, "v": 32000, "type": "bf16", "tokens": "i64", "top": 8, "scale": 0.8},
        # the same of whole prompts, over a large vocabulary
        {"name": "prompt_log_probs", "kind": "log_probs", "n": 4096, "v": 128000, "type": "bf16", "tokens": "i64", "top": 5, "scale": 1.0},
        # the loss of one batch of captions (odd vocabulary, 32 bits), with entropy
        {"name": "captions_loss_grad", "kind": "log_probs_grad", "n": 1003, "v": 30011, "type": "f32", "tokens": "i32", "entropy": True,
         "scale": 1.0},
        # the loss of long sequences
        {"name": "long_loss_grad", "kind": "log_probs_grad", "n": 4096, "v": 128000, "type": "bf16", "tokens": "i64", "entropy": False,
         "scale": 1.0},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "attention_grad", "log_probs", "log_probs_grad"])
    while True:
        if kind == "rotary":
            d = rng.choice([32, 50, 64, 80, 96, 100, 128, 256])
            case = {"kind": kind, "n": _between(rng, 1, 32768), "heads": _between(rng, 1, 64), "d": d,
                    "dims": d if rng.random() < 0.6 else 2 * rng.randrange(1, d // 2 + 1), "type": rng.choice(["f32", "f16", "bf16", "bf16"]),
                    "positions": rng.choice(["i32", "i64"]), "interleaved": rng.random() < 0.5, "scaled": rng.random() < 0.5,
                    "inverse": rng.random() < 0.3}
        elif kind in ("attention", "attention_grad"):
            key_heads, gradient = rng.choice([1, 2, 3, 4, 8, 12]), kind == "attention_grad"
            case = {"kind": kind, "b": _between(rng, 1, 64),
                    "longest": 1 if not gradient and rng.random() < 0.3 else _between(rng, 16 if gradient else 1, 4096),
                    "cache": 0 if rng.random() < 0.6 else _between(rng, 1, 16384), "heads": key_heads * rng.choice([1, 1, 2, 3, 4, 8]),
                    "key_heads": key_heads, "d": rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128]), "type": rng.choice(["f16", "bf16"]),
                    "causal": rng.random() < 0.6, "of": rng.randrange(1 << 20)}
            if not gradient:
                case["stats"] = rng.random() < 0.5
            if case["b"] * case["longest"] * (case["longest"] + case["cache"]) * case["heads"] > MOST_SCORES * (0.5 if gradient else 1):
                continue
        else:
            case = {"kind": kind, "n": _between(rng, 1, 16384), "v": _between(rng, 500, 160000), "type": rng.choice(["f32", "f16", "bf16", "bf16"]),
                    "tokens": rng.choice(["i32", "i64"]), "scale": rng.choice([1.0, 1.0, 0.7, 1.6])}
            if kind == "log_probs":
                case["top"] = rng.choice([0, 1, 5, 20, 32])
            else:
                case["entropy"] = rng.random() < 0.5
        if work(case)["bytes"] <= MOST_BYTES:
            return case


def _lengths(case):
    """(queries, keys) of each sequence: the first is as long as the case says, some of the others have nothing."""
    rng, made = random.Random(case["of"]), []
    for i in range(case["b"]):
        queries = case["longest"] if i == 0 else 0 if rng.random() < 0.03 else rng.randint(-(-case["longest"] // 4), case["longest"])
        cached = case["cache"] if i == 0 else rng.randint(case["cache"] // 4, case["cache"])
        made.append((queries, queries + cached))
    return made


# ---- inputs ----------------------------------------------------------------------------------------------------------
class _Source:
    """Random inputs on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, scale=1.0, dtype="f32"):
        return (torch.randn(shape, generator=self.gen, device="cuda") * scale).to(TORCH[dtype])

    def uniform(self, shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def whole(self, lo, hi, shape, dtype):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda").to(TORCH[dtype])


def _whole(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    made = [0]
    for n in lengths:
        made.append(made[-1] + n)
    return made


def _gradients(case):
    """How large gradients are: losses are scaled up where 16 bits would lose small ones."""
    return 1.0 if case["type"] == "f16" else 1e-3


def _prepare_attention(src, case, s):
    """One projection's result holds queries, keys and values side by side, unless the keys lie in a cache: there each
    sequence has room for the longest."""
    lengths = _lengths(case)
    queries, keys = [a for a, _ in lengths], [b for _, b in lengths]
    rows, heads, key_heads, d = sum(queries), case["heads"], case["key_heads"], case["d"]
    s["offsets"], s["key_offsets"], s["key_lengths"] = _whole(_starts(queries)), None, None
    s["longest"], s["longest_keys"], s["scale"] = max(queries), max(keys), d ** -0.5
    if case["cache"] == 0:
        qkv = src.normal((rows, heads + 2 * key_heads, d))
        qkv[:, :heads] *= 1.5
        s["q"], s["k"], s["v"] = qkv.to(TORCH[case["type"]]).split([heads, key_heads, key_heads], 1)
    else:
        room = case["longest"] + case["cache"]
        s["q"] = src.normal((rows, heads, d), 1.5, case["type"])
        s["k"], s["v"] = (src.normal((case["b"] * room, key_heads, d), 1.0, case["type"]) for _ in range(2))
        s["key_offsets"], s["key_lengths"] = _whole([room * i for i in range(case["b"] + 1)]), _whole(keys)
    # where each row stands: its sequence, and its place there
    counts = torch.tensor(queries, device="cuda")
    s["sequence"] = torch.repeat_interleave(torch.arange(case["b"], device="cuda"), counts)
    s["place"] = torch.arange(rows, device="cuda") - s["offsets"].long()[s["sequence"]]
    if case["kind"] == "attention_grad":
        s["grad"] = src.normal((rows, heads, d), _gradients(case), case["type"])
        s["out"], s["lse"] = _plain_attention(s, dict(case, stats=True))


def prepare(case, seed):
    kind, src, s = case["kind"], _Source(seed), {"kind": case["kind"], "case": case}
    if kind == "rotary":
        s["x"] = src.normal((case["n"], case["heads"], case["d"]), 1.0, case["type"])
        s["positions"] = src.whole(0, FARTHEST, (case["n"],), case["positions"])
    elif kind in ("attention", "attention_grad"):
        _prepare_attention(src, case, s)
    else:
        # a model's logits: most words are unlikely, a few stand out, and 16 bits make many of them equal
        x = src.normal((case["n"], case["v"]), 2.0)
        x += 6 * (src.uniform((case["v"],)) > 0.999)
        s["logits"], s["tokens"] = x.to(TORCH[case["type"]]), src.whole(0, case["v"], (case["n"],), case["tokens"])
        s["tokens"][src.uniform((case["n"],)) < 0.1] = -1  # padding
        if kind == "log_probs_grad":
            s["grad"] = torch.full((case["n"],), -1e3 * _gradients(case) / case["n"], device="cuda")
            z = s["logits"].float() * case["scale"]
            s["lse"] = torch.logsumexp(z, 1)
            if case["entropy"]:
                s["entropy"] = s["lse"] - (torch.exp(z - s["lse"][:, None]) * z).sum(1)
                s["grad_entropy"] = src.normal((case["n"],), 1e2 * _gradients(case) / case["n"])
    return s


# ---- the operators in plain operations, in 32 bits ---------------------------------------------------------------------
def _frequencies(case):
    """Of each pair of dimensions, in 64 bits, turned down for long contexts."""
    f = BASE ** (-torch.arange(0, case["dims"], 2, dtype=torch.float64, device="cuda") / case["dims"])
    if not case["scaled"]:
        return f, 1.0
    turns = SCALING["original"] * f / (2 * math.pi)
    kept = ((turns - SCALING["low"]) / (SCALING["high"] - SCALING["low"])).clamp(0, 1)
    return f * (kept + (1 - kept) / SCALING["factor"]), SCALING["magnitude"]


def _plain_rotary(s, case):
    f, magnitude = _frequencies(case)
    angles = (s["positions"].double()[:, None] * f)[:, None, :]  # (far positions: in 32 bits the angle would be gone)
    cos, sin = (torch.cos(angles) * magnitude).float(), (torch.sin(angles) * magnitude).float()
    if case["inverse"]:
        sin = -sin
    x, half = s["x"].float(), case["dims"] // 2
    out = x.clone()
    first, second = (slice(0, case["dims"], 2), slice(1, case["dims"], 2)) if case["interleaved"] else (slice(0, half), slice(half, case["dims"]))
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., first] * sin + x[..., second] * cos
    return out.to(TORCH[case["type"]])


def _padded(t, starts, length, key_heads):
    """Packed rows [T, heads, d] as [sequences * key_heads, (heads of a key head, rows), d], in 32 bits; behind each sequence's
    end stand other rows."""
    at = (starts.long()[:, None] + torch.arange(length, device="cuda")).clamp_(max=max(0, t.shape[0] - 1))
    t = t[at].float().unflatten(2, (key_heads, -1)).permute(0, 2, 3, 1, 4)  # [sequences, key_heads, group, rows, d]
    return t.reshape(t.shape[0] * key_heads, -1, t.shape[-1])


def _packed(t, s, case, heads):
    """The opposite of _padded, for the rows of the queries."""
    t = t.view(case["b"], heads, -1, t.shape[-1])
    return t[s["sequence"], :, s["place"]]


def _scores(s, case, q, k):
    """scale * q . k with -inf where a row does not see a key."""
    n, m = s["longest"], s["longest_keys"]
    lengths = s["offsets"][1:] - s["offsets"][:-1]
    keys = lengths if s["key_lengths"] is None else s["key_lengths"]
    j = torch.arange(m, device="cuda")
    hidden = (j >= keys[:, None])[:, None, :]
    if case["causal"]:
        i = torch.arange(n, device="cuda")
        hidden = hidden | (j > i[:, None] + (keys - lengths)[:, None, None])
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(s["scale"])
    scores.view(case["b"], case["heads"], n, m).masked_fill_(hidden[:, None], -math.inf)
    return scores


def _key_starts(s):
    return (s["offsets"] if s["key_offsets"] is None else s["key_offsets"])[:-1]


def _plain_attention(s, case):
    q = _padded(s["q"], s["offsets"][:-1], s["longest"], case["key_heads"])
    k, v = (_padded(s[name], _key_starts(s), s["longest_keys"], case["key_heads"]) for name in ("k", "v"))
    p = _scores(s, case, q, k)
    top = p.amax(2, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = p.sub_(top).exp_()
    total = p.sum(2, keepdim=True)
    out = torch.bmm(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    out = _packed(out, s, case, case["heads"]).to(TORCH[case["type"]])
    if not case["stats"]:
        return [out]
    return [out, _packed(top + torch.log(total), s, case, case["heads"])[..., 0].t().contiguous()]


def _plain_attention_grad(s, case):
    key_heads, n = case["key_heads"], s["longest"]
    starts = s["offsets"][:-1]
    q, grad, out = (_padded(s[name], starts, n, key_heads) for name in ("q", "grad", "out"))
    k, v = (_padded(s[name], _key_starts(s), s["longest_keys"], key_heads) for name in ("k", "v"))
    lse = _padded(s["lse"].t()[..., None], starts, n, key_heads)
    # (rows behind a sequence's end have no part in the sums over rows)
    there = (torch.arange(n, device="cuda") < (s["offsets"][1:] - starts)[:, None]).repeat_interleave(key_heads, 0)
    there = there.repeat(1, case["heads"] // key_heads)[..., None]
    grad = grad * there
    p = _scores(s, case, q, k).sub_(torch.where(lse == -math.inf, torch.zeros_like(lse), lse)).exp_()
    p *= there
    to_v = torch.bmm(p.transpose(1, 2).contiguous(), grad)
    p *= torch.bmm(grad, v.transpose(1, 2).contiguous()).sub_((grad * out).sum(2, keepdim=True))
    to_q = torch.bmm(p, k).mul_(s["scale"])
    to_k = torch.bmm(p.transpose(1, 2).contiguous(), q).mul_(s["scale"])
    kind = TORCH[case["type"]]
    made = [_packed(to_q, s, case, case["heads"]).to(kind)]
    # each key's gradient at its place; places of a cache that no sequence fills are left as they were: zeros
    keys = (s["offsets"][1:] - starts) if s["key_lengths"] is None else s["key_lengths"]
    filled = torch.arange(s["longest_keys"], device="cuda") < keys[:, None]
    at = (_key_starts(s).long()[:, None] + torch.arange(s["longest_keys"], device="cuda"))[filled]
    for part in (to_k, to_v):
        whole = torch.zeros(s["k"].shape, dtype=kind, device="cuda")
        whole[at] = part.view(case["b"], key_heads, -1, case["d"]).transpose(1, 2)[filled].to(kind)
        made.append(whole)
    return made


def _plain_log_probs(s, case):
    z = s["logits"].float() * case["scale"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    entropy = (torch.log(total) - (e * (z - top)).sum(1, keepdim=True) / total)[:, 0]
    tokens = s["tokens"].long()
    there = (tokens >= 0) & (tokens < case["v"])
    at = torch.where(there, tokens, torch.zeros_like(tokens))[:, None]
    logp = torch.where(there, (z.gather(1, at) - lse)[:, 0], torch.zeros_like(entropy))
    if case["top"] == 0:
        return [logp, entropy, lse[:, 0]]
    # whole numbers in the order of the values, of equal ones the first word's is the largest
    bits = s["logits"].float().add(0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + ((1 << 31) - torch.arange(case["v"], device="cuda"))
    words = torch.topk(order, case["top"], 1, sorted=True).indices
    return [logp, entropy, lse[:, 0], z.gather(1, words) - lse, words.int()]


def _plain_log_probs_grad(s, case):
    z = s["logits"].float() * case["scale"]
    logp = z - s["lse"][:, None]
    p = torch.exp(logp)
    tokens = s["tokens"].long()
    there = (tokens >= 0) & (tokens < case["v"])
    grad = torch.where(there, s["grad"], torch.zeros_like(s["grad"]))[:, None]
    to_z = p * -grad
    to_z.scatter_add_(1, torch.where(there, tokens, torch.zeros_like(tokens))[:, None], grad)
    if case["entropy"]:
        to_z -= p * s["grad_entropy"][:, None] * (logp + s["entropy"][:, None])
    return (to_z * case["scale"]).to(TORCH[case["type"]])


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return _RUN_OWN[case["kind"]](state, case, _package()) if own else _RUN_PLAIN[case["kind"]](state, case)


_loaded = []


def _package():
    if not _loaded:
        from __graft_entry__ import load_package
        load_package()
        import cvcuda_amd.pyapi as cvcuda
        _loaded.append(cvcuda)
    return _loaded[0]


def _own_rotary(s, case, cvcuda):
    out, wrap = torch.empty_like(s["x"]), cvcuda.as_tensor
    cvcuda.rotary_into(wrap(out), wrap(s["x"]), wrap(s["positions"]), case["dims"], base=BASE, interleaved=case["interleaved"],
                       scaling=cvcuda.RotaryScaling(**SCALING) if case["scaled"] else None, inverse=case["inverse"])
    return out


def _keys(s, wrap):
    if s["key_offsets"] is None:
        return {}
    return {"key_offsets": wrap(s["key_offsets"]), "key_lengths": wrap(s["key_lengths"])}


def _own_attention(s, case, cvcuda):
    wrap, made = cvcuda.as_tensor, [torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")]
    if case["stats"]:
        made.append(torch.empty((case["heads"], s["q"].shape[0]), device="cuda"))
    cvcuda.attention_into(wrap(made[0]), wrap(s["q"]), wrap(s["k"]), wrap(s["v"]), wrap(s["offsets"]), causal=case["causal"],
                          scale=s["scale"], lse=wrap(made[1]) if case["stats"] else None, **_keys(s, wrap))
    return made


def _own_attention_grad(s, case, cvcuda):
    wrap = cvcuda.as_tensor
    if s["key_offsets"] is None:  # side by side, as the projection's gradient takes them
        whole = torch.empty((s["q"].shape[0], case["heads"] + 2 * case["key_heads"], case["d"]), dtype=s["q"].dtype, device="cuda")
        made = whole.split([case["heads"], case["key_heads"], case["key_heads"]], 1)
    else:
        made = [torch.empty_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])]
    cvcuda.attention_grad_into(*[wrap(t) for t in made], wrap(s["grad"]), wrap(s["q"]), wrap(s["k"]), wrap(s["v"]), wrap(s["out"]),
                               wrap(s["lse"]), wrap(s["offsets"]), causal=case["causal"], scale=s["scale"], **_keys(s, wrap))
    return list(made)


def _own_log_probs(s, case, cvcuda):
    wrap, n, k = cvcuda.as_tensor, case["n"], case["top"]
    made = [torch.empty(n, device="cuda") for _ in range(3)]
    more = {}
    if k:
        made += [torch.empty((n, k), device="cuda"), torch.empty((n, k), dtype=torch.int32, device="cuda")]
        more = {"top_values": wrap(made[3]), "top_tokens": wrap(made[4])}
    cvcuda.log_probs_into(wrap(made[0]), wrap(s["logits"]), wrap(s["tokens"]), case["scale"], entropy=wrap(made[1]), lse=wrap(made[2]), **more)
    return made


def _own_log_probs_grad(s, case, cvcuda):
    wrap, made = cvcuda.as_tensor, torch.empty_like(s["logits"])
    more = {"entropy": wrap(s["entropy"]), "grad_entropy": wrap(s["grad_entropy"])} if case["entropy"] else {}
    cvcuda.log_probs_grad_into(wrap(made), wrap(s["logits"]), wrap(s["tokens"]), wrap(s["lse"]), wrap(s["grad"]), case["scale"], **more)
    return made


_RUN_PLAIN = {"rotary": _plain_rotary, "attention": _plain_attention, "attention_grad": _plain_attention_grad,
              "log_probs": _plain_log_probs, "log_probs_grad": _plain_log_probs_grad}
_RUN_OWN = {"rotary": _own_rotary, "attention": _own_attention, "attention_grad": _own_attention_grad,
            "log_probs": _own_log_probs, "log_probs_grad": _own_log_probs_grad}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def _seen(queries, keys, causal):
    """Pairs of a row and a key that it sees."""
    if not causal:
        return queries * keys
    return queries * (keys - queries) + queries * (queries + 1) // 2  # (no sequence has fewer keys than rows)


def work(case):
    kind = case["kind"]
    if kind == "rotary":
        px = case["n"] * case["heads"] * case["d"]
        return {"bytes": 2 * px * SIZE[case["type"]] + case["n"] * SIZE[case["positions"]], "flops": 3 * case["n"] * case["heads"] * case["dims"]}
    if kind in ("attention", "attention_grad"):
        lengths, e, d = _lengths(case), SIZE[case["type"]], case["d"]
        rows, keys = sum(a for a, _ in lengths) * case["heads"], sum(b for a, b in lengths if a) * case["key_heads"]
        pairs = sum(_seen(a, b, case["causal"]) for a, b in lengths) * case["heads"]
        if kind == "attention":
            return {"bytes": 2 * rows * d * e + 2 * keys * d * e + (4 * rows if case["stats"] else 0), "flops": 4 * pairs * d}
        return {"bytes": 4 * rows * d * e + 4 * keys * d * e + 4 * rows, "flops": 10 * pairs * d}
    px = case["n"] * case["v"]
    if kind == "log_probs":
        return {"bytes": px * SIZE[case["type"]] + case["n"] * (SIZE[case["tokens"]] + 12 + 8 * case["top"]), "flops": 5 * px}
    return {"bytes": 2 * px * SIZE[case["type"]] + case["n"] * (SIZE[case["tokens"]] + (16 if case["entropy"] else 8)),
            "flops": (7 if case["entropy"] else 4) * px}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    return {"rotary": _exact_rotary, "attention": _exact_attention, "attention_grad": _exact_attention_grad, "log_probs": _exact_log_probs,
            "log_probs_grad": _exact_log_probs_grad}[kind](s, case)


def _exact_rotary(s, case):
    """Pairs as complex numbers, turned."""
    x, half = s["x"].double(), case["dims"] // 2
    f = [BASE ** (-2.0 * i / case["dims"]) for i in range(half)]
    if case["scaled"]:
        for i, v in enumerate(f):
            share = (SCALING["original"] * v / (2 * math.pi) - SCALING["low"]) / (SCALING["high"] - SCALING["low"])
            share = min(1.0, max(0.0, share))
            f[i] = share * v + (1 - share) * v / SCALING["factor"]
    turn = torch.outer(s["positions"].double(), torch.tensor(f, dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(turn, SCALING["magnitude"] if case["scaled"] else 1.0), -turn if case["inverse"] else turn)[:, None]
    part = x[..., :case["dims"]]
    pairs = part.unflatten(-1, (half, 2)) if case["interleaved"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    turned = turned if case["interleaved"] else turned.transpose(-1, -2)
    return torch.cat([turned.reshape(part.shape), x[..., case["dims"]:]], -1)


def _each(s, case):
    """(rows, places of the keys, which keys each row sees) of every sequence that has rows."""
    first = 0
    for b, (queries, keys) in enumerate(_lengths(case)):
        at = first if s["key_offsets"] is None else int(s["key_offsets"][b])
        if queries:
            sees = torch.ones((queries, keys), dtype=torch.bool, device="cuda")
            yield slice(first, first + queries), slice(at, at + keys), sees.tril(keys - queries) if case["causal"] else sees
        first += queries


def _exact_attention(s, case):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros((case["heads"], s["q"].shape[0]), dtype=torch.float64, device="cuda")
    group = case["heads"] // case["key_heads"]
    for rows, keys, sees in _each(s, case):
        for h in range(case["heads"]):
            scores = s["q"][rows, h].double() @ s["k"][keys, h // group].double().t().contiguous() * s["scale"]
            scores = torch.where(sees, scores, -math.inf)
            lse[h, rows] = torch.logsumexp(scores, 1)
            out[rows, h] = torch.softmax(scores, 1) @ s["v"][keys, h // group].double()
    return [out, lse] if case["stats"] else [out]


def _exact_attention_grad(s, case):
    to_q, to_k, to_v = (torch.zeros(s[name].shape, dtype=torch.float64, device="cuda") for name in ("q", "k", "v"))
    group = case["heads"] // case["key_heads"]
    for rows, keys, sees in _each(s, case):
        for h in range(case["heads"]):
            q, k, v, g = (s[name][at, head].double() for name, at, head in (("q", rows, h), ("k", keys, h // group), ("v", keys, h // group), ("grad", rows, h)))
            p = torch.exp(q @ k.t().contiguous() * s["scale"] - s["lse"][h, rows, None].double()) * sees
            inner = p * (g @ v.t().contiguous() - (g * s["out"][rows, h].double()).sum(1, keepdim=True))
            to_q[rows, h] = s["scale"] * (inner @ k)
            to_k[keys, h // group] += s["scale"] * (inner.t().contiguous() @ q)
            to_v[keys, h // group] += p.t().contiguous() @ g
    return [to_q, to_k, to_v]


def _exact_log_probs(s, case):
    made = [torch.zeros(case["n"], dtype=torch.float64, device="cuda") for _ in range(3)]
    top = torch.zeros((case["n"], case["top"]), dtype=torch.float64, device="cuda")
    for at in range(0, case["n"], 512):
        z = s["logits"][at:at + 512].double() * case["scale"]
        logp = torch.log_softmax(z, 1)
        tokens = s["tokens"][at:at + 512].long()
        made[0][at:at + 512] = torch.where(tokens < 0, 0.0, logp[torch.arange(len(z), device="cuda"), tokens.clamp(min=0)])
        made[1][at:at + 512] = -(logp.exp() * logp).sum(1)
        made[2][at:at + 512] = torch.logsumexp(z, 1)
        top[at:at + 512] = torch.topk(logp, case["top"], 1).values
    return made + [top, None] if case["top"] else made


def _exact_log_probs_grad(s, case):
    made = torch.empty((case["n"], case["v"]), dtype=torch.float64, device="cuda")
    for at in range(0, case["n"], 512):
        part = slice(at, at + 512)
        logp = s["logits"][part].double() * case["scale"] - s["lse"][part, None].double()
        tokens, g = s["tokens"][part].long(), s["grad"][part, None].double()
        hit = torch.arange(case["v"], device="cuda") == tokens[:, None]
        made[part] = torch.where(tokens[:, None] < 0, 0.0, g * (hit.double() - logp.exp()))
        if case["entropy"]:
            made[part] -= s["grad_entropy"][part, None].double() * logp.exp() * (logp + s["entropy"][part, None].double())
    return made * case["scale"]
