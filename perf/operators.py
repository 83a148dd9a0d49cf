"""The work behind the image batches: the row operators and the weight update of a model that trains on them or answers
from them, as cases that can be timed and compared.

`listed()` names the smallest calls, ordinary ones and the largest of five operators (layer norm, its gradient, embedding
lookup, its gradient, AdamW over many tensors); `draw()` gives further cases of the same ranges; `prepare()` makes what a
program has in hand before the call and `run()` is one pass: in plain torch operations in 32 bits, or, where `own` is
true, by the calls of this package. `work()` counts what a pass cannot do without. `exact()` is the definition in 64 bits.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}
EPSILON = 1e-5  # of layer norm
BLOCK = 256     # elements of an 8-bit state that share a scale
ADAMW = {"lr": 3e-4, "betas": (0.9, 0.98), "epsilon": 1e-8, "weight_decay": 0.05}
FIRST_STEP = 100  # the states that prepare() makes are those of a program that has trained for a while
MOST_BYTES = 2e9  # of a drawn case: what a pass reads and writes (the largest listed one: 5.9 GB)


def listed():
    return [
        # the next token of eight conversations: rows of a table, where only latency counts
        {"name": "next_tokens", "kind": "embedding", "n": 8, "v": 32000, "d": 4096, "type": "bf16", "out": "bf16", "tokens": "i64"},
        # a batch of captions and prompts, from 32-bit weights to the 16 bits that the layers run in
        {"name": "prompts", "kind": "embedding", "n": 32768, "v": 100003, "d": 2048, "type": "f32", "out": "bf16", "tokens": "i32"},
        # the captions of one batch of images (a few hundred words, odd width), 32-bit gradients
        {"name": "captions_grad", "kind": "embedding_grad", "n": 1003, "v": 30011, "d": 515, "type": "f32", "grad": "f32",
         "tokens": "i64", "padding": True, "accumulate": False},
        # the gradient of a large vocabulary from a long batch, padded at the ends
        {"name": "vocabulary_grad", "kind": "embedding_grad", "n": 65536, "v": 128000, "d": 2048, "type": "bf16", "grad": "f32",
         "tokens": "i64", "padding": True, "accumulate": False},
        # one token's state on its way through a model that answers
        {"name": "token_norm", "kind": "layer_norm", "rows": 1, "d": 4096, "type": "bf16", "weights": "bf16", "stats": False},
        # the patches of a batch of 64 crops of 224 x 224: 14 x 14 patches of 16 x 16 x 3 values each
        {"name": "patch_norm", "kind": "layer_norm", "rows": 12544, "d": 768, "type": "f16", "weights": "f32", "stats": True},
        # the same of long sequences of wide rows: the largest call of the forward pass
        {"name": "long_norm", "kind": "layer_norm", "rows": 65536, "d": 4096, "type": "bf16", "weights": "bf16", "stats": False},
        # the patches' backward pass
        {"name": "patch_norm_grad", "kind": "layer_norm_grad", "rows": 12544, "d": 768, "type": "f16", "weights": "f32"},
        # and that of the long sequences
        {"name": "long_norm_grad", "kind": "layer_norm_grad", "rows": 65536, "d": 4096, "type": "bf16", "weights": "bf16"},
        # a classifier's head alone is trained: a few tensors, 32 bits throughout
        {"name": "adamw_head", "kind": "adamw", "layers": 0, "w": 768, "h": 1000, "grad": "f32", "copy": None, "bits": 32},
        # every tensor of a model in mixed precision: 16-bit gradients, 32-bit weights and states, 16-bit copies of the weights
        {"name": "adamw_model", "kind": "adamw", "layers": 12, "w": 1280, "h": 4096, "grad": "bf16", "copy": "bf16", "bits": 32},
        # the same with states of 8 bits; the pass also gives the states' values, as a program that saves them does
        {"name": "adamw_model_8bit", "kind": "adamw", "layers": 12, "w": 1024, "h": 2816, "grad": "bf16", "copy": None, "bits": 8},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n - 1 if n == 3072 else n


def _width(rng, lo, hi):
    """A row's width: a multiple of 64 as most models have it, or any number."""
    d = _between(rng, lo, hi)
    if rng.random() < 0.6:
        d = max(64, d // 64 * 64)
    return d + 64 if d == 3072 else d


def draw(rng):
    kind = rng.choice(["embedding", "embedding_grad", "layer_norm", "layer_norm_grad", "adamw"])
    kinds = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")]
    while True:
        if kind == "embedding":
            out, table = rng.choice(kinds)
            case = {"kind": kind, "n": _between(rng, 1, 65536), "v": _between(rng, 500, 160000), "d": _width(rng, 60, 8192),
                    "type": table, "out": out, "tokens": rng.choice(["i32", "i64"])}
        elif kind == "embedding_grad":
            of, grad = rng.choice(kinds)
            case = {"kind": kind, "n": _between(rng, 1, 65536), "v": _between(rng, 500, 160000), "d": _width(rng, 60, 8192),
                    "type": of, "grad": grad, "tokens": rng.choice(["i32", "i64"]), "padding": rng.random() < 0.5,
                    "accumulate": rng.random() < 0.3}
        elif kind == "layer_norm":
            of, weights = rng.choice(kinds)
            case = {"kind": kind, "rows": _between(rng, 1, 65536), "d": _width(rng, 60, 12288), "type": of, "weights": weights,
                    "stats": rng.random() < 0.5}
        elif kind == "layer_norm_grad":
            of, weights = rng.choice(kinds)
            case = {"kind": kind, "rows": _between(rng, 16, 65536), "d": _width(rng, 60, 12288), "type": of, "weights": weights}
        else:
            case = {"kind": kind, "layers": rng.randrange(0, 9), "w": _width(rng, 60, 1536), "h": _width(rng, 100, 4096),
                    "grad": rng.choice(["f32", "bf16", "f16"]), "copy": rng.choice([None, "bf16", "f16"]), "bits": rng.choice([32, 32, 8])}
        if work(case)["bytes"] <= MOST_BYTES:
            return case


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _shapes(case):
    """The tensors of a model of `layers` layers: projections, biases and norms, and a head."""
    w, h = case["w"], case["h"]
    layer = [(w, w), (w,), (w, w), (w,), (w, w), (w,), (w, w), (w,), (h, w), (h,), (w, h), (w,), (w,), (w,), (w,), (w,)]
    return [s for _ in range(case["layers"]) for s in layer] + [(h, w), (h,), (w,), (w,)]


def _places(case):
    """(first element, count, shape) of each tensor in one buffer, as an allocator places them, and the buffer's length."""
    places, at = [], 0
    for shape in _shapes(case):
        count = math.prod(shape)
        places.append((at, count, shape))
        at += -(-count // BLOCK) * BLOCK
    return places, at


class _Source:
    """Random inputs on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, scale=1.0, dtype="f32"):
        return (torch.randn(shape, generator=self.gen, device="cuda") * scale).to(TORCH[dtype])

    def uniform(self, shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def tokens(self, n, v, dtype):
        """Words as text has them: the k-th most frequent one about 1/k as often as the first."""
        u = torch.rand((n,), generator=self.gen, device="cuda", dtype=torch.float64)
        return (torch.exp(u * math.log(v + 1)) - 1).to(torch.int64).clamp_(0, v - 1).to(TORCH[dtype])

    def rows(self, rows, d, dtype):
        """States of a model: a mean that differs by row, and a few columns far larger than the others."""
        x = torch.randn((rows, d), generator=self.gen, device="cuda")
        x *= 1 + 20 * (self.uniform((d,)) > 0.995)
        x += 0.3 * self.normal((rows, 1))
        return x.to(TORCH[dtype])


def _normal_state(src, case, s):
    """Weights, gradients and moments of AdamW. Between tensors the buffers hold zeros."""
    places, length = _places(case)
    used = torch.zeros(length, device="cuda")
    for at, count, _ in places:
        used[at:at + count] = 1
    s["params"] = src.normal(length, 0.02) * used
    grads = src.normal(length, 1e-3) * used
    s["m"] = src.normal(length, 3e-4) * used
    s["v"] = (src.normal(length, 1e-3).square_() + 1e-9) * used
    s["grads"] = grads.to(TORCH[case["grad"]])
    s["grad_scale"] = 0.5 + 0.5 * src.uniform((1,))  # a clipped gradient's factor
    s["copies"] = s["params"].to(TORCH[case["copy"]]) if case["copy"] else None
    s["step"] = FIRST_STEP
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _encode_moment(s["m"])
        s["v"], s["v_scale"] = _encode_variance(s["v"])


def prepare(case, seed):
    kind, src, s = case["kind"], _Source(seed), {"kind": case["kind"], "case": case}
    if kind == "embedding":
        s["table"] = src.normal((case["v"], case["d"]), 0.02, case["type"])
        s["tokens"] = src.tokens(case["n"], case["v"], case["tokens"])
    elif kind == "embedding_grad":
        s["tokens"] = src.tokens(case["n"], case["v"], case["tokens"])
        if case["padding"]:  # the ends of the sequences
            s["tokens"][src.uniform((case["n"],)) < 0.1] = 0
        s["grad"] = src.normal((case["n"], case["d"]), 1e-3, case["type"])
        s["table"] = src.normal((case["v"], case["d"]), 1e-3, case["grad"])  # an earlier batch's, where it is added to
    elif kind in ("layer_norm", "layer_norm_grad"):
        s["x"] = src.rows(case["rows"], case["d"], case["type"])
        s["gamma"] = 1 + src.normal((case["d"],), 0.1)
        s["gamma"], s["beta"] = s["gamma"].to(TORCH[case["weights"]]), src.normal((case["d"],), 0.1, case["weights"])
        if kind == "layer_norm_grad":
            s["grad"] = src.normal((case["rows"], case["d"]), 1e-2, case["type"])
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square_().mean(1) + EPSILON)
    else:
        _normal_state(src, case, s)
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program that uses this package keeps beside its weights: their tensors, and those of the buffers that stay."""
    from __graft_entry__ import load_package
    load_package()
    import cvcuda_amd.pyapi as cvcuda
    s["cvcuda"] = cvcuda
    kept = ("table", "gamma", "beta") if s["kind"] != "adamw" else ("grad_scale",)
    s["kept"] = {name: cvcuda.as_tensor(s[name]) for name in kept if name in s}
    if s["kind"] == "adamw":
        places, _ = _places(s["case"])
        for name in ("params", "grads", "m", "v", "copies"):
            if s[name] is not None:
                s["kept"][name] = [cvcuda.as_tensor(s[name][at:at + count].view(shape)) for at, count, shape in places]
        if s["case"]["bits"] == 8:
            for name in ("m", "v"):
                scales = s[name + "_scale"]
                s["kept"][name + "_scale"] = [cvcuda.as_tensor(scales[at // BLOCK:-(-(at + count) // BLOCK)]) for at, count, _ in places]
                s[name + "_values"] = torch.zeros(s["params"].numel(), device="cuda")
                s["kept"][name + "_values"] = [cvcuda.as_tensor(s[name + "_values"][at:at + count].view(shape)) for at, count, shape in places]


# ---- the operators in plain operations, in 32 bits ---------------------------------------------------------------------
def _plain_embedding(s, case):
    rows = s["table"][s["tokens"]].float()
    return (rows * math.sqrt(case["d"])).to(TORCH[case["out"]])


def _plain_embedding_grad(s, case):
    grad = s["grad"].float()
    if case["padding"]:
        grad = grad * (s["tokens"] != 0)[:, None]
    total = torch.zeros((case["v"], case["d"]), device="cuda").index_add_(0, s["tokens"], grad).mul_(math.sqrt(case["d"]))
    if case["accumulate"]:
        total += s["table"]
    s["table"].copy_(total)
    return s["table"]


def _plain_layer_norm(s, case):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPSILON)
    y = (centred * rstd * s["gamma"].float() + s["beta"].float()).to(TORCH[case["type"]])
    return [y, mean[:, 0], rstd[:, 0]] if case["stats"] else [y]


def _plain_layer_norm_grad(s, case):
    grad, rstd = s["grad"].float(), s["rstd"][:, None]
    unit = (s["x"].float() - s["mean"][:, None]) * rstd
    w = grad * s["gamma"].float()
    to_x = rstd * (w - w.mean(1, keepdim=True) - unit * (w * unit).mean(1, keepdim=True))
    kind, weights = TORCH[case["type"]], TORCH[case["weights"]]
    return [to_x.to(kind), (grad * unit).sum(0).to(weights), grad.sum(0).to(weights)]


def _decode_moment(codes, scale):
    t = codes.float().view(-1, BLOCK) * (1 / 127)
    return (t * t.abs() * scale[:, None]).view(-1)


def _decode_variance(codes, scale):
    t = codes.float().view(-1, BLOCK) * (1 / 255)
    t = t * t
    return (t * t * scale[:, None]).view(-1)


def _shares(blocks, scale):
    """Each value over its block's largest, 0 in a block of zeros."""
    return torch.where(scale[:, None] > 0, blocks / scale[:, None], torch.zeros_like(blocks))


def _encode_moment(m):
    blocks = m.view(-1, BLOCK)
    scale = blocks.abs().amax(1)
    codes = (_shares(blocks.abs(), scale).sqrt() * 127).round() * blocks.sign()
    return codes.to(torch.int8).view(-1), scale


def _encode_variance(v):
    blocks = v.view(-1, BLOCK)
    scale = blocks.amax(1)
    codes = (_shares(blocks, scale).sqrt().sqrt() * 255).round()
    return torch.maximum(codes, (blocks > 0).float()).to(torch.uint8).view(-1), scale


def _plain_adamw(s, case):
    lr, (beta1, beta2), eps, decay = ADAMW["lr"], ADAMW["betas"], ADAMW["epsilon"], ADAMW["weight_decay"]
    t, short = s["step"], case["bits"] == 8
    g = s["grads"].float() * s["grad_scale"]
    m = _decode_moment(s["m"], s["m_scale"]) if short else s["m"]
    v = _decode_variance(s["v"], s["v_scale"]) if short else s["v"]
    m.mul_(beta1).add_(g * (1 - beta1))
    v.mul_(beta2).add_(g * (1 - beta2) * g)
    root = v.sqrt().mul_(1 / math.sqrt(1 - beta2 ** t)).add_(eps)
    s["params"].mul_(1 - lr * decay).sub_((m / root).mul_(lr / (1 - beta1 ** t)))
    if short:
        codes, s["m_scale"] = _encode_moment(m)
        s["m"].copy_(codes)
        codes, s["v_scale"] = _encode_variance(v)
        s["v"].copy_(codes)
        m, v = _decode_moment(s["m"], s["m_scale"]), _decode_variance(s["v"], s["v_scale"])
    if s["copies"] is None:
        return [s["params"], m, v]
    s["copies"].copy_(s["params"])
    return [s["params"], m, v, s["copies"]]


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    case, s = state["case"], state
    if case["kind"] == "adamw":
        s["step"] += 1
    if own:
        return _RUN_OWN[case["kind"]](s, case, s["cvcuda"], s["kept"])
    return _RUN_PLAIN[case["kind"]](s, case)


def _own_embedding(s, case, cvcuda, kept):
    out = torch.empty((case["n"], case["d"]), dtype=TORCH[case["out"]], device="cuda")
    cvcuda.embedding_into(cvcuda.as_tensor(out), kept["table"], cvcuda.as_tensor(s["tokens"]), math.sqrt(case["d"]))
    return out


def _own_embedding_grad(s, case, cvcuda, kept):
    cvcuda.embedding_grad_into(kept["table"], cvcuda.as_tensor(s["grad"]), cvcuda.as_tensor(s["tokens"]), math.sqrt(case["d"]),
                               padding=0 if case["padding"] else None, accumulate=case["accumulate"])
    return s["table"]


def _own_layer_norm(s, case, cvcuda, kept):
    out, mean, rstd = torch.empty_like(s["x"]), None, None
    if case["stats"]:
        mean, rstd = torch.empty((case["rows"],), device="cuda"), torch.empty((case["rows"],), device="cuda")
        cvcuda.layer_norm_into(cvcuda.as_tensor(out), cvcuda.as_tensor(s["x"]), kept["gamma"], kept["beta"], EPSILON,
                               mean=cvcuda.as_tensor(mean), rstd=cvcuda.as_tensor(rstd))
        return [out, mean, rstd]
    cvcuda.layer_norm_into(cvcuda.as_tensor(out), cvcuda.as_tensor(s["x"]), kept["gamma"], kept["beta"], EPSILON)
    return [out]


def _own_layer_norm_grad(s, case, cvcuda, kept):
    to_x, to_gamma, to_beta = torch.empty_like(s["x"]), torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
    wrap = cvcuda.as_tensor
    cvcuda.layer_norm_grad_into(wrap(to_x), wrap(to_gamma), wrap(to_beta), wrap(s["grad"]), wrap(s["x"]), kept["gamma"],
                                wrap(s["mean"]), wrap(s["rstd"]))
    return [to_x, to_gamma, to_beta]


def _own_adamw(s, case, cvcuda, kept):
    cvcuda.adamw_into(kept["params"], kept["m"], kept["v"], kept["grads"], s["step"], ADAMW["lr"], ADAMW["betas"], ADAMW["epsilon"],
                      ADAMW["weight_decay"], copies=kept.get("copies"), moment_scales=kept.get("m_scale"),
                      variance_scales=kept.get("v_scale"), grad_scale=kept["grad_scale"])
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        cvcuda.adamw_unpack_into(kept["m_values"], kept["m"], kept["m_scale"])
        cvcuda.adamw_unpack_into(kept["v_values"], kept["v"], kept["v_scale"])
        m, v = s["m_values"], s["v_values"]
    return [s["params"], m, v] + ([] if s["copies"] is None else [s["copies"]])


_RUN_PLAIN = {"embedding": _plain_embedding, "embedding_grad": _plain_embedding_grad, "layer_norm": _plain_layer_norm,
              "layer_norm_grad": _plain_layer_norm_grad, "adamw": _plain_adamw}
_RUN_OWN = {"embedding": _own_embedding, "embedding_grad": _own_embedding_grad, "layer_norm": _own_layer_norm,
            "layer_norm_grad": _own_layer_norm_grad, "adamw": _own_adamw}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def _distinct(n, v):
    """Expected number of different words among n of _Source.tokens."""
    k = torch.arange(1, v + 1, dtype=torch.float64)
    share = torch.log1p(1 / k) / math.log(v + 1)
    return float((-torch.expm1(n * torch.log1p(-share.clamp(max=1 - 1e-12)))).sum())


def work(case):
    kind = case["kind"]
    if kind == "embedding":
        n, d = case["n"], case["d"]
        return {"bytes": n * SIZE[case["tokens"]] + _distinct(n, case["v"]) * d * SIZE[case["type"]] + n * d * SIZE[case["out"]],
                "flops": n * d}
    if kind == "embedding_grad":
        n, d, e = case["n"], case["d"], SIZE[case["grad"]]
        table = 2 * _distinct(n, case["v"]) * d * e if case["accumulate"] else case["v"] * d * e
        return {"bytes": n * SIZE[case["tokens"]] + n * d * SIZE[case["type"]] + table, "flops": 2 * n * d}
    if kind == "layer_norm":
        px = case["rows"] * case["d"]
        return {"bytes": 2 * px * SIZE[case["type"]] + 2 * case["d"] * SIZE[case["weights"]] + (8 * case["rows"] if case["stats"] else 0),
                "flops": 8 * px}
    if kind == "layer_norm_grad":
        px = case["rows"] * case["d"]
        return {"bytes": 3 * px * SIZE[case["type"]] + 3 * case["d"] * SIZE[case["weights"]] + 8 * case["rows"], "flops": 14 * px}
    count = sum(math.prod(shape) for shape in _shapes(case))
    each = 8 + SIZE[case["grad"]] + (SIZE[case["copy"]] if case["copy"] else 0)
    # states: 32 bits read and written; 8 bits read and written with a scale for 256, and their values written out
    each += 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": count * each, "flops": count * 16}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "embedding":
        return torch.index_select(s["table"], 0, s["tokens"].long()).double() * case["d"] ** 0.5
    if kind == "embedding_grad":
        tokens, table = s["tokens"].long(), s["table"].double() if case["accumulate"] else torch.zeros_like(s["table"], dtype=torch.float64)
        keep = torch.nonzero(tokens != 0)[:, 0] if case["padding"] else torch.arange(case["n"], device="cuda")
        return table.index_put_((tokens[keep],), s["grad"][keep].double() * case["d"] ** 0.5, accumulate=True)
    if kind == "layer_norm":
        out = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        mean, rstd = torch.empty(case["rows"], dtype=torch.float64, device="cuda"), torch.empty(case["rows"], dtype=torch.float64, device="cuda")
        for at in range(0, case["rows"], 8192):
            x = s["x"][at:at + 8192].double()
            var, mean[at:at + 8192] = torch.var_mean(x, 1, correction=0)
            rstd[at:at + 8192] = (var + EPSILON) ** -0.5
            out[at:at + 8192] = torch.addcmul(s["beta"].double(), (x - mean[at:at + 8192, None]) * rstd[at:at + 8192, None], s["gamma"].double())
        return [out, mean, rstd] if case["stats"] else [out]
    if kind == "layer_norm_grad":
        to_x = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        to_gamma, to_beta = torch.zeros(case["d"], dtype=torch.float64, device="cuda"), torch.zeros(case["d"], dtype=torch.float64, device="cuda")
        for at in range(0, case["rows"], 8192):
            rstd = s["rstd"][at:at + 8192, None].double()
            h = (s["x"][at:at + 8192].double() - s["mean"][at:at + 8192, None].double()) * rstd
            g = s["grad"][at:at + 8192].double()
            w = g * s["gamma"].double()
            to_x[at:at + 8192] = (w - (w.sum(1, keepdim=True) + h * (w * h).sum(1, keepdim=True)) / case["d"]) * rstd
            to_gamma += (g * h).sum(0)
            to_beta += g.sum(0)
        return [to_x, to_gamma, to_beta]
    return _exact_adamw(s, case)


def _exact_adamw(s, case):
    (b1, b2), lr, t, short = ADAMW["betas"], ADAMW["lr"], s["step"] + 1, case["bits"] == 8
    g = s["grads"].double() * s["grad_scale"].double()
    if short:
        a, b = (s[k].double().repeat_interleave(BLOCK) for k in ("m_scale", "v_scale"))
        m = torch.sign(s["m"].double()) * (s["m"].double() / 127) ** 2 * a
        v = (s["v"].double() / 255) ** 4 * b
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = s["params"].double()
    p = p - lr * ADAMW["weight_decay"] * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + ADAMW["epsilon"])
    copies = [] if s["copies"] is None else [p]
    # (8-bit states have no 64-bit value: their codes are roundings of what 32 bits gave)
    return [p, None, None] + copies if short else [p, m, v] + copies
