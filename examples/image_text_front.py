"""Trains the front of an image-text model, from decoded images to updated weights, with the operators of this framework.

    python examples/image_text_front.py [--steps 20] [--batch 32] [--states 8]

A step:
  1. resize_crop_convert_reformat: 8-bit NHWC images -> normalized NCHW crops of 224 x 224
  2. layer_norm of the 16 x 16 x 3 = 768 values of each patch, a product with weights, layer_norm
  3. embedding of the captions' tokens (ragged: padding has no part in anything), layer_norm
  4. the products, means and the contrastive loss of torch
  5. their gradients: layer_norm_grad, embedding_grad (a table's gradient that is the same on every run)
  6. adamw over all weights in one call: F32 weights, their BF16 copies for the next step, states in 32 or in 8 bits

Images and captions are random, so that the loss falls as the weights learn the batch by heart.
"""
import argparse
import importlib
import importlib.util
import os
import sys
import time

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

PATCH, CROP, PADDING = 16, 224, 0


def load():
    """This framework's Python interface, from the tree that this file is in."""
    if "cvcuda_amd" not in sys.modules:
        where = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cv-cuda_amd")
        spec = importlib.util.spec_from_file_location("cvcuda_amd", os.path.join(where, "__init__.py"), submodule_search_locations=[where])
        sys.modules["cvcuda_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["cvcuda_amd"])
    return importlib.import_module("cvcuda_amd.pyapi")


cvcuda = load()
wrap = cvcuda.as_tensor


class LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta):
        y, mean, rstd = torch.empty_like(x), *(torch.empty(x.shape[:-1], device=x.device) for _ in range(2))
        cvcuda.layer_norm_into(wrap(y), wrap(x), wrap(gamma), wrap(beta), mean=wrap(mean), rstd=wrap(rstd))
        ctx.save_for_backward(x, gamma, mean, rstd)
        return y

    @staticmethod
    @once_differentiable  # (the gradients have none of their own)
    def backward(ctx, grad):
        x, gamma, mean, rstd = ctx.saved_tensors
        grad = grad.contiguous()
        made = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
        cvcuda.layer_norm_grad_into(*map(wrap, made), *map(wrap, (grad, x, gamma, mean, rstd)))
        return made


class Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale):
        rows = torch.empty(*tokens.shape, table.shape[1], dtype=table.dtype, device=table.device)
        cvcuda.embedding_into(wrap(rows), wrap(table), wrap(tokens), scale)
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale = table.shape[0], scale
        return rows

    @staticmethod
    @once_differentiable  # (the gradients have none of their own)
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        grad = grad.contiguous()
        made = torch.empty(ctx.rows, grad.shape[-1], dtype=grad.dtype, device=grad.device)
        cvcuda.embedding_grad_into(wrap(made), wrap(grad), wrap(tokens), ctx.scale, padding=PADDING)
        return made, None, None


class AdamW:
    """F32 weights with copies that the model computes with, and states in 32 bits or in 8 (0: what zeros stand for in both)."""

    def __init__(self, weights, copies, bits):
        def states(kinds):
            return [[torch.zeros(w.shape, dtype=kind, device=w.device) for w in weights] for kind in kinds]

        self.weights, self.copies, self.steps = weights, copies, 0
        self.moments, self.variances = states([torch.float32] * 2 if bits == 32 else [torch.int8, torch.uint8])
        self.scales = {}
        if bits == 8:
            self.scales = {name: [torch.zeros((w.numel() + 255) // 256, device=w.device) for w in weights]
                           for name in ("moment_scales", "variance_scales")}

    def step(self, **how):
        self.steps += 1
        lists = [[wrap(t) for t in part] for part in (self.weights, self.moments, self.variances, [c.grad for c in self.copies])]
        cvcuda.adamw_into(*lists, self.steps, copies=[wrap(c.detach()) for c in self.copies],
                          **{name: [wrap(t) for t in part] for name, part in self.scales.items()}, **how)
        for c in self.copies:
            c.grad = None


class Front:
    """The weights: F32 in `weights`, BF16 for the products and lookups in `copies`."""

    def __init__(self, vocabulary, width, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        values = PATCH * PATCH * 3

        def random(*shape, scale):
            return torch.randn(shape, generator=g, device="cuda") * scale

        def norm(width):
            return {"gamma": torch.ones(width, device="cuda"), "beta": torch.zeros(width, device="cuda")}

        made = {"patches": norm(values), "product": {"weight": random(width, values, scale=values ** -0.5)}, "vectors": norm(width),
                "table": {"rows": random(vocabulary, width, scale=width ** -0.5)}, "words": norm(width)}
        self.weights = [w for part in made.values() for w in part.values()]
        self.copies = [w.bfloat16().requires_grad_() for w in self.weights]
        given = iter(self.copies)
        self.parts = {name: {key: next(given) for key in part} for name, part in made.items()}

    def crops(self, images):
        """Images [N, H, W, 3] of 8 bits -> [N, 3, 224, 224] from -1 to 1: the shorter side 256, the middle of that."""
        height, width = images.shape[1:3]
        short = 256 / min(height, width)
        size = max(256, round(width * short)), max(256, round(height * short))
        made = cvcuda.resize_crop_convert_reformat(wrap(images, "NHWC"), size, cvcuda.Interp.LINEAR,
                                                   cvcuda.RectI((size[0] - CROP) // 2, (size[1] - CROP) // 2, CROP, CROP),
                                                   layout="NCHW", data_type=cvcuda.Type.F32, scale=1 / 127.5, offset=-1.0)
        return made.torch()

    def images(self, images, norm=LayerNorm.apply):
        crops = self.crops(images)
        n, side = len(images), CROP // PATCH
        patches = crops.view(n, 3, side, PATCH, side, PATCH).permute(0, 2, 4, 3, 5, 1).reshape(n, side * side, -1).bfloat16()
        normed = norm(patches, *self.parts["patches"].values())
        vectors = F.linear(normed.view(-1, normed.shape[-1]), self.parts["product"]["weight"]).view(n, side * side, -1)
        return norm(vectors, *self.parts["vectors"].values()).float().mean(1)

    def captions(self, tokens, norm=LayerNorm.apply, lookup=Embedding.apply):
        table = self.parts["table"]["rows"]
        words = norm(lookup(table, tokens, table.shape[1] ** 0.5), *self.parts["words"].values())
        there = (tokens != PADDING).unsqueeze(-1)
        return (words.float() * there).sum(1) / there.sum(1).clamp(min=1)

    def loss(self, images, tokens, **how):
        a = F.normalize(self.images(images, **{k: v for k, v in how.items() if k == "norm"}), dim=-1)
        b = F.normalize(self.captions(tokens, **how), dim=-1)
        scores, right = a @ b.t() / 0.07, torch.arange(len(a), device=a.device)
        return (F.cross_entropy(scores, right) + F.cross_entropy(scores.t(), right)) / 2


def batch_of(n, vocabulary, longest, seed=1):
    """(random images, captions of 1 to `longest` tokens; the rest is padding)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    images = torch.randint(0, 256, (n, 12, 16, 3), generator=g, device="cuda", dtype=torch.uint8)
    images = images.repeat_interleave(40, 1).repeat_interleave(40, 2)
    tokens = torch.randint(1, vocabulary, (n, longest), generator=g, device="cuda")
    lengths = torch.randint(1, longest + 1, (n, 1), generator=g, device="cuda")
    return images, tokens.masked_fill_(torch.arange(longest, device="cuda") >= lengths, PADDING)


def train(steps=20, batch=32, vocabulary=32000, width=768, longest=77, bits=32, lr=1e-3):
    """The loss before each step."""
    front = Front(vocabulary, width)
    optimizer = AdamW(front.weights, front.copies, bits)
    images, tokens = batch_of(batch, vocabulary, longest)
    losses = []
    for _ in range(steps):
        loss = front.loss(images, tokens)
        loss.backward()
        optimizer.step(lr=lr, weight_decay=0.01)
        losses.append(loss.detach())
    return [float(x) for x in losses]


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--batch", type=int, default=32)
    parser.add_argument("--states", type=int, choices=(8, 32), default=32, help="bits of the optimizer's states")
    args = parser.parse_args()
    train(1, args.batch, bits=args.states)  # (the libraries are loaded on the way)
    start = time.perf_counter()
    losses = train(args.steps, args.batch, bits=args.states)
    seconds = time.perf_counter() - start
    for i, loss in enumerate(losses):
        print("step %3d  loss %.4f" % (i + 1, loss))
    print("%.0f images/s" % (args.steps * args.batch / seconds))


if __name__ == "__main__":
    main()
