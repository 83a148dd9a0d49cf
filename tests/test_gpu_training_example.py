"""examples/image_text_front.py: its step is the one that torch's own operators and derivatives make, and it learns."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

WHERE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "image_text_front.py")


@pytest.fixture(scope="module")
def example(cv, gpu):
    spec = importlib.util.spec_from_file_location("image_text_front", WHERE)
    made = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(made)
    return made


@pytest.fixture(autouse=True)
def no_default_stream_is_followed(example, monkeypatch):
    monkeypatch.setattr(example.cvcuda, "_followed", {})


def plain_norm(x, gamma, beta):
    return F.layer_norm(x.float(), x.shape[-1:], gamma.float(), beta.float()).to(x.dtype)


def plain_lookup(table, tokens, scale):
    return (F.embedding(tokens, table.float()) * scale).to(table.dtype)


def test_gradients_are_those_of_the_formulas(example):
    """Against torch's operators in F32 at the same roundings to BF16: what remains is the order of sums and a last bit here and
    there, a share of 2^-8 of the values that are added up; 2^-5 of a gradient's norm is well above it and far below any
    term of a formula."""
    front = example.Front(500, 256)
    images, tokens = example.batch_of(6, 500, 20)
    loss = front.loss(images, tokens)
    loss.backward()
    loss = float(loss.detach())
    got = [c.grad.float() for c in front.copies]
    for c in front.copies:
        c.grad = None
    plain = front.loss(images, tokens, norm=plain_norm, lookup=plain_lookup)
    plain.backward()
    assert abs(loss - float(plain.detach())) <= 2 ** -6 * abs(loss)
    for g, c in zip(got, front.copies):
        want = c.grad.float()
        assert float((g - want).norm()) <= 2 ** -5 * float(want.norm())
    table = got[-3]
    unused = torch.ones(500, dtype=torch.bool, device="cuda")
    unused[tokens[tokens != example.PADDING]] = False
    assert (table[unused] == 0).all() and not table[~unused].any(1).logical_not().any()


@pytest.mark.parametrize("bits", [32, 8])
def test_it_learns(example, bits):
    losses = example.train(steps=12, batch=8, vocabulary=1000, width=128, longest=16, bits=bits)
    assert losses[-1] < losses[0] / 2


def test_the_copies_follow_the_weights(example):
    front = example.Front(300, 64)
    optimizer = example.AdamW(front.weights, front.copies, 8)
    images, tokens = example.batch_of(4, 300, 9)
    before = [w.clone() for w in front.weights]
    front.loss(images, tokens).backward()
    optimizer.step(lr=1e-2)
    for w, c, b in zip(front.weights, front.copies, before):
        assert torch.equal(c.detach(), w.bfloat16()) and not torch.equal(w, b) and c.grad is None


def test_second_derivatives_are_refused(example):
    """The gradients are differentiated no further: a derivative of theirs is refused, not taken without their part in it."""
    x, gamma, beta = (torch.randn(s, device="cuda", requires_grad=True) for s in ((5, 64), 64, 64))
    table, tokens = torch.randn(9, 64, device="cuda", requires_grad=True), torch.tensor([3, 1, 3], device="cuda")
    for out, of in ((example.LayerNorm.apply(x, gamma, beta), x), (example.Embedding.apply(table, tokens, 2.0), table)):
        grad, = torch.autograd.grad((out * out).sum(), of, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            (grad * grad).sum().backward()
