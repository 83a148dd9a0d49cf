"""The references of rotary positions, attention and log probabilities (head_reference.py) by themselves, on the CPU: their gradients'
formulas in 64 bits against central differences of the definitions (steps of 1e-5: 1e-9 or less of third derivatives, 1e-10 of
roundings)."""
import math

import pytest
import torch

import head_reference as ref


def differences(f, tensors, grads):
    for t, grad in zip(tensors, grads):
        for i in range(t.numel()):
            ends = []
            for h in (1e-5, -1e-5):
                t.view(-1)[i] += h
                ends.append(float(f()))
                t.view(-1)[i] -= h
            assert abs((ends[0] - ends[1]) / 2e-5 - float(grad.reshape(-1)[i])) < 1e-7


def random(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys", [(4, 4), (3, 6), (5, 2)])
def test_attention_gradient_against_differences(rows, keys, causal):
    q, k, v, grad = random((rows, 8), 1), random((keys, 8), 2), random((keys, 8), 3), random((rows, 8), 4)

    def loss():
        return (ref.attention(q, k, v, 0.4, causal, torch.bfloat16)[0] * grad).sum()

    out, lse, _, _ = ref.attention(q, k, v, 0.4, causal, torch.bfloat16)
    differences(loss, (q, k, v), ref.attention_grad(grad, q, k, v, out, lse, 0.4, causal, torch.bfloat16, 1.0)[0])


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_gradient_against_differences(interleaved):
    x, grad, positions = random((3, 2, 10), 1), random((3, 2, 10), 2), torch.tensor([0, 7, 100000])
    how = dict(interleaved=interleaved, magnitude=1.3, factor=4.0, original=4096.0, low=1.0, high=4.0)
    differences(lambda: (ref.rotary(x, positions, 6, **how)[0] * grad).sum(), (x,), (ref.rotary(grad, positions, 6, inverse=True, **how)[0],))


def test_log_probs_gradient_against_differences():
    x, g, h = random((4, 9), 1), random((4,), 2), random((4,), 3)
    tokens = torch.tensor([0, 8, -1, 3])

    def loss():
        (logp, entropy, _), _ = ref.log_probs(x, tokens, 0.7)
        return (logp * g).sum() + (entropy * h).sum()

    (_, entropy, lse), _ = ref.log_probs(x, tokens, 0.7)
    differences(loss, (x,), (ref.log_probs_grad(x, tokens, lse, g, 0.7, entropy, h)[0],))


def test_scaled_frequencies():
    plain = ref.frequencies(64)
    assert plain[0] == 1 and all(a > b for a, b in zip(plain, plain[1:]))
    scaled = ref.frequencies(64, factor=8.0, original=8192.0, low=1.0, high=4.0)
    for f, s in zip(plain, scaled):
        turns = 8192 * f / (2 * math.pi)
        assert math.isclose(s, f if turns >= 4 else f / 8 if turns <= 1 else s, rel_tol=1e-12) and f / 8 <= s * (1 + 1e-12) and s <= f * (1 + 1e-12)
    assert all(math.isclose(a / 3, b, rel_tol=1e-12) for a, b in zip(plain, ref.frequencies(64, factor=3.0)))
