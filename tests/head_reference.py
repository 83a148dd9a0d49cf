"""Rotary positions, attention and log probabilities: their definitions in 64 bits, and how far a result in fewer bits may be
from them (row_reference.close adds the rounding of the result itself).

U32 is the unit roundoff of 32 bits; a sum of n terms in any order is off by at most n * U32 of the magnitudes that are added. The
hardware's exponential and logarithm to the base 2 are off by at most 2 * U32 of their result (the logarithm also by 2 * U32)."""
import math

import torch

from row_reference import U, U32


# ---- rotary positions ------------------------------------------------------------------------------------------------------
def frequencies(dims, base=10000.0, factor=1.0, original=0.0, low=0.0, high=0.0):
    made = []
    for i in range(dims // 2):
        f = base ** (-2.0 * i / dims)
        if original > 0:
            g = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low)))
            f *= g + (1 - g) / factor
        else:
            f /= factor
        made.append(f)
    return made


def rotary(x, positions, dims, interleaved=False, inverse=False, magnitude=1.0, **how):
    """(result, how far off 32 bits may be). x: [T, H, D] in 64 bits. An angle's cosine and sine are off by 2^-24 for what the
    reduction to an eighth of a turn leaves, by the polynomials' 7 roundings and last terms (2^-27), and, for far positions, by position
    times the error of a frequency, 2^-50 of it, and of its fraction, 2^-63 turns; products and sum: 4 roundings."""
    f = torch.tensor(frequencies(dims, **how), dtype=torch.float64, device=x.device)
    angle = positions.double()[:, None, None] * f
    c, s = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude * (-1 if inverse else 1)
    out, error = x.clone(), torch.zeros_like(x)
    half = dims // 2
    at = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, half), slice(half, dims))
    a, b = x[..., at[0]], x[..., at[1]]
    out[..., at[0]], out[..., at[1]] = a * c - b * s, a * s + b * c
    off = magnitude * (8 * U32 + positions.double().abs()[:, None, None] * (f * 2.0 ** -50 + 2.0 ** -60)) * (a.abs() + b.abs())
    off = off + 3 * U32 * magnitude * (a.abs() + b.abs())
    error[..., at[0]], error[..., at[1]] = off, off
    return out, error


# ---- attention ---------------------------------------------------------------------------------------------------------------
def sees(rows, keys, causal, device):
    every = torch.ones((rows, keys), dtype=torch.bool, device=device)
    return every.tril(keys - rows) if causal else every


def _scores(q, k, scale):
    """Scores, and how far off 32 bits may be: sums of D products, the scale, the sum's exponent and what it is taken relative to."""
    s = scale * (q @ k.t().contiguous())
    return s, U32 * ((q.shape[1] + 4) * scale * (q.abs() @ k.abs().t().contiguous()) + 4 * s.abs())


def attention(q, k, v, scale, causal, kind):
    """(out, lse, error of out, error of lse) of one head of one sequence, in 64 bits; kind: the type that shares are rounded to
    (F16: of a 64th of the largest, so that small ones are off by 2^-25 / 64 of it)."""
    s, e_s = _scores(q, k, scale)
    seen = sees(len(q), len(k), causal, q.device)
    s = torch.where(seen, s, -math.inf)
    none = ~seen.any(1) if len(k) else torch.ones(len(q), dtype=torch.bool, device=q.device)
    if len(k) == 0:
        zero = torch.zeros_like(q)
        return zero, torch.full((len(q),), -math.inf, dtype=torch.float64, device=q.device), zero, zero[:, 0]
    lse = torch.logsumexp(s, 1)
    p = torch.where(none[:, None], 0.0, torch.exp(s - torch.where(none, 0.0, lse)[:, None]))
    out, size, n = p @ v, p @ v.abs(), len(k)
    # the largest score is in the sum and as far off as the others: relative to it each exponential is off by 2 * e_s and 4 roundings, and
    # as many for each time that the largest changed (once for each 32 keys at most)
    e_rel = 2 * torch.where(seen, e_s, 0.0).amax(1) + (8 + n / 8) * U32 + 2 * U32 * torch.where(none, 0.0, lse).abs()
    most = p.amax(1)
    floor = 2.0 ** -31 * most if kind is torch.float16 else torch.zeros_like(most)
    e_sum = e_rel + n * U32
    e_out = (U[kind] + e_sum)[:, None] * size + floor[:, None] * (seen.double() @ v.abs()) + (e_sum + 4 * U32)[:, None] * out.abs()
    e_lse = torch.where(none, 0.0, e_sum + 4 * U32 * (lse.abs() + 1))
    return out, lse, e_out, e_lse


def attention_grad(grad, q, k, v, out, lse, scale, causal, kind, bound):
    """(gradients of q, k, v, and their errors) of one head of one sequence, in 64 bits. bound: the largest |gradOut| times the largest |v| of the
    call, which F16 takes t relative to: it is off by 2^-25 at a largest of 2^11 to 2^13 for that; shares by 2^-25 / 2^15."""
    s, e_s = _scores(q, k, scale)
    seen = sees(len(q), len(k), causal, q.device)
    some = lse > -math.inf
    p = torch.where(seen & some[:, None], torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
    # (an exponential below the smallest normal number of 32 bits is 0, and one rounded to BF16 likewise)
    e_p = p * (e_s + U32 * (8 + 4 * torch.where(some, lse, 0.0).abs()[:, None])) + 2.0 ** -125 * seen
    dp, size = grad @ v.t().contiguous(), grad.abs() @ v.abs().t().contiguous()
    delta, size2 = (grad * out).sum(1, keepdim=True), (grad * out).abs().sum(1, keepdim=True)
    t = p * (dp - delta)
    d = q.shape[1]
    e_t = p * U32 * ((d + 3) * (size + size2) + 4 * (dp - delta).abs()) + e_p * (dp - delta).abs()
    small = (2.0 ** -36 * bound, 2.0 ** -40) if kind is torch.float16 else (0.0, 0.0)
    e_t = e_t + U[kind] * (t.abs() + e_t) + (small[0] + 2.0 ** -125) * seen
    e_p = e_p + U[kind] * (p + e_p) + small[1] * seen
    n, m = len(k), len(q)
    to_q, to_k, to_v = scale * (t @ k), scale * (t.t().contiguous() @ q), p.t().contiguous() @ grad
    ta, pa = t.abs() + e_t, p + e_p
    e_q = scale * (e_t @ k.abs() + (n + 8) * U32 * (ta @ k.abs()))
    e_k = scale * (e_t.t().contiguous() @ q.abs() + (m + 8) * U32 * (ta.t().contiguous() @ q.abs()))
    e_v = e_p.t().contiguous() @ grad.abs() + (m + 8) * U32 * (pa.t().contiguous() @ grad.abs())
    return (to_q, to_k, to_v), (e_q, e_k, e_v)


# ---- log probabilities -----------------------------------------------------------------------------------------------------------
def log_probs(logits, tokens, scale):
    """(log probabilities, entropy, lse) and their errors, of logits in 64 bits. Each exponential is taken of a difference that is off by U32 of it
    and is itself rounded; sums go by lanes, runs and rescalings, of which a term meets at most V / 64 + 64."""
    z = scale * logits
    v = z.shape[1]
    lse = torch.logsumexp(z, 1)
    nothing = lse == -math.inf
    base = torch.where(nothing, 0.0, lse)
    # (relative to the largest: beside logits of 1e38 the sum's logarithm is less than a step of 64 bits)
    less = z - torch.where(nothing, 0.0, z.amax(1))[:, None]
    logp = less - torch.where(nothing, 0.0, torch.logsumexp(less, 1))[:, None]
    p = logp.exp()
    entropy = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
    there = (tokens >= 0) & (tokens < v)
    got = torch.where(nothing, -math.inf, logp.gather(1, tokens.long().clamp(0, v - 1)[:, None])[:, 0])
    got = torch.where(there, got, 0.0)
    n = v / 64 + 64
    far = torch.where(p > 0, (z - z.amax(1, keepdim=True)).abs(), 0.0)  # from the largest
    e_rel = ((4 * U32 * far + 4 * U32) * p).sum(1) + n * U32
    top = torch.where(nothing, 0.0, z.amax(1)).abs()
    e_lse = e_rel + 4 * U32 * (top + base.abs() + 1)
    e_logp = torch.where(there & ~nothing, e_rel + 4 * U32 * (got.abs() + 1), 0.0)
    e_entropy = 2 * e_rel * (1 + (p * far).sum(1)) + ((8 + n) * U32 * p * far).sum(1) + ((4 * U32 * far + 4 * U32) * p * far).sum(1) + 4 * U32
    return (got, entropy, lse), (e_logp, torch.where(nothing, 0.0, e_entropy), torch.where(nothing, 0.0, e_lse))


def log_probs_grad(logits, tokens, lse, grad, scale, entropy=None, grad_entropy=None):
    """(gradient, its error) in 64 bits."""
    z = scale * logits
    some = lse > -math.inf
    logp = z - torch.where(some, lse, 0.0)[:, None]
    p = torch.where(some[:, None], logp.exp(), 0.0)
    there = (tokens >= 0) & (tokens < z.shape[1]) & some
    g = torch.where(there, grad, 0.0)[:, None]
    hit = (torch.arange(z.shape[1], device=z.device) == tokens.long()[:, None]).double()
    made = g * (hit - p)
    size = g.abs() * (hit + p)
    far = torch.where(p > 0, z.abs(), 0.0)  # (-infinity has no share)
    e_p = p * U32 * (4 * far + 4 * torch.where(some, lse, 0.0).abs()[:, None] + 6)
    error = g.abs() * e_p
    if grad_entropy is not None:
        part = torch.where(p > 0, logp, 0.0) + entropy[:, None]
        h = grad_entropy[:, None]
        made = made - h * p * part
        size = size + h.abs() * p * part.abs()
        error = error + h.abs() * (e_p * part.abs() + p * U32 * (2 * far + 2 * torch.where(some, lse, 0.0).abs()[:, None] + 2 * entropy.abs()[:, None]))
    # (an exponential below the smallest normal number of 32 bits is 0)
    return scale * made, scale * (error + 6 * U32 * size + 2.0 ** -125 * (g.abs() + (0 if grad_entropy is None else 100 * grad_entropy.abs()[:, None])))
