"""The row operators' definitions in 64 bits, and how far a result in fewer bits may be from them.

U[type] is the unit roundoff. A result is one rounding to its type of a value computed in 32 bits: besides that rounding
(half a step, also below the smallest normal number) each test allows the 32-bit errors that its formula can collect: n * 2^-24
of the magnitudes that are added for a sum of n terms in any order, 2^-24 of the result for each further operation."""
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest step
U32 = 2.0 ** -24


def layer_norm(x, gamma, beta, eps):
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean) ** 2).mean(-1, keepdim=True).add(eps) ** -0.5
    return (x - mean) * rstd * gamma + beta, mean[..., 0], rstd[..., 0]


def layer_norm_grad(dy, x, gamma, mean, rstd):
    h = (x - mean[..., None]) * rstd[..., None]
    w = dy * gamma
    dx = rstd[..., None] * (w - w.mean(-1, keepdim=True) - h * (w * h).mean(-1, keepdim=True))
    over = tuple(range(x.ndim - 1))
    return dx, (dy * h).sum(over), dy.sum(over)


def close(got, want, error, what=""):
    """got (of a type in U) is within one rounding of something within `error` of want (64 bits)."""
    bound = (want.abs() + error) * U[got.dtype] + error + STEP[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d, the worst %.3g times the bound (%.9g, %.9g)" % (
        what, int(bad.sum()), bad.numel(), float((off / bound)[bad].max()), float(got[bad].double().flatten()[0]), float(want[bad].flatten()[0]))


def layer_norm_errors(x, gamma, beta, mean, rstd, eps):
    """32-bit errors of (out, mean, rstd). Sums in runs per lane and then over the lanes: at most D / 64 + 16 roundings on the way
    of a term, so the mean is off by that of the mean magnitude. The squares' sum likewise, with the mean's own error in each
    (its first power cancels in the sum); rstd by half of its relative error and 4 operations' own."""
    n = x.shape[-1] / 64 + 16
    e_mean = n * U32 * x.abs().mean(-1)
    far = (x - mean[..., None]).abs()
    var = (far ** 2).mean(-1)
    e_var = (n + 4) * U32 * var + 2 * far.mean(-1) * U32 * x.abs().amax(-1) + e_mean ** 2
    e_rstd = rstd * (0.5 * e_var / (var + eps) + 4 * U32)
    e_far = e_mean[..., None] + U32 * far
    e_out = gamma.abs() * (e_far * rstd[..., None] + far * e_rstd[..., None]) + 4 * U32 * (gamma.abs() * far * rstd[..., None] + beta.abs())
    return e_out, e_mean, e_rstd


def layer_norm_grad_errors(dy, x, gamma, mean, rstd):
    """32-bit errors of (dx, dgamma, dbeta). h: 2 operations, and the difference's rounding of x - mean. The sums over a row as
    above; those over rows in any order."""
    d, rows = x.shape[-1], x.numel() // x.shape[-1]
    n = d / 64 + 20
    h = (x - mean[..., None]) * rstd[..., None]
    e_h = 3 * U32 * h.abs()
    w = (dy * gamma).abs()
    s, sh = w.mean(-1, keepdim=True), (w * h.abs()).mean(-1, keepdim=True)
    e_sh = n * U32 * sh + (w * e_h).mean(-1, keepdim=True)
    e_dx = rstd[..., None].abs() * (8 * U32 * (w + s + h.abs() * sh) + n * U32 * s + h.abs() * e_sh + e_h * sh)
    over = tuple(range(x.ndim - 1))
    return (e_dx, ((rows + 4) * U32 * dy.abs() * h.abs() + dy.abs() * e_h).sum(over) if rows else None,
            ((rows + 4) * U32 * dy.abs()).sum(over))
