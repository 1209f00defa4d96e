"""Attention from its definition in 64 bits, and how far a kernel with 16-bit weights and results may be from it."""
import torch


def attend(q, k, v, first, length, window=0, sinks=0, scale=None):
    """Rows of ``q[n, d]`` at positions first, first + 1, ... over the first ``length`` of ``k``, ``v`` ``[m, d]``: the
    result and, beside it, the bound of its error for a kernel that rounds each weight and the result to q's type.
    What is not finite in k and v counts as zero: rows that see such a token are not this function's to judge."""
    n, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    length = max(0, min(length, k.shape[0]))
    i = (first + torch.arange(n, device=q.device))[:, None]
    j = torch.arange(length, device=q.device)[None]
    see = (j <= i) & (i < length)
    if window:
        see &= (j > i - window) | (j < sinks)
    qd, kd, vd = (torch.nan_to_num(x.double(), 0.0, 0.0, 0.0) for x in (q, k[:length], v[:length]))
    m = see.sum(1, keepdim=True)
    s = (qd @ kd.t() * scale).masked_fill(~see, float("-inf"))
    w = torch.nan_to_num(torch.softmax(s, 1), 0.0)      # rows that see nothing
    out, spread = w @ vd, w @ vd.abs()
    # A score is a sum of d products in fp32, each addition off by at most 2^-23 of what has been added up, then two roundings
    # and an exponential of 2^-22: `delta` bounds the relative error of a weight.
    size = ((qd.abs() @ kd.abs().t()) * abs(scale)).masked_fill(~see, 0.0)
    delta = (size.amax(1, keepdim=True) if length else torch.zeros_like(m, dtype=torch.float64)) * (d + 4) * 2.0 ** -23 + 2.0 ** -21
    # rounding of the result; rounding of the weights (half a step each); the error of the weights and of their sum (twice
    # delta); sums of m terms in fp32; fp16 weights below 2^-14 keep an absolute error of 2^-25
    tol = (eps / 2 * out.abs() + (eps / 2 + 2 * delta + m * 2.0 ** -23) * spread) * 1.01
    if q.dtype == torch.float16 and length:
        tol += m * 2.0 ** -25 * vd.abs().amax(0) + 2.0 ** -25
    return out, tol


def check(got, want, tol, what=""):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    worst = (err - tol).max().item()
    assert worst <= 0, f"{what}: off by {err.max().item():.3e}, {worst:.3e} more than allowed"
