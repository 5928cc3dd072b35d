"""64-bit definitions of the projection and softmax-loss operators, with a
bound on each result's error.

The bounds follow from how the results are made. A sum over K of products of
operands with magnitudes |a||b| (sum A) is added by the tensor cores in pieces
of 128 or 1024 with truncation, each addition off by at most 2^-23 of A, then
piece by piece: SUM(K) = (min(K, 1024) + K / 128 + 8) 2^-23 bounds the relative
error against A. A result of unit roundoff u adds u of itself; an operand that
is rounded on the way (dz, g) adds u of the sum of its magnitudes. fp32
operands are three bf16 parts, 2^-26 from whole, far below SUM. Exponentials
and the activations are good to 2^-20.
"""
from __future__ import annotations

import math

import torch

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}  # subnormal spacing
FUNC = 2.0 ** -20


def sum_error(k: int) -> float:
    return (min(k, 1024) + k / 128 + 8) * 2.0 ** -23


def act64(z, name):
    """(act(z), act'(z)) in float64."""
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def linear64(x, w, bias, residual, act, out_dtype):
    """((y, bound), (pre, bound))."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs()
    y = act64(z, act)[0]
    err = mag * sum_error(x.shape[1])
    pre_bound = err + ROUND[x.dtype] * z.abs() + TINY[x.dtype]
    err = 1.2 * err + FUNC * z.abs()  # |act'| < 1.13
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return (y, err + ROUND[out_dtype] * y.abs() + TINY[out_dtype]), (z, pre_bound)


def linear_backward64(dy, x, w, pre, act):
    """dx, dw, db, each (value, bound)."""
    u, tiny = ROUND[x.dtype], TINY[x.dtype]
    dz = dy.double()
    if act != "none":
        dz = dz * act64(pre.double(), act)[1]
    # The slope's own terms are up to 1.2 and may cancel; dz is then rounded to the operands' type.
    off = dy.double().abs() * 4 * FUNC + u * dz.abs() + tiny
    xd, wd = x.double(), w.double()
    m, n = dy.shape
    dx, dw, db = dz @ wd, dz.t() @ xd, dz.sum(0)
    return (
        (dx, off @ wd.abs() + sum_error(n) * (dz.abs() @ wd.abs()) + u * dx.abs() + tiny),
        (dw, off.t() @ xd.abs() + sum_error(m) * (dz.abs().t() @ xd.abs()) + u * dw.abs() + tiny),
        (db, dy.double().abs().sum(0) * 4 * FUNC + sum_error(m) * dz.abs().sum(0) + u * db.abs() + tiny),
    )


def xent64(x, w, labels, scale):
    """((loss, bound), (lse, bound), z, bound of z)."""
    xd, wd = x.double(), w.double()
    z = scale * (xd @ wd.t())
    ez = scale * (xd.abs() @ wd.abs().t()) * sum_error(x.shape[1]) + z.abs() * 2.0 ** -22
    lse = torch.logsumexp(z, 1)
    n = w.shape[0]
    kept = (labels >= 0) & (labels < n)
    at = torch.where(kept, labels, torch.zeros_like(labels)).long()[:, None]
    elem = ez.max(1).values + FUNC + 2.0 ** -21 * lse.abs()
    loss = torch.where(kept, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    return (loss, torch.where(kept, elem + ez.gather(1, at)[:, 0] + 2.0 ** -22 * loss.abs(), torch.zeros_like(loss))), \
        (lse, elem), z, ez


def xent_backward64(dloss, x, w, labels, lse, scale):
    """dx, dw, each (value, bound)."""
    u, tiny = ROUND[x.dtype], TINY[x.dtype]
    _, _, z, ez = xent64(x, w, labels, scale)
    m, n = z.shape
    kept = (labels >= 0) & (labels < n)
    p = torch.exp(z - lse.double()[:, None])
    hot = torch.zeros_like(p)
    hot[kept, labels[kept].long()] = 1.0
    coef = (dloss.double() * scale * kept)[:, None]
    g = coef * (p - hot)
    # p from the scores' error, then g rounded (fp16: relative to max |coef|, spacing 2^-24 at 2^14).
    off = coef.abs() * p * (ez + FUNC + 2.0 ** -22 * lse.double().abs()[:, None]) + (u + 2.0 ** -22) * g.abs()
    if x.dtype == torch.float16:
        off = off + coef.abs().max() * 2.0 ** -38
    xd = torch.where(kept[:, None], x.double(), torch.zeros_like(x.double()))
    wd = w.double()
    dx, dw = g @ wd, g.t() @ xd
    return (
        (dx, off @ wd.abs() + sum_error(n) * (g.abs() @ wd.abs()) + u * dx.abs() + tiny),
        (dw, off.t() @ xd.abs() + sum_error(m) * (g.abs().t() @ xd.abs()) + u * dw.abs() + tiny),
    )
