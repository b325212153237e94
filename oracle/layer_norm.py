"""Layer norm in 64 bits on the CPU: results, gradients, and how far kernels that compute in fp32 may be off.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

y = xhat w + b, xhat = (x - mean) r, r = (var + eps)^-1/2;  g = dy w, dx = r (g - mean(g) - xhat mean(g xhat)),
dw = sum dy xhat, db = sum dy.  Bounds, with v = 2^-24 and u half a step of the result's type (bf16 2^-8, fp32 v), each widened
by 1/16 for second-order terms: a lane adds up to 16 values one after the other and the lanes are joined in up to 20 steps, so a
row's sum is off by 36 v of the sum of the magnitudes, and its 1/n by 2 more; a column's sum over rows takes at most ROWS steps.
The mean is a first one, m0, and the mean of the differences from it, which is as exact as those are small; the forward takes both
from x one after the other, the backward their rounded sum.
"""
from __future__ import annotations

import torch

V = 2.0 ** -24
SUM = 36 * V
MEAN = SUM + 2 * V
ROWS = 256 * V
WIDEN = 1 + 1 / 16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def layer_norm(x, weight, bias, eps, dy=None, dtype=torch.bfloat16, param_dtype=None):
    """x [rows, n] (any floating type) -> dict of float64 y, mean, rstd and, with dy, dx, dweight, dbias, each with ``e_...``."""
    if param_dtype is None:  # the type that dweight and dbias are rounded to: the parameters' own
        param_dtype = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)
    x = x.double()
    n = x.shape[1]
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.double()
    u, up = half_step(dtype), half_step(param_dtype)
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    var = (xc * xc).mean(1, keepdim=True)
    r = (var + eps) ** -0.5
    xhat = xc * r
    y = xhat * w + b
    e_m0 = MEAN * x.abs().mean(1, keepdim=True)
    e_rest = (MEAN + V) * (xc.abs().mean(1, keepdim=True) + e_m0)
    e_mean = e_rest + V * mean.abs()
    e_xc = e_rest + V * (2 * xc.abs() + e_m0)
    rel_r = (MEAN + 2 * (xc.abs() * e_xc).mean(1, keepdim=True) / (var + eps)) / 2 + 4 * V
    e_xhat = r * e_xc + xhat.abs() * (rel_r + 2 * V)
    res = dict(y=y, mean=mean[:, 0], rstd=r[:, 0], e_mean=WIDEN * e_mean[:, 0], e_rstd=WIDEN * (rel_r * r)[:, 0],
               e_y=WIDEN * (w.abs() * e_xhat + 3 * V * ((w * xhat).abs() + b.abs()) + u * y.abs()))
    if dy is None:
        return res
    dy = dy.double()
    g = dy * w
    e_xhat = r * (e_mean + V * (xc.abs() + e_mean)) + xhat.abs() * (rel_r + 2 * V)  # by the rounded mean
    s1, s2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    e_s1 = SUM * g.abs().mean(1, keepdim=True)
    e_s2 = SUM * (g * xhat).abs().mean(1, keepdim=True) + (g.abs() * e_xhat).mean(1, keepdim=True)
    dx = r * (g - s1 - xhat * s2)
    inner = e_s1 + xhat.abs() * e_s2 + e_xhat * s2.abs() + 5 * V * (g.abs() + s1.abs() + (xhat * s2).abs())
    dw, db = (dy * xhat).sum(0), dy.sum(0)
    res |= dict(dx=dx, dweight=dw, dbias=db, e_dx=WIDEN * (r * inner + (rel_r + u) * dx.abs()),
                e_dweight=WIDEN * ((dy.abs() * e_xhat).sum(0) + ROWS * (dy * xhat).abs().sum(0) + up * dw.abs()),
                e_dbias=WIDEN * (ROWS * dy.abs().sum(0) + up * db.abs()))
    return res
