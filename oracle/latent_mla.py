"""Dense latent attention in 64 bits on the CPU: results, gradients, and how far bf16 kernels may be off.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

Row m of q [M, D] sees the keys [lo_m, hi_m): z = scale q k^T, p = softmax(z), out = p v,
lse2 = logsumexp(z) / ln 2; ds = p (dO v^T - out . dO) scale, dq = ds k, dk = ds^T q, dv = p^T dO.

Bounds, with u = 2^-8 (half a bf16 step, relative): a kernel rounds p and ds to bf16 for its
products and every result once more, and takes out . dO from the rounded out.  So
  |out err| <= u sum p |v| + u |out|              =: e_out
  |delta err| <= sum_c |dO_c| e_out_c             =: e_delta
  |ds err| <= u |ds| + p scale e_delta            =: e_ds
  |dq err| <= sum_j e_ds |k_j| + u |dq|, |dk err| <= sum_m e_ds |q_m| + u |dk|, |dv err| <= u sum_m p |dO_m| + u |dv|
each widened by 1/16 for the second-order terms and fp32's own roundings (a sum of n products of bf16 is off by
at most n 2^-24 of the sum of their magnitudes: below u / 16 for n < 4096, and exp2 of an exponent off by x is off
by a factor 1 + x).  fp32 sums of lse2: 2^-24 (|lse2| + the exponents' magnitudes, times D / 16 for their dots).
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -8
WIDEN = 1 + 1 / 16


def windows(B, S, S_kv, causal=True, starts=None, ends=None):
    """lo, hi [B, S] (int64), clipped; an empty row has lo = hi = 0."""
    if starts is not None:
        lo, hi = starts.long().clamp(min=0), ends.long().clamp(max=S_kv)
    else:
        t = torch.arange(S).expand(B, S)
        lo = torch.zeros(B, S, dtype=torch.int64)
        hi = (t + 1 + S_kv - S).clamp(0, S_kv) if causal else torch.full_like(lo, S_kv)
    empty = hi <= lo
    return lo.masked_fill(empty, 0), hi.masked_fill(empty, 0)


def attend(q, k, v, lo, hi, scale, do=None):
    """q [M, D], k [K, D], v [K, V], lo / hi [M] -> dict of float64 results, each with a bound ``e_...``.
    Keys outside a row's window do not reach it, whatever they hold."""
    q, k, v = q.double(), k.double(), v.double()
    j = torch.arange(k.shape[0])
    seen = (j >= lo[:, None]) & (j < hi[:, None])
    z = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(z, -1)
    empty = hi <= lo
    p = torch.exp(z - lse.masked_fill(empty, 0.0)[:, None]).masked_fill(~seen, 0.0)
    out = _product(p, v, seen)
    r = dict(out=out, lse=lse / math.log(2))
    r["e_out"] = WIDEN * (U * _product(p, v.abs(), seen) + U * out.abs())
    mag = (q.abs() @ k.abs().T * scale / math.log(2)).masked_fill(~seen, 0.0).amax(-1) if k.shape[0] else torch.zeros(len(q)).double()
    r["e_lse"] = 2.0 ** -23 * (4 + r["lse"].abs().masked_fill(empty, 0.0) + mag * q.shape[1] / 16)
    if do is None:
        return r
    do = do.double()
    delta = (out * do).sum(-1, keepdim=True)
    e_delta = (r["e_out"] * do.abs()).sum(-1, keepdim=True)
    ds = torch.where(seen, p * (do @ v.T - delta) * scale, 0.0)
    e_ds = torch.where(seen, U * ds.abs() + p * scale * e_delta, 0.0)
    r["dq"], e = _product(ds, k, seen), _product(e_ds, k.abs(), seen)
    r["e_dq"] = WIDEN * (e + U * r["dq"].abs())
    r["dk"], r["a_dk"] = _product(ds.T, q, seen.T), _product(e_ds.T, q.abs(), seen.T)
    r["dv"], r["a_dv"] = _product(p.T, do, seen.T), U * _product(p.T, do.abs(), seen.T)
    return r


def _product(x, y, seen):
    """x @ y over the admitted pairs alone: where y is not finite, a pair of weight 0 that is not admitted adds nothing."""
    if torch.isfinite(y).all():
        return x @ y
    out = torch.zeros(x.shape[0], y.shape[1], dtype=torch.float64)
    for m in range(x.shape[0]):
        out[m] = x[m, seen[m]] @ y[seen[m]]
    return out


def bound(value, accumulated):
    """The bound on a key gradient rounded once, from the summed error of its terms."""
    return WIDEN * (accumulated + U * value.abs())


def absorbed(q, kv, d_v, scale, lo, hi, do=None):
    """q [B, S, H, D], kv [B, K, G, D] -> dict(out, lse, dq, dkv and e_ of each) in float64."""
    B, S, H, D = q.shape
    K, G = kv.shape[1], kv.shape[2]
    hpg = H // G
    new = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    r = {n: new(B, S, H, *w) for n, w in (("out", (d_v,)), ("e_out", (d_v,)), ("lse", ()), ("e_lse", ()), ("dq", (D,)), ("e_dq", (D,)))}
    dkv, acc = new(B, K, G, D), new(B, K, G, D)
    for b in range(B):
        for h in range(H):
            g = h // hpg
            x = attend(q[b, :, h], kv[b, :, g], kv[b, :, g, :d_v], lo[b], hi[b], scale, None if do is None else do[b, :, h])
            for n in r:
                if n in x:
                    r[n][b, :, h] = x[n]
            if do is not None:
                dkv[b, :, g] += x["dk"]
                acc[b, :, g] += x["a_dk"]
                dkv[b, :, g, :d_v] += x["dv"]
                acc[b, :, g, :d_v] += x["a_dv"]
    if do is not None:
        r["dkv"], r["e_dkv"] = dkv, bound(dkv, acc)
    return r


def expanded(q, k_nope, k_pe, v, scale, lo, hi, do=None):
    """The expanded form: dict(out, lse, dq, dk_nope, dk_pe, dv and e_ of each) in float64."""
    B, S, H, D = q.shape
    K, dn, d_v = k_nope.shape[1], k_nope.shape[3], v.shape[3]
    new = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    r = {n: new(B, S, H, *w) for n, w in (("out", (d_v,)), ("e_out", (d_v,)), ("lse", ()), ("e_lse", ()), ("dq", (D,)), ("e_dq", (D,)))}
    dk, ak, dv, av = new(B, K, H, D), new(B, K, H, D), new(B, K, H, d_v), new(B, K, H, d_v)
    for b in range(B):
        for h in range(H):
            k = torch.cat([k_nope[b, :, h], k_pe[b]], dim=-1)
            x = attend(q[b, :, h], k, v[b, :, h], lo[b], hi[b], scale, None if do is None else do[b, :, h])
            for n in r:
                if n in x:
                    r[n][b, :, h] = x[n]
            if do is not None:
                dk[b, :, h], ak[b, :, h], dv[b, :, h], av[b, :, h] = x["dk"], x["a_dk"], x["dv"], x["a_dv"]
    if do is not None:
        pe, ape = dk[..., dn:].sum(2), ak[..., dn:].sum(2)
        r |= dict(dk_nope=dk[..., :dn], e_dk_nope=bound(dk[..., :dn], ak[..., :dn]), dk_pe=pe, e_dk_pe=bound(pe, ape), dv=dv,
                  e_dv=bound(dv, av))
    return r
