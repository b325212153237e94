"""The paged cache of index keys, the indexer's scores over it, and sparse attention over the latent cache, on the CPU.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  Formats and rules as include/dsa_hip.h states them.
"""
from __future__ import annotations

import math

import torch

from .latent_cache import E2M1, _nearest
from .latent_mla import WIDEN, attend

E4M3 = [(c & 7) * 2.0 ** -9 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)]


def _nearest_e4m3(a):
    """Code of the e4m3 value nearest to a >= 0 (ties: the even code), by distance; at most 448."""
    a = min(a, 448.0)
    return min(range(127), key=lambda c: (abs(E4M3[c] - a), c & 1))


def pack_key(k, fmt):
    """bf16 [d] -> (code bytes, exponent bytes) of an MX key as lists of ints."""
    x = k.double().tolist()
    codes, exps = [], []
    for i in range(0, len(x), 32):
        blk = x[i:i + 32]
        sign = [1 if math.copysign(1.0, v) < 0 else 0 for v in blk]
        if not all(math.isfinite(v) for v in blk):
            exps.append(255)
            codes += [s << (7 if fmt == "mxfp8" else 3) for s in sign]
            continue
        amax = max(abs(v) for v in blk)
        if fmt == "mxfp8":
            e = 0 if amax == 0 else next(e for e in range(-117, 120) if amax <= 448 * 2.0 ** e or e == 119)
            codes += [_nearest_e4m3(abs(v) / 2.0 ** e) | s << 7 for v, s in zip(blk, sign)]
        else:
            e = 0 if amax == 0 else max(-125, min(125, math.frexp(amax)[1] - 1 - 2))
            codes += [_nearest(abs(v) / 2.0 ** e) | s << 3 for v, s in zip(blk, sign)]
        exps.append(e + 127)
    if fmt == "mxfp4":
        codes = [codes[i] | codes[i + 1] << 4 for i in range(0, len(codes), 2)]
    return codes, exps + [0] * (4 - len(exps))


def unpack_pages(data, d):
    """A cache's data -> float64 [slots, d]."""
    if data.dtype == torch.bfloat16:
        return data.flatten(0, 1).double()
    blocks, bs, width = data.shape
    n = width - 4
    page = data.reshape(blocks, -1)
    raw, e = page[:, : bs * n].reshape(blocks * bs, n).long(), page[:, bs * n:].reshape(blocks * bs, 4)[:, : d // 32].double()
    if n == d:
        table = torch.tensor(E4M3 + [math.nan], dtype=torch.float64)
        val = table[raw & 127] * torch.where(raw > 127, -1.0, 1.0).double()
    else:
        code = torch.stack([raw & 15, raw >> 4], -1).flatten(1)
        val = torch.tensor(E2M1, dtype=torch.float64)[code & 7] * torch.where(code > 7, -1.0, 1.0).double()
    scale = torch.where(e == 255, math.nan, torch.exp2(e - 127))
    return (val.unflatten(1, (-1, 32)) * scale[..., None]).flatten(1)


def _request_rows(table, r, kv, bs, blocks):
    """Slots of positions 0 .. kv - 1 of request r (-1: on no page)."""
    key = torch.arange(kv)
    page = table[r].long()[key // bs]
    return torch.where((page >= 0) & (page < blocks), page * bs + key % bs, torch.full_like(page, -1))


def _tokens(table, starts, kv_lens, bs):
    """(token, request, keys that it sees)"""
    W = table.shape[1]
    for r in range(table.shape[0]):
        a, b = int(starts[r]), int(starts[r + 1])
        kv = max(0, min(int(kv_lens[r]), W * bs))
        for t in range(a, b):
            yield t, r, max(kv - (b - a) + (t - a) + 1, 0)


def scores(q, w, rows, table, starts, kv_lens, bs, L, use_relu=True):
    """-> scores [T, L], their bounds (NaN: a row of no request), limits [T].  A product of bf16 is exact in fp32 and a sum of D
    of them off by at most 2 D v of their magnitudes (v = 2^-24; the matrix unit may truncate), the sum over heads by H + 2."""
    T, H, D = q.shape
    v = 2.0 ** -24
    out, tol = torch.full((T, L), -math.inf, dtype=torch.float64), torch.full((T, L), math.nan, dtype=torch.float64)
    limits = torch.zeros(T, dtype=torch.int32)
    for t, r, n in _tokens(table, starts, kv_lens, bs):
        tol[t] = 0.0
        limits[t] = min(n, L)
        n = min(n, L)
        slot = _request_rows(table, r, n, bs, rows.shape[0] // bs)
        k = rows[slot.clamp(min=0)]
        x = q[t].double() @ k.T
        mag = q[t].double().abs() @ k.abs().T
        if use_relu:
            x = torch.where(x.isnan(), x, x.clamp(min=0))
        wt = w[t].double()
        s = wt @ x
        e = WIDEN * 2 * v * (D * (wt.abs() @ mag) + (H + 2) * (wt.abs() @ x.abs()))
        out[t, :n] = torch.where(slot >= 0, s, torch.full_like(s, -math.inf))
        tol[t, :n] = torch.where(slot >= 0, e.nan_to_num(0.0), torch.zeros_like(e))
    return out, tol, limits


def sparse(q, rows, indices, table, starts, kv_lens, bs, d_v, scale):
    """q [T, H, D]; rows float64 [slots, D] -> out, lse, e_out, e_lse; rows of no request: NaN."""
    T, H, _ = q.shape
    nan = lambda *s: torch.full(s, math.nan, dtype=torch.float64)  # noqa: E731
    res = dict(out=nan(T, H, d_v), e_out=nan(T, H, d_v), lse=nan(T, H), e_lse=nan(T, H))
    for t, r, n in _tokens(table, starts, kv_lens, bs):
        slot = _request_rows(table, r, n, bs, rows.shape[0] // bs)
        pos = indices[t].long()
        pos = pos[(pos >= 0) & (pos < n)]
        slot = slot[pos]
        k = rows[slot[slot >= 0]]
        m = k.shape[0]
        x = attend(q[t], k, k[:, :d_v], torch.zeros(H, dtype=torch.int64), torch.full((H,), m), scale)
        for name in res:
            res[name][t] = x[name]
    return res
