"""The paged latent cache on the CPU: MXFP4 rows, the plan of a serving step, attention over pages.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  Formats and rules as include/dsa_hip.h states them.
"""
from __future__ import annotations

import math

import torch

from .latent_mla import attend

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def row_bytes(d_qk, d_v):
    return -(-(d_v // 2 + 2 * (d_qk - d_v) + d_v // 32) // 16) * 16


def _nearest(a):
    """Code of the e2m1 value nearest to a >= 0 (ties: the even code), by distance."""
    best = min(range(8), key=lambda c: (abs(E2M1[c] - min(a, 6.0)), c & 1))
    return best


def pack_row(latent, rope):
    """bf16 [d_v], [d_rope] -> bytes of an MXFP4 row (list of ints; the padding is None: not written)."""
    x = latent.double().tolist()
    codes, exps = [], []
    for i in range(0, len(x), 32):
        blk = x[i:i + 32]
        if not all(math.isfinite(v) for v in blk):
            exps.append(255)
            codes += [8 if math.copysign(1.0, v) < 0 else 0 for v in blk]
            continue
        amax = max(abs(v) for v in blk)
        e = 0 if amax == 0 else max(-125, min(125, math.frexp(amax)[1] - 1 - 2))
        exps.append(e + 127)
        codes += [_nearest(abs(v) / 2.0 ** e) | (8 if math.copysign(1.0, v) < 0 else 0) for v in blk]
    out = [codes[i] | codes[i + 1] << 4 for i in range(0, len(codes), 2)]
    out += rope.contiguous().view(torch.uint8).tolist() + exps
    return out + [None] * (row_bytes(len(x) + rope.numel(), len(x)) - len(out))


def unpack_rows(rows, d_qk, d_v):
    """uint8 [N, row bytes] -> float64 [N, d_qk]."""
    at = d_v // 2 + 2 * (d_qk - d_v)
    half = rows[:, : d_v // 2].long()
    code = torch.stack([half & 15, half >> 4], -1).flatten(1)
    val = torch.tensor(E2M1, dtype=torch.float64)[code & 7] * torch.where(code > 7, -1.0, 1.0).double()
    e = rows[:, at: at + d_v // 32].double()
    scale = torch.where(e == 255, math.nan, torch.exp2(e - 127))
    lat = (val.unflatten(1, (-1, 32)) * scale[..., None]).flatten(1)
    return torch.cat([lat, rows[:, d_v // 2: at].contiguous().view(torch.bfloat16).double()], 1)


def plan(ctx, new, table, free, count, T, bs):
    """Lists of ints -> the plan's tensors as lists, request by request."""
    R, W, F = len(ctx), len(table[0]) if table else 0, len(free)
    have = max(0, min(count, F))
    out = [[-1] * W for _ in range(R)]
    slots, pos, starts, kv, nxt, granted, back = [-1] * T, [-1] * T, [], [], [], [], []
    at = upto = used = 0
    for r in range(R):
        c, n = max(0, min(ctx[r], W * bs)), max(new[r], 0)
        held = -(-c // bs)                       # its context's pages, and what lies behind them up to the first -1
        while held < W and table[r][held] >= 0:
            held += 1
        starts.append(min(at, T))
        if new[r] < 0:
            back += table[r][:held]
            kv.append(0), nxt.append(0), granted.append(0)
            continue
        ok = at + n <= T and c + n <= W * bs
        need = max(-(-(c + n) // bs) - held, 0) if ok else 0
        ok = ok and (need == 0 or upto + need <= have)
        out[r][:held] = table[r][:held]
        if ok:
            for j in range(need):
                out[r][held + j] = free[have - 1 - upto - j]
            used = max(used, upto + need) if need else used
            for i in range(n):
                b = out[r][(c + i) // bs]
                pos[at + i] = c + i
                slots[at + i] = b * bs + (c + i) % bs if b >= 0 else -1
        upto += need
        kv.append(c + n if ok else 0), nxt.append(c + n if ok else c), granted.append(int(ok))
        at += n
    starts.append(min(at, T))
    left = (free[: have - used] + back)[:F]
    return dict(block_table=out, slots=slots, positions=pos, query_starts=starts, kv_lens=kv, context_lens=nxt, granted=granted,
                free_blocks=left + [-1] * (F - len(left)), free_count=[len(left)])


def paged(q, rows, table, starts, kv_lens, bs, d_v, scale):
    """q [T, H, D]; rows float64 [slots, D] of the whole cache; -> out, lse, e_out, e_lse; rows of no request: NaN."""
    T, H, D = q.shape
    nan = lambda *s: torch.full(s, math.nan, dtype=torch.float64)  # noqa: E731
    r_ = dict(out=nan(T, H, d_v), e_out=nan(T, H, d_v), lse=nan(T, H), e_lse=nan(T, H))
    blocks, W = rows.shape[0] // bs, table.shape[1]
    for r in range(table.shape[0]):
        a, b = int(starts[r]), int(starts[r + 1])
        kv = max(0, min(int(kv_lens[r]), W * bs))
        key = torch.arange(kv)
        page = table[r].long()[key // bs]
        there = (page >= 0) & (page < blocks)
        k = rows[(page.clamp(0, blocks - 1) * bs + key % bs)[there]]
        where = key[there]
        for t in range(a, b):
            seen = int((where < kv - (b - a) + (t - a) + 1).sum())
            lo, hi = torch.zeros(H, dtype=torch.int64), torch.full((H,), seen)
            x = attend(q[t], k, k[:, :d_v], lo, hi, scale)
            for n in r_:
                r_[n][t] = x[n]
    return r_
