"""Dense latent attention and its paged cache: the timed workloads and their plain forms.

Each case is one call, or one training step, through the package's public entry points; ``kind`` names the operator:

  absorbed   LatentMLA step: every token's one latent row (V its first d_v channels) serves all heads; out, lse and the
             gradients of q and kv
  expanded   LatentMLAExpanded step: keys and values of every head, one shared rope part; out, lse and all gradients
  paged      paged_latent_mla_fwd: absorbed attention of new tokens over a paged cache (bf16, or MXFP4 latent + bf16 rope)
  cache      latent_cache_append of new tokens' rows, then latent_cache_gather of the same slots
  plan       plan_latent_step: block table, slot map, positions and lengths of a serving step, from request lengths

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, by the package's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

LOG2E = 1.4426950408889634
# (d_qk, d_v): 64 latent + 64 rope (NAM56R) and 512 latent + 64 rope (DeepSeek-V3.2); the un-absorbed 192/128 and 128/128
_LATENT = ((128, 64), (576, 512))


def _train(name, kind, B, S, S_kv, H, d_qk, d_v, mask):
    return dict(name=name, kind=kind, B=B, S=S, S_kv=S_kv, H=H, d_qk=d_qk, d_v=d_v, mask=mask)


def _paged(name, fmt, R, n_lo, n_hi, kv_lo, kv_hi, H, d_qk, d_v, block):
    return dict(name=name, kind="paged", fmt=fmt, R=R, n_lo=n_lo, n_hi=n_hi, kv_lo=kv_lo, kv_hi=kv_hi, H=H, d_qk=d_qk,
                d_v=d_v, block=block)


def _cache(name, fmt, T, d_qk, d_v, block, blocks):
    return dict(name=name, kind="cache", fmt=fmt, T=T, d_qk=d_qk, d_v=d_v, block=block, blocks=blocks)


def _plan(name, R, n_lo, n_hi, ctx, block):
    return dict(name=name, kind="plan", R=R, n_lo=n_lo, n_hi=n_hi, ctx=ctx, block=block)


def listed():
    return [
        # the smallest training call (cfg1's shape): a unit test, a debug run, the last short micro-batch
        _train("absorbed_small", "absorbed", 1, 512, 512, 16, 128, 64, "causal"),
        # the production layer in the dense warm-up before its indexer selects (cfg2, NAM56R)
        _train("absorbed_train", "absorbed", 2, 4096, 4096, 32, 128, 64, "causal"),
        # the long-context model's heads, un-absorbed, as dense layers are trained
        _train("expanded_train", "expanded", 1, 4096, 4096, 128, 192, 128, "causal"),
        # a packed batch of documents with padding behind the last one: no size fills a tile, some rows see nothing
        _train("expanded_ragged", "expanded", 3, 1531, 1531, 28, 192, 128, "docs"),
        # one new token of one short conversation on a small model: latency
        _paged("decode_one", "bf16", 1, 1, 1, 513, 513, 16, 128, 64, 64),
        # generation: 64 conversations of mixed length, every head on one card
        _paged("decode_bf16", "bf16", 64, 1, 1, 301, 16384, 128, 576, 512, 64),
        # generation with the heads split over eight cards, cache in 4 bits
        _paged("decode_mxfp4", "mxfp4", 96, 1, 1, 1023, 16384, 16, 576, 512, 64),
        # chunked prefill beside decoding: a few hundred new tokens on cached prompts, cache in 4 bits
        _paged("prefill_mxfp4", "mxfp4", 6, 40, 512, 1024, 4096, 32, 128, 64, 16),
        # a decode step's new rows
        _cache("cache_step", "bf16", 64, 576, 512, 64, 512),
        # a prefill batch's new rows, quantised
        _cache("cache_prefill", "mxfp4", 16384, 576, 512, 64, 512),
        # the plan of a small decode step
        _plan("plan_step", 16, 1, 1, 2048, 64),
        # the plan of a full server's mixed step: prompts and single tokens
        _plan("plan_mixed", 768, 0, 64, 16384, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(("absorbed", "absorbed", "expanded", "expanded", "paged", "paged", "paged", "paged", "cache", "plan"))
    if kind in ("absorbed", "expanded"):
        S_kv = _log(rng, 65, 4096)
        mask = rng.choice(("causal", "causal", "docs", "full"))
        S = S_kv if mask == "docs" or rng.random() < 0.7 else rng.randint(max(1, S_kv // 4), S_kv)
        d_qk, d_v = rng.choice(((128, 64), (128, 64), (192, 128), (128, 128)) if kind == "absorbed" else ((192, 128), (128, 64)))
        c = _train("", kind, rng.randint(1, 3), S, S_kv, rng.choice((8, 12, 16, 28, 32, 64, 128)), d_qk, d_v, mask)
    elif kind == "paged":
        one = rng.random() < 0.6
        R = _log(rng, 1, 96 if one else 12)
        kv_hi = _log(rng, 600, 16384 if one else 4096)
        n_hi = 1 if one else _log(rng, 2, 512)
        c = _paged("", rng.choice(("bf16", "mxfp4")), R, 1 if one else rng.randint(1, n_hi), n_hi,
                   max(n_hi, _log(rng, 500, kv_hi)), kv_hi, rng.choice((8, 16, 32, 64, 128)), *rng.choice(_LATENT),
                   rng.choice((16, 64, 64, 128)))
    elif kind == "cache":
        T, block = _log(rng, 1, 16384), rng.choice((16, 64, 128))
        c = _cache("", rng.choice(("bf16", "mxfp4")), T, *rng.choice(_LATENT), block, T // block + rng.randint(2, 256))
    else:
        c = _plan("", _log(rng, 1, 768), rng.randint(0, 1), _log(rng, 1, 64), _log(rng, 64, 16384), rng.choice((16, 64)))
    del c["name"]
    return c


def draw(rng):
    most = [work(c) for c in listed()]
    flops, size = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        c = _draw_once(rng)
        w = work(c)
        if w["flops"] <= flops and w["bytes"] <= size and _plain_bytes(c) <= 40e9:
            return c


def _plain_bytes(c):
    """Scores of the plain form: a bound on what it holds."""
    if c["kind"] in ("absorbed", "expanded"):
        return 4 * c["B"] * c["H"] * c["S"] * c["S_kv"]
    if c["kind"] == "paged":
        return 4 * c["R"] * c["kv_hi"] * (c["n_hi"] * c["H"] + c["d_qk"])
    return 0


# ---------------------------------------------------------------- inputs


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread (one of them: hi)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _doc_lengths(S):
    """Packed documents of a row of S tokens and the padding behind them."""
    pad = S // 11
    left, parts = S - pad, (5, 1, 9, 3, 2)
    lens = [left * p // sum(parts) for p in parts]
    lens[0] += left - sum(lens)
    return lens, pad


def _requests(c):
    """(kv length, new tokens) of a paged case's requests: the same numbers for every seed."""
    return list(zip(_spread(c["kv_lo"], c["kv_hi"], c["R"]), reversed(_spread(c["n_lo"], c["n_hi"], c["R"]))))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _row_bytes(d_qk, d_v):
    """An MXFP4 cache row: d_v / 2 bytes of codes (element 2 i in the low half of byte i), the rope part in bf16, one
    exponent byte per 32 latent channels, padded to 16 bytes."""
    return (d_v // 2 + 2 * (d_qk - d_v) + d_v // 32 + 15) // 16 * 16


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    c, kind = case, case["kind"]
    s = dict(case=c)
    if kind in ("absorbed", "expanded"):
        B, S, S_kv, H, D, V = c["B"], c["S"], c["S_kv"], c["H"], c["d_qk"], c["d_v"]
        s["q"], s["do"] = _normal(g, B, S, H, D), _normal(g, B, S, H, V)
        if kind == "absorbed":
            s["kv"] = _normal(g, B, S_kv, 1, D)
        else:
            # one up-projection gives both: k_nope and v are views of its rows
            up = _normal(g, B, S_kv, H, D - 64 + V)
            s["k_nope"], s["v"], s["k_pe"] = up[..., : D - 64], up[..., D - 64:], _normal(g, B, S_kv, 64)
        s["leaves"] = [s[n].requires_grad_() for n in ("q", "kv", "k_nope", "k_pe", "v") if n in s]
        if c["mask"] == "docs":
            lens, pad = _doc_lengths(S)
            starts, ends = [], []
            for _ in range(B):
                row, at = rng.sample(lens, len(lens)), 0
                for n in row:
                    starts += [at] * n
                    ends += range(at + 1, at + n + 1)
                    at += n
                starts += [0] * pad
                ends += [0] * pad
            s["starts"], s["ends"] = _int32(starts).view(B, S), _int32(ends).view(B, S)
        else:
            s["starts"] = s["ends"] = None
        s["scale"] = D ** -0.5
    elif kind == "paged":
        reqs = _requests(c)
        rng.shuffle(reqs)
        bs = c["block"]
        need = [-(-kv // bs) for kv, _ in reqs]
        W, blocks = max(need) + 1, sum(need) + 3
        order, at, table = torch.randperm(blocks, generator=g, device="cuda").tolist(), 0, []
        for n in need:
            table.append(order[at:at + n] + [-1] * (W - n))
            at += n
        starts = [0]
        for _, n in reqs:
            starts.append(starts[-1] + n)
        s["table"], s["kv_lens"], s["query_starts"] = _int32(table), _int32([kv for kv, _ in reqs]), _int32(starts)
        s["q"] = _normal(g, starts[-1], c["H"], c["d_qk"])
        rows = _normal(g, blocks * bs, c["d_qk"])
        if c["fmt"] == "mxfp4":
            rows = _pack_rows(rows[:, : c["d_v"]], rows[:, c["d_v"]:])
        s["cache"] = rows.view(blocks, bs, -1)
        s["scale"] = c["d_qk"] ** -0.5
        s["one"] = c["n_hi"] == 1
    elif kind == "cache":
        T, bs, blocks = c["T"], c["block"], c["blocks"]
        # the down-projection's row: latent and rope are views of it; magnitudes differ from channel to channel
        row = _normal(g, T, c["d_qk"]) * torch.exp(torch.randn(c["d_qk"], generator=g, device="cuda")).to(torch.bfloat16)
        s["latent"], s["rope"] = row[:, : c["d_v"]], row[:, c["d_v"]:]
        s["slots"] = torch.randperm(bs * blocks, generator=g, device="cuda")[:T]
        if c["fmt"] == "mxfp4":
            s["cache"] = torch.zeros(blocks, bs, _row_bytes(c["d_qk"], c["d_v"]), dtype=torch.uint8, device="cuda")
        else:
            s["cache"] = torch.zeros(blocks, bs, c["d_qk"], dtype=torch.bfloat16, device="cuda")
    else:
        R, bs = c["R"], c["block"]
        new, ctx = _spread(c["n_lo"], c["n_hi"], R), _spread(0, c["ctx"], R)
        rng.shuffle(new)
        rng.shuffle(ctx)
        done = [r % 13 == 5 for r in range(R)]
        rng.shuffle(done)
        W = (c["ctx"] + c["n_hi"]) // bs + 2
        held = [-(-n // bs) for n in ctx]
        blocks = sum(held) + R * (c["n_hi"] // bs + 1)
        order, at, table = torch.randperm(blocks, generator=g, device="cuda").tolist(), 0, []
        for n in held:
            table.append(order[at:at + n] + [-1] * (W - n))
            at += n
        s["context_lens"], s["query_lens"] = _int32(ctx), _int32([-1 if d else n for d, n in zip(done, new)])
        s["table"] = _int32(table)
        s["free"], s["free_count"] = _int32(order[at:] + [-1] * at), _int32([blocks - at])
        # a captured step's token count: what the requests may have at most
        s["tokens"] = R * c["n_hi"] + 3
    return s


# ---------------------------------------------------------------- plain forms


def _attend(q, k, v, lo, hi, scale, do=None):
    """Rows q [N, M, D] over keys k [N, K, D], values v [N, K, V], row m at keys [lo, hi) ([N, M]): out, lse2 and, for an
    upstream gradient, dq, dk, dv.  A row without keys: out 0, lse2 -inf, no gradient."""
    j = torch.arange(k.shape[1], device=k.device)
    off = (j < lo[..., None]) | (j >= hi[..., None])
    z = torch.matmul(q, k.transpose(1, 2)).mul_(scale).masked_fill_(off, -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = z.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse2 = (total.log() + top)[..., 0] * LOG2E
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = torch.matmul(p, v)
    if do is None:
        return out, lse2
    dv = torch.matmul(p.transpose(1, 2), do)
    ds = torch.matmul(do, v.transpose(1, 2)).sub_((out * do).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return out, lse2, torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2), q), dv


def _windows(s, copies):
    """lo, hi [B, S, copies]: a row's keys."""
    c = s["case"]
    B, S, S_kv = c["B"], c["S"], c["S_kv"]
    if c["mask"] == "docs":
        lo, hi = s["starts"], s["ends"]
    else:
        t = torch.arange(S, device="cuda")
        lo = torch.zeros(B, S, dtype=torch.int64, device="cuda")
        hi = (t + 1 + S_kv - S if c["mask"] == "causal" else torch.full_like(t, S_kv)).expand(B, S)
    return lo[..., None].expand(B, S, copies), hi[..., None].expand(B, S, copies)


def _absorbed_plain(s):
    c = s["case"]
    B, S, H, D, V = c["B"], c["S"], c["H"], c["d_qk"], c["d_v"]
    lo, hi = (x.reshape(B, S * H) for x in _windows(s, H))
    q, k, do = s["q"].detach().float().view(B, S * H, D), s["kv"].detach().float()[:, :, 0], s["do"].float().view(B, S * H, V)
    out, lse, dq, dkv, dv = _attend(q, k, k[..., :V].contiguous(), lo, hi, s["scale"], do)
    dkv[..., :V] += dv
    return dict(out=out.view(B, S, H, V).bfloat16(), lse=lse.view(B, S, H), dq=dq.view(B, S, H, D).bfloat16(),
                dkv=dkv[:, :, None].bfloat16())


def _expanded_plain(s):
    c = s["case"]
    B, S, K, H, D, V = c["B"], c["S"], c["S_kv"], c["H"], c["d_qk"], c["d_v"]
    lo, hi = (x.transpose(1, 2).reshape(B * H, S) for x in _windows(s, H))
    rows = lambda x: x.detach().float().transpose(1, 2).reshape(B * H, x.shape[1], -1)  # noqa: E731
    k = torch.cat([s["k_nope"].detach().float(), s["k_pe"].detach().float()[:, :, None].expand(B, K, H, 64)], dim=-1)
    out, lse, dq, dk, dv = _attend(rows(s["q"]), rows(k), rows(s["v"]), lo, hi, s["scale"], rows(s["do"]))
    back = lambda x: x.view(B, H, x.shape[1], -1).transpose(1, 2)  # noqa: E731
    dk = back(dk)
    return dict(out=back(out).bfloat16().contiguous(), lse=back(lse)[..., 0].contiguous(), dq=back(dq).bfloat16().contiguous(),
                dk_nope=dk[..., : D - 64].bfloat16().contiguous(), dk_pe=dk[..., D - 64:].sum(2).bfloat16(),
                dv=back(dv).bfloat16().contiguous())


def _pack_rows(latent, rope):
    """bf16 [T, d_v], [T, d_rope] -> MXFP4 cache rows uint8 [T, row bytes]: per 32 channels the scale is
    2^(floor(log2 amax) - 2), its exponent held to +-125 (all zeros: 2^0; Inf or NaN among them: byte 255), the codes are
    e2m1 of x / scale, nearest, ties to even, at most 6."""
    T, V = latent.shape
    x = latent.float().view(T, V // 32, 32)
    amax = x.abs().amax(-1)
    e = (torch.frexp(amax).exponent - 3).clamp(-125, 125)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    bad = ~torch.isfinite(x).all(-1)
    e = torch.where(bad, torch.zeros_like(e), e)
    a = torch.ldexp(x.abs(), -e[..., None])
    a = torch.where(bad[..., None], torch.zeros_like(a), a)
    # nearest of 0 0.5 1 1.5 2 3 4 6, whose codes are 0..7: a tie goes to the even code
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code | (torch.signbit(x).int() << 3)).to(torch.uint8).view(T, V // 2, 2)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    row = torch.zeros(T, _row_bytes(V + rope.shape[1], V), dtype=torch.uint8, device=latent.device)
    at = V // 2 + 2 * rope.shape[1]
    row[:, : V // 2] = code[..., 0] | code[..., 1] << 4
    row[:, V // 2: at] = rope.contiguous().view(torch.uint8)
    row[:, at: at + V // 32] = byte
    return row


def _unpack_rows(rows, d_qk, d_v, dtype):
    """MXFP4 cache rows uint8 [..., row bytes] -> [..., d_qk] values."""
    at = d_v // 2 + 2 * (d_qk - d_v)
    codes = torch.stack([rows[..., : d_v // 2] & 15, rows[..., : d_v // 2] >> 4], dim=-1).flatten(-2).long()
    value = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=dtype, device=rows.device)[codes & 7]
    value = torch.where(codes > 7, -value, value)
    byte = rows[..., at: at + d_v // 32].int()
    scale = torch.ldexp(torch.ones((), dtype=dtype, device=rows.device), byte - 127)
    scale = torch.where(byte == 255, torch.full_like(scale, math.nan), scale)
    latent = (value.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)
    rope = rows[..., d_v // 2: at].contiguous().view(torch.bfloat16).to(dtype)
    return torch.cat([latent, rope], dim=-1)


def _cached(s, dtype):
    """The requests' cached rows [R, longest, d_qk] (what lies behind a request's own is of block 0)."""
    c = s["case"]
    pos = torch.arange(c["kv_hi"], device="cuda")
    slot = s["table"].long().clamp(min=0)[:, pos // c["block"]] * c["block"] + pos % c["block"]
    rows = s["cache"].flatten(0, 1)[slot]
    return _unpack_rows(rows, c["d_qk"], c["d_v"], dtype) if c["fmt"] == "mxfp4" else rows.to(dtype)


def _paged_plain(s):
    c = s["case"]
    R, H, D, V, n = c["R"], c["H"], c["d_qk"], c["d_v"], c["n_hi"]
    k = _cached(s, torch.float32)
    first, count = s["query_starts"][:-1].long(), s["query_starts"].diff().long()
    i = torch.arange(n, device="cuda")
    at = (first[:, None] + i).clamp(max=s["q"].shape[0] - 1)                     # [R, n]: a short request's rest is dropped below
    hi = (s["kv_lens"].long() - count)[:, None] + i + 1
    hi = torch.minimum(hi, s["kv_lens"].long()[:, None])[..., None].expand(R, n, H).reshape(R, n * H)
    q = s["q"].float()[at].view(R, n * H, D)
    out, lse = _attend(q, k, k[..., :V].contiguous(), torch.zeros_like(hi), hi, s["scale"])
    owner = torch.repeat_interleave(torch.arange(R, device="cuda"), count, output_size=s["q"].shape[0])
    mine = torch.arange(s["q"].shape[0], device="cuda") - first[owner]
    return dict(out=out.view(R, n, H, V)[owner, mine].bfloat16(), lse=lse.view(R, n, H)[owner, mine])


def _cache_plain(s):
    c = s["case"]
    flat = s["cache"].flatten(0, 1)
    if c["fmt"] == "mxfp4":
        flat[s["slots"]] = _pack_rows(s["latent"], s["rope"])
        return dict(rows=_unpack_rows(flat[s["slots"]], c["d_qk"], c["d_v"], torch.float32).bfloat16())
    flat[s["slots"]] = torch.cat([s["latent"], s["rope"]], dim=-1)
    return dict(rows=flat[s["slots"]])


def _plan_plain(s):
    bs, T = s["case"]["block"], s["tokens"]
    table, free = s["table"].long(), s["free"].long()
    R, W = table.shape
    F = free.shape[0]
    ctx = s["context_lens"].long().clamp(0, W * bs)
    asked = s["query_lens"].long()
    done, n = asked < 0, asked.clamp(min=0)
    ends = n.cumsum(0)
    starts = ends - n
    held = (ctx + bs - 1) // bs
    fits = ~done & (ends <= T) & (ctx + n <= W * bs)
    need = torch.where(fits, (ctx + n + bs - 1) // bs - held, torch.zeros_like(n))
    upto = need.cumsum(0)
    have = s["free_count"].long().clamp(0, F)
    granted = fits & ((need == 0) | (upto <= have))
    got = torch.where(granted, need, torch.zeros_like(need))
    after = torch.where(granted, ctx + n, ctx)
    j = torch.arange(W, device="cuda")
    kth = (upto - need)[:, None] + j - held[:, None]                             # which of the step's new blocks
    fresh = (j >= held[:, None]) & (j < (held + got)[:, None])
    new = free[(have - 1 - kth).clamp(0, F - 1)]
    out = torch.where(fresh, new, torch.where((j < held[:, None]) & ~done[:, None], table, torch.full_like(table, -1)))
    tok = torch.arange(T, device="cuda")
    r = torch.searchsorted(ends, tok, right=True)
    real = r < R
    r = r.clamp(max=R - 1)
    real &= granted[r]
    pos = ctx[r] + tok - starts[r]
    block = out[r, (pos // bs).clamp(0, W - 1)]
    slots = torch.where(real & (block >= 0), block * bs + pos % bs, torch.full_like(pos, -1))
    kept = have - got.sum()
    back = torch.where(done, held, torch.zeros_like(held))
    to = kept + back.cumsum(0) - back
    where = torch.where(done[:, None] & (j < held[:, None]), to[:, None] + j, torch.full_like(table, F)).clamp(max=F)
    i = torch.arange(F + 1, device="cuda")
    left = torch.where(i < kept, torch.nn.functional.pad(free, (0, 1)), torch.full_like(i, -1))
    left = left.scatter(0, where.flatten(), table.flatten())[:F]
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    zero = torch.zeros_like(after)
    return dict(block_table=whole(out), slots=slots, positions=whole(torch.where(real, pos, torch.full_like(pos, -1))),
                query_starts=whole(torch.cat([starts[:1], ends]).clamp(max=T)), kv_lens=whole(torch.where(granted, after, zero)),
                context_lens=whole(torch.where(done, zero, after)), granted=whole(granted), free_blocks=whole(left),
                free_count=whole((kept + back.sum()).clamp(max=F)).view(1))


# ---------------------------------------------------------------- one pass


def _own(s):
    from cppmega_amd import latent_mla_ops as ops

    c, kind = s["case"], s["case"]["kind"]
    if kind == "absorbed":
        out, lse = ops.LatentMLA.apply(s["q"], s["kv"], s["scale"], c["d_v"], c["mask"] == "causal", s["starts"], s["ends"])
        dq, dkv = torch.autograd.grad(out, (s["q"], s["kv"]), s["do"])
        return dict(out=out.detach(), lse=lse.detach(), dq=dq, dkv=dkv)
    if kind == "expanded":
        leaves = (s["q"], s["k_nope"], s["k_pe"], s["v"])
        out, lse = ops.LatentMLAExpanded.apply(*leaves, s["scale"], c["mask"] == "causal", s["starts"], s["ends"])
        dq, dk_nope, dk_pe, dv = torch.autograd.grad(out, leaves, s["do"])
        return dict(out=out.detach(), lse=lse.detach(), dq=dq, dk_nope=dk_nope, dk_pe=dk_pe, dv=dv)
    if kind == "paged":
        cache = ops.LatentCache(s["cache"], c["d_qk"], c["d_v"])
        out, lse = ops.paged_latent_mla_fwd(s["q"], cache, s["table"], s["kv_lens"], None if s["one"] else s["query_starts"],
                                            sm_scale=s["scale"])
        return dict(out=out, lse=lse)
    if kind == "cache":
        cache = ops.LatentCache(s["cache"], c["d_qk"], c["d_v"])
        ops.latent_cache_append(cache, s["latent"], s["rope"], s["slots"])
        return dict(rows=ops.latent_cache_gather(cache, s["slots"]))
    p = ops.plan_latent_step(s["context_lens"], s["query_lens"], s["table"], s["free"], s["free_count"], s["tokens"], c["block"])
    return dict(block_table=p.block_table, slots=p.slots, positions=p.positions, query_starts=p.query_starts,
                kv_lens=p.kv_lens, context_lens=p.context_lens, granted=p.granted, free_blocks=p.free_blocks,
                free_count=p.free_count)


def run(state):
    if own:
        return _own(state)
    return {"absorbed": _absorbed_plain, "expanded": _expanded_plain, "paged": _paged_plain, "cache": _cache_plain,
            "plan": _plan_plain}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without


def _pairs(c):
    """(token, key) pairs of a training case, of one head."""
    B, S, K = c["B"], c["S"], c["S_kv"]
    if c["mask"] == "docs":
        return B * sum(n * (n + 1) // 2 for n in _doc_lengths(S)[0])
    return B * (S * K if c["mask"] == "full" else S * (K - S) + S * (S + 1) // 2)


def work(case):
    c, kind = case, case["kind"]
    if kind in ("absorbed", "expanded"):
        B, S, K, H, D, V = c["B"], c["S"], c["S_kv"], c["H"], c["d_qk"], c["d_v"]
        rows = K * D if kind == "absorbed" else K * (H * (D - 64 + V) + 64)
        size = 2 * B * (2 * S * H * (D + V) + 2 * rows) + 4 * B * S * H          # q, out, dO, dq; keys, values and gradients; lse
        return dict(bytes=size, flops=2 * H * _pairs(c) * (4 * D + 3 * V))       # forward, and the five products of the backward
    if kind == "paged":
        D, V, H = c["d_qk"], c["d_v"], c["H"]
        row = 2 * D if c["fmt"] == "bf16" else V // 2 + 2 * (D - V) + V // 32
        reqs = _requests(c)
        tokens = sum(n for _, n in reqs)
        pairs = sum(n * kv - n * (n - 1) // 2 for kv, n in reqs)
        return dict(bytes=sum(kv for kv, _ in reqs) * row + tokens * H * (2 * D + 2 * V + 4), flops=2 * H * (D + V) * pairs)
    if kind == "cache":
        row = 2 * c["d_qk"] if c["fmt"] == "bf16" else c["d_v"] // 2 + 2 * (c["d_qk"] - c["d_v"]) + c["d_v"] // 32
        return dict(bytes=c["T"] * (4 * c["d_qk"] + 2 * row + 16), flops=c["T"] * c["d_v"])
    W = (c["ctx"] + c["n_hi"]) // c["block"] + 2
    held = sum(-(-n // c["block"]) for n in _spread(0, c["ctx"], c["R"]))
    blocks = held + c["R"] * (c["n_hi"] // c["block"] + 1)
    # the held part of the table read, the whole written; both lists; slots and positions
    return dict(bytes=4 * held + 4 * c["R"] * W + 8 * blocks + 12 * (c["R"] * c["n_hi"] + 3) + 24 * c["R"], flops=c["R"] * W)


# ---------------------------------------------------------------- the same in 64 bits


def _softmax64(z):
    """Weights and log2 of the sum of e^z over the last axis; a row of -inf alone has weights 0."""
    lse = torch.logsumexp(z, dim=-1)
    p = torch.exp(z - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    return p, lse / math.log(2)


def _train_exact(s):
    """Head by head: scores, weights, and the gradients by the chain rule."""
    c = s["case"]
    B, S, K, H, D, V = c["B"], c["S"], c["S_kv"], c["H"], c["d_qk"], c["d_v"]
    absorbed = c["kind"] == "absorbed"
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    res = dict(out=new(B, S, H, V), lse=new(B, S, H), dq=new(B, S, H, D))
    if absorbed:
        res["dkv"] = new(B, K, 1, D)
    else:
        res |= dict(dk_nope=new(B, K, H, D - 64), dk_pe=new(B, K, 64), dv=new(B, K, H, V))
    key, t = torch.arange(K, device="cuda"), torch.arange(S, device="cuda")
    for b in range(B):
        if c["mask"] == "docs":
            seen = (key >= s["starts"][b, :, None]) & (key < s["ends"][b, :, None])
        elif c["mask"] == "causal":
            seen = key <= t[:, None] + (K - S)
        else:
            seen = torch.ones(S, K, dtype=torch.bool, device="cuda")
        for h in range(H):
            if absorbed:
                k = s["kv"][b, :, 0].detach().double()
                v = k[:, :V]
            else:
                k = torch.cat([s["k_nope"][b, :, h], s["k_pe"][b]], dim=1).detach().double()
                v = s["v"][b, :, h].detach().double()
            q, do = s["q"][b, :, h].detach().double(), s["do"][b, :, h].double()
            p, res["lse"][b, :, h] = _softmax64((q @ k.T * s["scale"]).masked_fill_(~seen, -math.inf))
            res["out"][b, :, h] = p @ v
            dp = do @ v.T
            dz = p * (dp - (p * dp).sum(1, keepdim=True)) * s["scale"]
            res["dq"][b, :, h] = dz @ k
            dk, dv = dz.T @ q, p.T @ do
            if absorbed:
                res["dkv"][b, :, 0] += dk
                res["dkv"][b, :, 0, :V] += dv
            else:
                res["dk_nope"][b, :, h], res["dv"][b, :, h] = dk[:, : D - 64], dv
                res["dk_pe"][b] += dk[:, D - 64:]
    return res


def _e2m1_64(latent):
    """The values that MXFP4 holds of bf16 rows, in 64 bits: the nearest representable one, by distance."""
    x = latent.double().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0 ** -140))).clamp(-123, 127) - 2)
    grid = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device="cuda")  # even codes first: they take ties
    near = grid[(torch.minimum(x.abs() / scale, grid[-1])[..., None] - grid).abs().argmin(-1)]
    return (torch.copysign(near, x) * scale).flatten(-2)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] in ("absorbed", "expanded"):
        return _train_exact(s)
    if c["kind"] == "paged":
        V, bs = c["d_v"], c["block"]
        out = torch.zeros(s["q"].shape[0], c["H"], V, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["q"].shape[0], c["H"], dtype=torch.float64, device="cuda")
        lens, first = s["kv_lens"].tolist(), s["query_starts"].tolist()
        for r, kv in enumerate(lens):
            rows = s["cache"][s["table"][r, : -(-kv // bs)].long()].flatten(0, 1)[:kv]
            if c["fmt"] == "mxfp4":
                half = rows[:, : V // 2].int()
                code = torch.stack([half % 16, half // 16], dim=2).reshape(kv, V // 32, 32)
                mag, e = (code % 8).double(), rows[:, V // 2 + 2 * (c["d_qk"] - V):][:, : V // 32].double()
                # e2m1: code 2 x + m is 2^(x - 1) (1 + m / 2), codes 0 and 1 are 0 and 1/2
                lat = torch.where(mag < 2, mag / 2, torch.exp2(torch.floor(mag / 2) - 1) * (1 + mag % 2 / 2))
                lat = torch.where(code > 7, -lat, lat) * torch.exp2(e - 127)[..., None]
                pe = rows[:, V // 2: V // 2 + 2 * (c["d_qk"] - V)].contiguous().view(torch.bfloat16).double()
                rows = torch.cat([lat.reshape(kv, V), pe], dim=1)
            rows = rows.double()
            n = first[r + 1] - first[r]
            seen = torch.arange(kv, device="cuda") <= torch.arange(kv - n, kv, device="cuda")[:, None]
            z = (s["q"][first[r]:first[r + 1]].double() @ rows.T * s["scale"]).masked_fill_(~seen[:, None], -math.inf)
            p, lse[first[r]:first[r + 1]] = _softmax64(z)
            out[first[r]:first[r + 1]] = p @ rows[:, :V]
        return dict(out=out, lse=lse)
    if c["kind"] == "cache":
        latent = _e2m1_64(s["latent"]) if c["fmt"] == "mxfp4" else s["latent"].double()
        return dict(rows=torch.cat([latent, s["rope"].double()], dim=-1))
    return None
