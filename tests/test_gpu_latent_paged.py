"""The paged latent cache (append, gather, plan, attention) against the CPU oracle: bytes and
integers exactly, attention within the bounds that oracle/latent_mla.py derives."""
import pytest
import torch

from cppmega_amd import latent_mla_ops as ops
from oracle import latent_cache as orc

pytestmark = pytest.mark.gpu

DIMS = [(576, 512), (128, 64)]


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16)


def _cache_rows(cache):
    flat = cache.data.flatten(0, 1).cpu()
    return orc.unpack_rows(flat, cache.d_qk, cache.d_v) if cache.fmt == "mxfp4" else flat.double()


# ---------------------------------------------------------------- rows


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("T", [1, 7, 300])
def test_append_and_gather(dev, d_qk, d_v, fmt, T):
    gen = torch.Generator().manual_seed(T)
    bs, blocks = 16, 29
    rows = _normal(gen, T, d_qk + 8) * torch.exp2(torch.randint(-30, 30, (T, 1), generator=gen).float()).to(torch.bfloat16)
    rows[0, :32] = 0.0
    slots = torch.randperm(bs * blocks, generator=gen)[:T]
    if T > 4:
        slots[2], slots[3] = -1, bs * blocks      # outside the cache: skipped
    cache = ops.LatentCache.empty(blocks, bs, d_qk, d_v, fmt, dev)
    cache.data.view(torch.uint8).fill_(0xA5)
    before = cache.data.flatten(0, 1).view(torch.uint8).cpu()
    on = rows.to(dev)
    ops.latent_cache_append(cache, on[:, :d_v], on[:, d_v:d_qk], slots.to(dev))   # strided views
    after = cache.data.flatten(0, 1).view(torch.uint8).cpu()
    expect = before.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < bs * blocks:
            if fmt == "bf16":
                expect[s] = rows[t, :d_qk].contiguous().view(torch.uint8)
            else:
                b = orc.pack_row(rows[t, :d_v], rows[t, d_v:d_qk])
                n = sum(x is not None for x in b)
                expect[s, :n] = torch.tensor(b[:n], dtype=torch.uint8)
    assert torch.equal(after, expect)
    got = ops.latent_cache_gather(cache, slots.to(dev)).cpu().double()
    ok = (slots >= 0) & (slots < bs * blocks)
    assert torch.equal(got[ok], _cache_rows(cache)[slots[ok]])
    assert (got[~ok] == 0).all()


def test_mxfp4_every_code_and_scale(dev):
    """Every code under every exponent that the append writes reads back as its exact value, and the
    append gives the codes of values at, and next to, every border between two codes."""
    cache = ops.LatentCache.empty(8, 32, 576, 512, "mxfp4", dev)
    flat = cache.data.flatten(0, 1)
    gen = torch.Generator().manual_seed(3)
    raw = torch.randint(0, 256, (256, flat.shape[1]), generator=gen, dtype=torch.uint8)
    raw[:, 256:384] = 0
    raw[:, 384:] = torch.arange(256, dtype=torch.uint8)[:, None].clamp(2, 252)
    flat.copy_(raw)
    got = ops.latent_cache_gather(cache, torch.arange(256, device=dev)).cpu()
    assert torch.equal(got.double(), orc.unpack_rows(raw, 576, 512))
    edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 0.0], dtype=torch.float64)
    vals = torch.cat([edge, edge * (1 + 2 ** -7), edge * (1 - 2 ** -8)]).to(torch.bfloat16)   # neighbours in bf16
    blk = torch.zeros(32, dtype=torch.bfloat16)
    blk[:30], blk[30] = vals, 4.0
    blk[31] = -3.5
    rows = torch.stack([torch.cat([blk * s for s in torch.tensor([2.0 ** e for e in range(-120, 120, 15)]).to(torch.bfloat16)])])
    ops.latent_cache_append(cache, rows.to(dev), torch.zeros(1, 64, dtype=torch.bfloat16, device=dev), torch.tensor([5], device=dev))
    b = orc.pack_row(rows[0], torch.zeros(64, dtype=torch.bfloat16))
    assert flat[5].cpu().tolist() == b
    # the ends of the range, zeros, and blocks that are not finite
    rows = torch.zeros(1, 512, dtype=torch.bfloat16)
    rows[0, 0], rows[0, 32], rows[0, 64], rows[0, 97] = 3.38e38, 1e-40, float("inf"), float("nan")
    rows[0, 128:160] = -0.0
    ops.latent_cache_append(cache, rows.to(dev), torch.zeros(1, 64, dtype=torch.bfloat16, device=dev), torch.tensor([5], device=dev))
    b = orc.pack_row(rows[0], torch.zeros(64, dtype=torch.bfloat16))
    assert flat[5].cpu().tolist() == b
    back = ops.latent_cache_gather(cache, torch.tensor([5], device=dev)).cpu()[0]
    assert back[64:128].isnan().all() and torch.isfinite(back[:64]).all() and (back[128:] == 0).all()


# ---------------------------------------------------------------- plan


PLANS = [
    # context, new, W, free pages, count, T, block
    ([0], [1], 4, 8, 8, 1, 16),
    ([0, 15, 16, 17, 40], [1, 1, 1, 1, 0], 4, 16, 12, 6, 16),
    ([5, 33, 0, 64, 12], [-1, 3, 40, -1, 7], 5, 30, 9, 50, 16),
    ([10, 10, 10, 10], [20, 20, 20, 6], 8, 12, 3, 80, 16),       # the pool runs out at the second request
    ([10, 10, 10], [20, 20, 20], 8, 12, 12, 41, 16),             # the batch does at the third
    ([60, 3], [10, 10], 4, 12, 12, 20, 16),                      # a request passes its table
    ([-5, 1000, 7], [2, 1, -3], 3, 6, 100, 9, 16),               # lengths and counts out of range
    ([1] * 700, [1] * 700, 2, 1500, 1500, 703, 3),
    ([0] * 300, [2] * 300, 1, 90, 77, 600, 64),
    ([4000, 0], [0, 4000], 70, 200, 130, 4000, 64),
]


@pytest.mark.parametrize("ctx,new,W,F,count,T,bs", PLANS)
def test_plan(dev, ctx, new, W, F, count, T, bs):
    order, at = torch.randperm(4 * F, generator=torch.Generator().manual_seed(W)).tolist(), 0
    free = order[:F]
    at = F
    table = []
    for c in ctx:
        n = -(-max(0, min(c, W * bs)) // bs)
        table.append([(order * 4)[at + i] for i in range(n)] + [-1] * (W - n))
        at += n
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = ops.plan_latent_step(i32(ctx), i32(new), i32(table), i32(free), i32([count]), T, bs)
    ref = orc.plan(ctx, new, table, free, count, T, bs)
    for name in got._fields:
        assert getattr(got, name).cpu().tolist() == ref[name], name


HELD = [
    # context, pages in the table, new, W, free pages, count, T, block
    ([16], [2], [1], 4, 8, 8, 1, 16),                                       # a page that a draft took: not taken anew
    ([16, 1, 0, 33], [3, 1, 2, 3], [17, 40, 0, -1], 6, 20, 12, 60, 16),     # partly enough; unused; done with one behind
    ([5] * 300, [1 + i % 5 for i in range(300)], [i % 61 - 1 for i in range(300)], 70, 900, 700, 9001, 16),
    ([10, 3], [64, 0], [600, 900], 64, 90, 3, 1500, 16),                    # a table reserved whole; the pool runs out
    ([0, 20, 7], [5, 9, 8], [-1, -1, -1], 9, 30, 8, 4, 8),
]


@pytest.mark.parametrize("ctx,held,new,W,F,count,T,bs", HELD)
def test_plan_keeps_pages_behind_a_context(dev, ctx, held, new, W, F, count, T, bs):
    """Pages of tokens that were not kept: used before new ones, given back at the end."""
    gen = torch.Generator().manual_seed(W)
    held = [max(h, -(-c // bs)) for c, h in zip(ctx, held)]
    order = torch.randperm(F + sum(held), generator=gen).tolist()
    free, at, table = order[:F], F, []
    for n in held:
        table.append(order[at:at + n] + [-1] * (W - n))
        at += n
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = ops.plan_latent_step(i32(ctx), i32(new), i32(table), i32(free), i32([count]), T, bs)
    ref = orc.plan(ctx, new, table, free, count, T, bs)
    for name in got._fields:
        assert getattr(got, name).cpu().tolist() == ref[name], name


def test_rejected_drafts_lose_no_page(dev):
    """Many steps of draft tokens of which few are kept, across page borders, with requests that end and begin: every page
    is in exactly one table row or on the free list, and a kept token's page stays its own."""
    gen = torch.Generator().manual_seed(13)
    R, W, bs, F = 5, 6, 4, 26
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, free, count = i32([[-1] * W] * R), i32(list(range(F))), i32([F])
    ctx = [0] * R
    for step in range(80):
        draft = torch.randint(0, 7, (R,), generator=gen).tolist()
        new = [-1 if c + d > W * bs - 6 else d for c, d in zip(ctx, draft)]
        before = table.cpu().tolist()
        p = ops.plan_latent_step(i32(ctx), i32(new), table, free, count, 40, bs)
        table, free, count = p.block_table, p.free_blocks, p.free_count
        rows, n, ok = table.cpu().tolist(), int(count), p.granted.cpu().tolist()
        pages = [e for r in rows for e in r if e >= 0] + free.cpu().tolist()[:n]
        assert sorted(pages) == list(range(F)), step
        for r in range(R):
            if new[r] < 0:
                ctx[r] = 0
                continue
            kept = -(-ctx[r] // bs)
            assert rows[r][:kept] == before[r][:kept]
            if ok[r]:
                ctx[r] += int(torch.randint(0, new[r] + 1, (1,), generator=gen))


# ---------------------------------------------------------------- attention


def _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, bs, spare=2):
    need = [-(-kv // bs) for kv in lens]
    blocks = sum(need) + spare
    order, at, W = torch.randperm(blocks, generator=gen).tolist(), 0, max(need + [0]) + 1
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    cache = ops.LatentCache.empty(blocks, bs, d_qk, d_v, fmt, dev)
    rows = _normal(gen, blocks * bs, d_qk).to(dev)
    ops.latent_cache_append(cache, rows[:, :d_v], rows[:, d_v:], torch.arange(blocks * bs, device=dev))
    starts = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32)
    q = _normal(gen, int(starts[-1]), H, d_qk)
    return cache, table, torch.tensor(lens, dtype=torch.int32), starts, q


def _check(got, ref):
    for n, a in zip(("out", "lse"), got):
        a, e, tol = a.double().cpu(), ref[n], ref["e_" + n]
        known = ~torch.isnan(tol)
        bad = ~((a - e).abs() <= tol) & (a != e) & known
        assert not bad.any(), (n, int(bad.sum()), a[bad][:4], e[bad][:4], tol[bad][:4])


PAGED = [
    # H, key lengths, new tokens, block
    (16, [1], [1], 16),
    (1, [33, 5, 200], [1, 1, 1], 16),
    (128, [1, 31, 32, 33, 700], [1] * 5, 64),
    (8, [2000, 3], [1, 1], 64),
    (40, [257, 64, 1024], [1, 1, 1], 7),
    (16, [90, 5, 300], [3, 5, 1], 16),          # speculative tokens, a prompt without a prefix
    (20, [130, 40], [70, 33], 48),              # prefill chunks
    (4, [3, 0, 50], [7, 2, 0], 16),             # more tokens than keys, no keys, no tokens
]


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H,lens,news,bs", PAGED)
def test_paged(dev, d_qk, d_v, fmt, H, lens, news, bs):
    gen = torch.Generator().manual_seed(H + bs)
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, bs)
    ref = orc.paged(q, _cache_rows(cache), table, starts, kv, bs, d_v, d_qk ** -0.5)
    args = (q.to(dev), cache, table.to(dev), kv.to(dev))
    _check(ops.paged_latent_mla_fwd(*args, starts.to(dev)), ref)
    if all(n == 1 for n in news):
        _check(ops.paged_latent_mla_fwd(*args), ref)
