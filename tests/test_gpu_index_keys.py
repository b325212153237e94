"""The paged cache of index keys against the CPU oracle: bytes and values exactly."""
import pytest
import torch

from cppmega_amd import paged_sparse_ops as ops
from oracle import index_keys as orc

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
FMTS = ["bf16", "mxfp8", "mxfp4"]


def _expected(before, k, slots, bs):
    """The cache's bytes after the append, from those before."""
    out = before.clone()
    if out.dtype == BF:
        flat = out.view(-1, out.shape[-1])
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < flat.shape[0]:
                flat[s] = k[t]
        return out
    pages, n = out.view(out.shape[0], -1), out.shape[2] - 4
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < out.shape[0] * bs:
            page, at = divmod(s, bs)
            codes, expo = orc.pack_key(k[t], "mxfp8" if n == k.shape[1] else "mxfp4")
            pages[page, at * n:(at + 1) * n] = torch.tensor(codes, dtype=torch.uint8)
            pages[page, bs * n + 4 * at: bs * n + 4 * at + 4] = torch.tensor(expo, dtype=torch.uint8)
    return out


def _bytes(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,bs", [(1, 64), (7, 16), (150, 12), (150, 4)])
def test_append_and_gather(dev, fmt, d, T, bs):
    gen = torch.Generator().manual_seed(T + bs)
    blocks = 160 // bs + 3
    wide = (torch.randn(T, d + 24, generator=gen) * torch.exp2(torch.randint(-30, 30, (T, 1), generator=gen).float())).to(BF)
    k = wide[:, 8:8 + d]
    k[0, :32] = 0.0
    slots = torch.randperm(bs * blocks, generator=gen)[:T]
    if T > 4:
        slots[2], slots[3] = -1, bs * blocks
    cache = ops.IndexKeyCache.empty(blocks, bs, d, fmt, dev)
    _bytes(cache.data).fill_(0x25)
    before = cache.data.cpu()
    ops.index_key_append(cache, wide.to(dev)[:, 8:8 + d], slots.to(dev))          # strided rows
    after = cache.data.cpu()
    assert torch.equal(_bytes(after), _bytes(_expected(before, k, slots, bs)))
    got = ops.index_key_gather(cache, slots.to(dev)).cpu().double()
    there = (slots >= 0) & (slots < bs * blocks)
    assert torch.equal(got[there], orc.unpack_pages(after, d)[slots[there]])
    assert (got[~there] == 0).all()
    odd = torch.zeros(T * d + 1, dtype=BF, device=dev)[1:].view(T, d)               # misaligned: copied
    odd.copy_(k)
    again = ops.IndexKeyCache(cache.data.clone(), d)
    ops.index_key_append(again, odd, slots.to(dev))
    assert torch.equal(_bytes(again.data), _bytes(cache.data))


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_every_code_reads_back(dev, fmt):
    d, bs = 128, 16
    cache = ops.IndexKeyCache.empty(16, bs, d, fmt, dev)
    n = cache.data.shape[2] - 4
    gen = torch.Generator().manual_seed(1)
    raw = torch.randint(0, 256, (16, bs * (n + 4)), generator=gen, dtype=torch.uint8)
    if fmt == "mxfp8":
        raw[:, : bs * n] = torch.arange(256, dtype=torch.uint8).repeat(bs * n // 256)
    least, most = (10, 246) if fmt == "mxfp8" else (2, 252)
    raw[:, bs * n:] = torch.randint(least, most + 1, (16, 4 * bs), generator=gen, dtype=torch.uint8)
    cache.data.view(16, -1).copy_(raw)
    got = ops.index_key_gather(cache, torch.arange(16 * bs, device=dev)).cpu().double()
    ref = orc.unpack_pages(raw.view(16, bs, n + 4), d)
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(), ref.nan_to_num())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_borders_of_codes_and_scales(dev, fmt):
    """Values at, and next to, the middle of two codes; largest magnitudes at, and next to, the borders of two scales; the ends
    of the exponents; zeros; blocks that are not finite."""
    d, bs, rows = 128, 16, []
    grid = sorted(set(orc.E4M3)) if fmt == "mxfp8" else list(orc.E2M1)
    top = 448.0 if fmt == "mxfp8" else 6.0
    mid = [(a + b) / 2 for a, b in zip(grid, grid[1:])]
    for i in range(0, len(mid), 10):
        m = torch.tensor(mid[i:i + 10], dtype=torch.float64)
        near = torch.cat([m, m * (1 + 2.0 ** -7), m * (1 - 2.0 ** -7)]).to(BF)       # exact in bf16, and its neighbours
        row = torch.zeros(d, dtype=BF)
        for blk, scale in enumerate((1.0, 2.0 ** -70, 2.0 ** 60, -1.0)):
            row[32 * blk: 32 * blk + near.numel()] = near * scale
            row[32 * blk + 31] = top * abs(scale)
        rows.append(row)
    for e in (-126, -118, -110, -60, 0, 60, 118, 119, 120, 126, 127):
        row = torch.randn(d, generator=torch.Generator().manual_seed(e)).clamp(-1, 1).to(BF) * 2.0 ** (e - 1)
        for blk, m in enumerate((1.0, 1.75, 1.7578125, 1.9921875)):
            row[32 * blk + 5] = m * 2.0 ** e
        rows.append(row)
    row = torch.zeros(d, dtype=BF)
    row[0], row[32], row[64], row[97] = 3.38e38, 1e-40, float("inf"), float("nan")
    row[98], row[33] = -2.0, -0.0
    rows.append(row)
    rows += [torch.zeros(d, dtype=BF), -torch.zeros(d, dtype=BF)]
    k = torch.stack(rows)
    slots = torch.arange(k.shape[0])
    cache = ops.IndexKeyCache.empty(k.shape[0] // bs + 1, bs, d, fmt, dev)
    cache.data.fill_(7)
    before = cache.data.cpu()
    ops.index_key_append(cache, k.to(dev), slots.to(dev))
    assert torch.equal(cache.data.cpu(), _expected(before, k, slots, bs))
    got = ops.index_key_gather(cache, slots.to(dev)).cpu().double()
    ref = orc.unpack_pages(cache.data.cpu(), d)[slots]
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(), ref.nan_to_num())
    assert got[-3, 64:].isnan().all() and torch.isfinite(got[-3, :64]).all()


def test_slots_far_into_a_large_cache(dev):
    """Byte offsets past 32 bits."""
    d, bs, blocks = 128, 64, 1 << 19                       # 8.6 GB of bf16 keys
    cache = ops.IndexKeyCache.empty(blocks, bs, d, "bf16", dev)
    slots = torch.tensor([0, 1 << 24, (1 << 24) + 1, bs * blocks - 1], device=dev)
    k = torch.randn(4, d, generator=torch.Generator().manual_seed(0)).to(BF).to(dev)
    ops.index_key_append(cache, k, slots)
    assert torch.equal(ops.index_key_gather(cache, slots), k)
    assert torch.equal(cache.data.view(-1, d)[slots], k)


def test_empty_calls(dev):
    cache = ops.IndexKeyCache.empty(2, 16, 64, "mxfp8", dev)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    ops.index_key_append(cache, torch.zeros(0, 64, dtype=BF, device=dev), none)
    assert ops.index_key_gather(cache, none).shape == (0, 64)
