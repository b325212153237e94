"""Edges of the paged index scores and of sparse attention over the paged latent cache: many requests, pages of one key, long
top-k, slots far into a large cache, calls side by side and in graphs."""
import pytest
import torch

from cppmega_amd import latent_mla_ops as lat
from cppmega_amd import paged_sparse_ops as ops
from cppmega_amd import topk_indices
from oracle import index_keys as orc
from tests.test_gpu_latent_paged import DIMS, _cache_rows, _check, _normal, _paged_case
from tests.test_gpu_paged_sparse import FMTS, INF, _compare, _lims, _picks, _score_case

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32


def _scores(dev, fmt, H, d, lens, news, bs, first=None, L=None):
    gen = torch.Generator().manual_seed(len(lens) + bs)
    cache, table, kv, starts, q, w = _score_case(dev, gen, fmt, H, d, lens, news, bs)
    L = table.shape[1] * bs if L is None else L
    ref = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), d), table, starts, kv, bs, L)
    return (q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev)), starts.to(dev), L, ref


# ---------------------------------------------------------------- scores


@pytest.mark.parametrize("news", ["one", "mixed", "empty"])
def test_many_requests(dev, news):
    """More requests than are numbered at once, some without tokens or keys, a whole 256 of them among them."""
    R = 700
    lens = [(37 * r) % 90 for r in range(R)]
    new = {"one": [1] * R, "mixed": [(r * 7) % 5 for r in range(R)], "empty": [0 if 200 <= r < 600 else 3 for r in range(R)]}[news]
    args, starts, L, (ref, tol, limits) = _scores(dev, "mxfp8", 16, 64, lens, new, 16)
    _compare(ops.paged_index_scores(*args, starts), ref, tol)
    if news == "one":
        _compare(ops.paged_index_scores(*args), ref, tol)
    picks = ops.paged_indexer_topk(*args, 8, starts).cpu()
    assert torch.equal((picks >= 0).sum(1).to(I32), limits.clamp(max=8))
    chunks = ops.paged_indexer_topk(*args, 8, starts, max_scratch_bytes=4 * L * 301).cpu()
    assert torch.equal(picks, chunks)


@pytest.mark.parametrize("news", [[1, 1, 1], [17, 3, 40]])
@pytest.mark.parametrize("fmt,bs", [("bf16", 1), ("bf16", 3), ("mxfp8", 4)])
def test_small_pages_of_long_requests(dev, fmt, bs, news):
    """Requests of more pages than a workgroup keeps at once."""
    n = 2048 * bs
    args, starts, _, (ref, tol, _) = _scores(dev, fmt, 16, 64, [n + n // 2 + 5, 30, n - 1], news, bs)
    _compare(ops.paged_index_scores(*args, starts), ref, tol)


@pytest.mark.parametrize("news", [[1], [9]])
def test_one_long_request(dev, news):
    """Keys past a window of large pages."""
    args, starts, _, (ref, tol, _) = _scores(dev, "mxfp4", 16, 64, [140_000], news, 128)
    _compare(ops.paged_index_scores(*args, starts), ref, tol)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,d", [(16, 64), (16, 128), (32, 64), (32, 128), (64, 128)])
@pytest.mark.parametrize("lens,news,bs", [([300, 77, 2100], [2, 2, 2], 16), ([90, 64, 0, 700, 33], [3, 1, 2, 0, 4], 64), ([50, 5], [4, 4], 4), ([1000], [2], 128),
                                          ([129, 4500, 3], [1, 7, 4], 16)])
def test_few_tokens(dev, fmt, H, d, lens, news, bs):
    """A few tokens of each request: units that they fill, or not."""
    args, starts, L, (ref, tol, limits) = _scores(dev, fmt, H, d, lens, news, bs)
    _compare(ops.paged_index_scores(*args, starts), ref, tol)
    part = max(1, max(lens) - 5)
    _compare(ops.paged_index_scores(*args, starts, num_keys=part), ref[:, :part], tol[:, :part])
    picks = ops.paged_indexer_topk(*args, 16, starts, max_scratch_bytes=4 * L * 3)     # chunks of three tokens
    assert torch.equal(picks, ops.paged_indexer_topk(*args, 16, starts))
    assert torch.equal((picks >= 0).sum(1).cpu().to(I32), limits.clamp(max=16))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H", [16, 32])
def test_few_tokens_and_keys_that_are_not_seen(dev, fmt, H):
    """NaN behind a token's own position, of a later token's key, reaches nothing; pages that are not there hide their keys."""
    gen = torch.Generator().manual_seed(15)
    lens, news, bs, d = [100, 66, 50], [3, 1, 2], 16, 128
    cache, table, kv, starts, q, w = _score_case(dev, gen, fmt, H, d, lens, news, bs)
    bad = torch.full((1, d), float("nan"), dtype=BF, device=dev)
    flat = torch.arange(cache.num_blocks * bs, device=dev)
    for r, pos in ((0, 99), (0, 40), (2, 49)):
        s = int(table[r, pos // bs]) * bs + pos % bs
        ops.index_key_append(cache, bad, flat[s:s + 1])
    table[0, 1], table[1, 0] = cache.num_blocks + 1, -3
    ref, tol, _ = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), d), table, starts, kv, bs, table.shape[1] * bs)
    assert ref[0, 40].isnan() and (ref[0, 98:] == -INF).all() and ref[2, 99].isnan() and (ref[1, 16:32] == -INF).all()
    _compare(ops.paged_index_scores(q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev)), ref, tol)


@pytest.mark.parametrize("L", [1, 2, 5, 63, 65, 127, 129, 321])
def test_odd_columns(dev, L):
    for news in ([1, 1, 1], [30, 8, 2]):
        args, starts, _, (ref, tol, _) = _scores(dev, "mxfp4", 32, 128, [321, 64, 0], news, 64, L=L)
        _compare(ops.paged_index_scores(*args, starts, num_keys=L), ref, tol)


@pytest.mark.parametrize("news", [[1, 1], [40, 9]])
def test_missing_pages_of_64_keys(dev, news):
    """Tiles that lie on one page, the page missing; NaN on the page that stands for it and behind the last key."""
    gen = torch.Generator().manual_seed(4)
    cache, table, kv, starts, q, w = _score_case(dev, gen, "bf16", 64, 128, [500, 290], news, 64)
    table[0, 2], table[1, 0], table[1, 4] = -1, cache.num_blocks, -7
    spare = [p for p in range(cache.num_blocks) if not (table == p).any()]
    cache.data[spare] = float("nan")
    cache.data[int(table[0, 7]), 500 % 64:] = float("nan")
    if 0 not in spare:                                               # page 0 is somebody's: it is moved, and left with NaN
        at = (table == 0).nonzero()[0]
        cache.data[spare[0]] = cache.data[0]
        table[at[0], at[1]] = spare[0]
        cache.data[0] = float("nan")
    ref, tol, _ = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), 128), table, starts, kv, 64, 512)
    assert (ref[0, 128:192] == -INF).all() and not ref.isnan().any()
    _compare(ops.paged_index_scores(q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), num_keys=512), ref, tol)


@pytest.mark.parametrize("lens,news", [([700, 20, 0, 512] * 5, [1] * 20), ([700, 20, 30, 512], [30, 2, 0, 11])])
def test_topk_over_a_scratch_that_held_anything(dev, lens, news):
    """Columns that no token sees are not written for the top-k, and not read."""
    args, starts, L, (_, _, limits) = _scores(dev, "mxfp8", 16, 64, lens, news, 64, L=4096 * 64)
    q, w, cache, table, kv = args
    table = torch.cat([table, torch.full((len(lens), 4096 - table.shape[1]), -1, dtype=I32, device=dev)], 1)
    T = len(q)
    s = ops.paged_index_scores(q, w, cache, table, kv, starts, num_keys=1024)
    want = topk_indices(s, 40, causal=False, starts=torch.zeros(T, dtype=I32, device=dev), ends=limits.to(dev))
    for value in (float("nan"), INF):
        for num_keys in (None, 1024, 40_000):
            n = T * (num_keys or L)
            held = torch.full((n,), value, device=dev)
            del held                                                   # its memory is the scratch's
            assert torch.equal(ops.paged_indexer_topk(q, w, cache, table, kv, 40, starts, num_keys=num_keys), want)
    assert torch.equal(ops.paged_indexer_topk(q, w, cache, table, kv, 300, starts, num_keys=128) >= 0,
                       torch.arange(300, device=dev)[None] < limits.clamp(max=128).to(dev)[:, None])   # more picks than columns


def test_nothing_to_score(dev):
    gen = torch.Generator().manual_seed(1)
    cache, table, kv, starts, q, w = _score_case(dev, gen, "mxfp8", 16, 64, [40, 20], [1, 1], 16)
    q, w, table, kv = q.to(dev), w.to(dev), table.to(dev), kv.to(dev)
    assert ops.paged_index_scores(q[:0], w[:0], cache, table[:0], kv[:0]).shape == (0, table.shape[1] * 16)
    assert ops.paged_index_scores(q, w, cache, table, kv, num_keys=0).shape == (2, 0)
    assert (ops.paged_indexer_topk(q, w, cache, table, kv, 4, num_keys=0) == -1).all()
    assert ops.paged_indexer_topk(q[:0], w[:0], cache, table[:0], kv[:0], 4).shape == (0, 4)
    none = torch.zeros(1, dtype=I32, device=dev)                      # no request: two tokens that belong to none
    held = torch.full((2, 16), 2.0, device=dev)
    ops.paged_index_scores(q, w, cache, table[:0], kv[:0], none, num_keys=16, out=held)
    assert (held == 2.0).all()
    assert (ops.paged_indexer_topk(q, w, cache, table[:0], kv[:0], 4, none) == -1).all()
    zero = torch.zeros(2, dtype=I32, device=dev)                      # requests without a key
    assert (ops.paged_index_scores(q, w, cache, table, zero) == -INF).all()
    assert (ops.paged_indexer_topk(q, w, cache, table, zero, 4) == -1).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_keys_far_into_a_large_cache(dev, fmt):
    """The same pages past the first 2^32 bytes give the same bits."""
    gen = torch.Generator().manual_seed(6)
    for news in ([1, 1], [30, 20]):
        cache, table, kv, starts, q, w = _score_case(dev, gen, fmt, 64, 128, [700, 90], news, 64)
        page = cache.data[0].numel() * cache.data.element_size()
        blocks = (1 << 32) // page + cache.num_blocks + 3
        far = ops.IndexKeyCache.empty(blocks, 64, 128, fmt, dev)
        far.data[-cache.num_blocks:] = cache.data
        moved = torch.where(table >= 0, table + (blocks - cache.num_blocks), table)
        args = (q.to(dev), w.to(dev))
        want = ops.paged_index_scores(*args, cache, table.to(dev), kv.to(dev), starts.to(dev))
        got = ops.paged_index_scores(*args, far, moved.to(dev), kv.to(dev), starts.to(dev))
        assert torch.equal(got, want)
        del far


# ---------------------------------------------------------------- sparse attention


def _sparse(dev, fmt, d_qk, d_v, H, lens, news, bs, topk, seed=0):
    gen = torch.Generator().manual_seed(seed + H + topk)
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, bs)
    idx = _picks(gen, len(q), topk, _lims(kv, starts))
    ref = orc.sparse(q, _cache_rows(cache), idx, table, starts, kv, bs, d_v, d_qk ** -0.5)
    return (q.to(dev), cache, idx.to(dev), table.to(dev), kv.to(dev), starts.to(dev)), ref


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H,news", [(1, [1]), (17, [2]), (128, [1, 1]), (16, [70, 69])])
def test_long_topk(dev, d_qk, d_v, fmt, H, news):
    """More picks than a workgroup keeps at once; with 139 tokens a range holds pieces of several tokens."""
    args, ref = _sparse(dev, fmt, d_qk, d_v, H, [6000, 5000][: len(news)], news, 64, 4500)
    _check(ops.paged_sparse_mla_fwd(*args), ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("H", [1, 8, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 256])
def test_head_counts(dev, d_qk, d_v, H):
    for fmt, T in (("bf16", 3), ("mxfp4", 45)):
        args, ref = _sparse(dev, fmt, d_qk, d_v, H, [150], [T], 16, 130)
        _check(ops.paged_sparse_mla_fwd(*args), ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("T,H,topk", [(5, 128, 320), (100, 20, 512), (128, 16, 192), (140, 16, 64), (140, 16, 200), (160, 16, 1000), (150, 32, 1900), (300, 16, 130),
                                      (300, 32, 700), (290, 33, 129), (520, 8, 200)])
def test_units_cut_and_whole(dev, d_qk, d_v, T, H, topk):
    """Numbers of tokens and picks at which units are cut, in equal pieces or by ranges of several, or left whole."""
    args, ref = _sparse(dev, "mxfp4" if T % 20 else "bf16", d_qk, d_v, H, [T + 50], [T], 16, topk)
    _check(ops.paged_sparse_mla_fwd(*args), ref)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("T,H,topk", [(257, 64, 320), (257, 64, 640), (257, 40, 1000), (130, 128, 640), (257, 16, 512), (300, 32, 640)])
def test_units_by_the_blocks_that_whole_ones_cost(dev, fmt, T, H, topk):
    """Both sides of the rule that leaves units whole, which differs by type and rows."""
    args, ref = _sparse(dev, fmt, 576, 512, H, [T + 700], [T], 16, topk)
    _check(ops.paged_sparse_mla_fwd(*args), ref)


@pytest.mark.parametrize("T,H", [(270, 100), (270, 65), (140, 200), (262, 127)])
@pytest.mark.parametrize("topk", [100, 1000])
def test_units_of_128_rows_with_fewer(dev, T, H, topk):
    """Many tokens, more than 64 heads, bf16: units of 128 rows of which some are no head's, whole and cut."""
    args, ref = _sparse(dev, "bf16", 576, 512, H, [T + 900], [T], 16, topk)
    _check(ops.paged_sparse_mla_fwd(*args), ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("H,T", [(16, 5), (16, 280), (64, 90), (128, 40), (128, 270)])
def test_tokens_without_picks(dev, d_qk, d_v, H, T):
    """Every other token picks nothing, or keys past its own alone; in cut units, whole ones and ranges of several."""
    args, _ = _sparse(dev, "bf16", d_qk, d_v, H, [T + 100], [T], 16, 200)
    q, cache, idx, table, kv, starts = args
    idx[::2] = -1
    idx[::4] = T + 100
    idx[1::4, :150] = -1                                             # the first blocks hold none
    idx[3::4, 70:] = -1                                              # the last ones
    ref = orc.sparse(q.cpu(), _cache_rows(cache), idx.cpu(), table.cpu(), starts.cpu(), kv.cpu(), 16, d_v, d_qk ** -0.5)
    out, lse = ops.paged_sparse_mla_fwd(*args)
    assert (out[::2] == 0).all() and (lse[::2] == -INF).all()
    _check((out, lse), ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
def test_one_position_over_and_over(dev, d_qk, d_v):
    """A repeated pick counts every time: its row's values, and log2 of the count in lse."""
    (q, cache, idx, table, kv, starts), _ = _sparse(dev, "bf16", d_qk, d_v, 20, [300], [4], 16, 256)
    one = ops.paged_sparse_mla_fwd(q, cache, torch.full_like(idx[:, :1], 77), table, kv, starts)
    many = ops.paged_sparse_mla_fwd(q, cache, torch.full_like(idx, 77), table, kv, starts)
    assert (many[0].float() - one[0].float()).abs().max() <= 2.0 ** -7 * one[0].float().abs().max()   # P's rounding and out's
    assert (many[1] - one[1] - 8.0).abs().max() <= 1e-4


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
def test_rows_far_into_a_large_cache(dev, d_qk, d_v, fmt):
    for H, news in ((16, [1, 1]), (128, [30, 20])):
        (q, cache, idx, table, kv, starts), _ = _sparse(dev, fmt, d_qk, d_v, H, [700, 90], news, 64, 200)
        page = cache.data[0].numel() * cache.data.element_size()
        blocks = (1 << 32) // page + cache.num_blocks + 3
        far = lat.LatentCache.empty(blocks, 64, d_qk, d_v, fmt, dev)
        far.data[-cache.num_blocks:] = cache.data
        moved = torch.where(table >= 0, table + (blocks - cache.num_blocks), table)
        want = ops.paged_sparse_mla_fwd(q, cache, idx, table, kv, starts)
        got = ops.paged_sparse_mla_fwd(q, far, idx, moved, kv, starts)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del far


@pytest.mark.parametrize("d_qk,d_v", DIMS)
def test_no_tokens(dev, d_qk, d_v):
    (q, cache, idx, table, kv, starts), _ = _sparse(dev, "bf16", d_qk, d_v, 16, [30], [2], 16, 8)
    out, lse = ops.paged_sparse_mla_fwd(q[:0], cache, idx[:0], table[:0], kv[:0])
    assert out.shape == (0, 16, d_v) and lse.shape == (0, 16)
    held, kept = torch.full((2, 16, d_v), 1.5, dtype=BF, device=dev), torch.full((2, 16), 2.5, device=dev)
    ops.paged_sparse_mla_fwd(q, cache, idx, table[:0], kv[:0], starts[:1], out=held, lse=kept)
    assert (held == 1.5).all() and (kept == 2.5).all()
    out, lse = ops.paged_sparse_mla_fwd(q, cache, idx, table, torch.zeros_like(kv), starts)
    assert (out == 0).all() and (lse == -INF).all()


# ---------------------------------------------------------------- calls side by side


@pytest.mark.parametrize("d_qk,d_v", DIMS)
def test_two_graphs_and_two_streams(dev, d_qk, d_v):
    """Two captured steps of different sizes, replayed in turn with eager calls between them and on two streams at once."""
    jobs = []
    for seed, (H, news) in enumerate((((16, [1, 1, 1]), (40, [20, 9])))):
        lens = [400, 90, 33][: len(news)]
        (q, cache, idx, table, kv, starts), _ = _sparse(dev, "mxfp4", d_qk, d_v, H, lens, news, 16, 160, seed)
        gen = torch.Generator().manual_seed(seed)
        keys = ops.IndexKeyCache.empty(cache.num_blocks, 16, 64, "mxfp8", dev)
        ops.index_key_append(keys, _normal(gen, cache.num_blocks * 16, 64).to(dev), torch.arange(cache.num_blocks * 16, device=dev))
        T = len(q)
        jobs.append(dict(q=q, cache=cache, keys=keys, qi=_normal(gen, T, 32, 64).to(dev), w=torch.randn(T, 32, generator=gen).to(dev),
                         req=(table, kv), starts=starts))

    def step(j):
        picks = ops.paged_indexer_topk(j["qi"], j["w"], j["keys"], *j["req"], 160, j["starts"])
        return (picks, *ops.paged_sparse_mla_fwd(j["q"], j["cache"], picks, *j["req"], j["starts"]))

    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    want, graphs, kept = [step(j) for j in jobs], [], []
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kept.append(step(j))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in jobs]
    for turn in range(3):
        for k in range(2):
            for x in kept[k]:
                x.zero_()
            graphs[k].replay()
            assert same(step(jobs[1 - k]), want[1 - k])
            torch.cuda.synchronize()
            assert same(kept[k], want[k])
        got = []
        for k, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append([step(jobs[k]) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(same(x, want[k]) for k in range(2) for x in got[k])
        for j in jobs:                                               # new inputs, which the graphs read
            j["q"].copy_(j["q"].flip(0).clone())
            j["w"].mul_(-1.0)
        want = [step(j) for j in jobs]
        torch.cuda.synchronize()
