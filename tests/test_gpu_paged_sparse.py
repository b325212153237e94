"""The indexer's scores and top-k over paged index keys, sparse attention over the paged latent cache, and a served layer."""
import numpy as np
import pytest
import torch

from cppmega_amd import LayerNorm, layer_norm
from cppmega_amd import latent_mla_ops as lat
from cppmega_amd import paged_sparse_ops as ops
from cppmega_amd.sparse_mla_ops import sparse_mla_fwd_interface
from oracle import index_keys as orc
from oracle import layer_norm as oln
from oracle import topk as otk
from tests.test_gpu_latent_paged import DIMS, _cache_rows, _check, _normal, _paged_case

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32
NAN, INF = float("nan"), float("inf")
FMTS = ["bf16", "mxfp8", "mxfp4"]
SHAPES = [(16, 64), (32, 64), (64, 64), (16, 128), (32, 128), (64, 128)]


def _requests(gen, lens, news, bs, spare=2):
    need = [-(-kv // bs) for kv in lens]
    blocks = sum(need) + spare
    order, at, W = torch.randperm(blocks, generator=gen).tolist(), 0, max(need + [0]) + 1
    table = torch.full((len(lens), W), -1, dtype=I32)
    for r, n in enumerate(need):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=I32)
        at += n
    starts = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=I32)
    return table, torch.tensor(lens, dtype=I32), starts, blocks


def _score_case(dev, gen, fmt, H, d, lens, news, bs, wdtype=torch.float32):
    table, kv, starts, blocks = _requests(gen, lens, news, bs)
    T = int(starts[-1])
    cache = ops.IndexKeyCache.empty(blocks, bs, d, fmt, dev)
    ops.index_key_append(cache, _normal(gen, blocks * bs, d).to(dev), torch.arange(blocks * bs, device=dev))
    return cache, table, kv, starts, _normal(gen, T, H, d), torch.randn(T, H, generator=gen).to(wdtype)


def _compare(got, ref, tol):
    a = got.double().cpu()
    known = ~tol.isnan()
    same = (a == ref) | (a.isnan() & ref.isnan())
    bad = ~((a - ref).abs() <= tol) & ~same & known
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4], a[bad][:4], ref[bad][:4], tol[bad][:4])


REQUESTS = [
    # key lengths, new tokens, block
    ([1], [1], 16),
    ([33, 5, 200, 0], [1, 1, 1, 1], 16),
    ([700, 129, 128, 64, 2100], [1] * 5, 64),
    ([90, 5, 300], [3, 5, 2], 4),               # speculative tokens, a prompt without a prefix
    ([130, 40, 0, 77], [70, 33, 0, 9], 48),     # prefill chunks, a request without tokens
    ([3, 0, 50], [7, 2, 4], 16),                # more tokens than keys, no keys
    ([4500], [150], 64),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,d", SHAPES)
@pytest.mark.parametrize("lens,news,bs", REQUESTS)
def test_scores(dev, fmt, H, d, lens, news, bs):
    gen = torch.Generator().manual_seed(H + d + bs)
    cache, table, kv, starts, q, w = _score_case(dev, gen, fmt, H, d, lens, news, bs)
    L = table.shape[1] * bs
    ref, tol, limits = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), d), table, starts, kv, bs, L)
    args = (q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev))
    _compare(ops.paged_index_scores(*args, starts.to(dev)), ref, tol)
    if all(n == 1 for n in news):
        _compare(ops.paged_index_scores(*args), ref, tol)
    # fewer columns, an odd number of them, no ReLU, bf16 weights
    L = max(1, max(lens) - 3)
    wb = w.to(BF)
    ref, tol, _ = orc.scores(q, wb, orc.unpack_pages(cache.data.cpu(), d), table, starts, kv, bs, L, use_relu=False)
    _compare(ops.paged_index_scores(args[0], wb.to(dev), *args[2:], starts.to(dev), num_keys=L, use_relu=False), ref, tol)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("news", [[1, 1, 1], [40, 9, 3]])
def test_keys_that_are_not_seen(dev, fmt, news):
    """Pages outside the cache hide their keys; NaN behind a token's own position reaches nothing, a seen one its scores alone."""
    gen = torch.Generator().manual_seed(5)
    lens, bs, d, H = [300, 150, 64], 16, 128, 64
    cache, table, kv, starts, q, w = _score_case(dev, gen, fmt, H, d, lens, news, bs)
    flat = torch.arange(cache.num_blocks * bs, device=dev)
    bad = torch.full((1, d), NAN, dtype=BF, device=dev)
    unseen = [int(table[r, (n - 1) // bs]) * bs + (n - 1) % bs + 1 for r, n in enumerate(lens) if n % bs]
    unseen += [s for p in range(cache.num_blocks) if p not in table.tolist() and not (table == p).any() for s in range(p * bs, p * bs + bs)]
    for s in unseen:
        ops.index_key_append(cache, bad, flat[s:s + 1])
    at = int(table[0, 3]) * bs + 2                                   # position 50 of request 0
    ops.index_key_append(cache, bad, flat[at:at + 1])
    table[0, 7], table[1, 0] = cache.num_blocks + 3, -5
    rows = orc.unpack_pages(cache.data.cpu(), d)
    L = table.shape[1] * bs
    ref, tol, _ = orc.scores(q, w, rows, table, starts, kv, bs, L)
    assert ref[0, 50].isnan() and (ref[0, 112:128] == -INF).all()
    _compare(ops.paged_index_scores(q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev)), ref, tol)


def test_queries_and_weights_that_are_not_finite(dev):
    gen = torch.Generator().manual_seed(7)
    for news in ([1, 1, 1], [5, 20, 3]):
        cache, table, kv, starts, q, w = _score_case(dev, gen, "mxfp8", 64, 128, [60, 90, 33], news, 16)
        q[1, 3, 5], w[int(starts[2]), 9] = NAN, INF
        ref, tol, lim = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), 128), table, starts, kv, 16, 96)
        got = ops.paged_index_scores(q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), num_keys=96)
        keep = torch.ones(len(q), dtype=torch.bool)
        keep[1] = keep[int(starts[2])] = False
        _compare(got[keep.to(dev)], ref[keep], tol[keep])
        assert got[1, : int(lim[1])].isnan().all()
        assert not torch.isfinite(got[int(starts[2]), :20]).all()


@pytest.mark.parametrize("form", ["rows", "tiles"])
def test_rows_of_no_request_are_left(dev, form):
    """Tokens before the first and behind the last request keep what the output held."""
    gen = torch.Generator().manual_seed(3)
    lens, news = ([40, 70, 20, 33, 64, 10], [1] * 6) if form == "rows" else ([40, 70], [9, 30])
    cache, table, kv, starts, q, w = _score_case(dev, gen, "mxfp4", 32, 128, lens, news, 16)
    T = len(q)
    pad = lambda x: torch.cat([x[:2], x, x[:3]]).to(dev)  # noqa: E731
    held = torch.full((T + 5, 70), 3.25, device=dev)
    got = ops.paged_index_scores(pad(q), pad(w), cache, table.to(dev), kv.to(dev), (starts + 2).to(dev), num_keys=70, out=held)
    assert got is held and (held[:2] == 3.25).all() and (held[T + 2:] == 3.25).all()
    ref, tol, _ = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), 128), table, starts, kv, 16, 70)
    _compare(held[2:T + 2], ref, tol)
    picks = ops.paged_indexer_topk(pad(q), pad(w), cache, table.to(dev), kv.to(dev), 8, (starts + 2).to(dev))
    assert (picks[:2] == -1).all() and (picks[T + 2:] == -1).all() and (picks[2:T + 2, 0] >= 0).all()


@pytest.mark.parametrize("news", [[1] * 6, [30, 2, 0, 11, 1, 64]])
def test_topk(dev, news):
    """The picks are the top-k of the scores of the call itself; chunks of tokens give the same."""
    gen = torch.Generator().manual_seed(9)
    lens = [700, 20, 33, 512, 1, 300]
    cache, table, kv, starts, q, w = _score_case(dev, gen, "mxfp8", 16, 64, lens, news, 16)
    args = (q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev))
    L = 704
    s = ops.paged_index_scores(*args, starts.to(dev), num_keys=L)
    _, _, limits = orc.scores(q, w, orc.unpack_pages(cache.data.cpu(), 64), table, starts, kv, 16, L)
    want = otk.topk_ascending(s.cpu().numpy(), 64, np.zeros(len(q), dtype=np.int64), limits.numpy().astype(np.int64))
    got = ops.paged_indexer_topk(*args, 64, starts.to(dev), num_keys=L)
    assert np.array_equal(got.cpu().numpy(), want)
    for scratch in (0, 4 * L * 7, 4 * L * 33):
        assert torch.equal(ops.paged_indexer_topk(*args, 64, starts.to(dev), num_keys=L, max_scratch_bytes=scratch), got)
    assert torch.equal(ops.paged_indexer_topk(*args, 64, starts.to(dev)), got)


def test_topk_of_a_long_request(dev):
    """More keys than one pass of the top-k takes."""
    gen = torch.Generator().manual_seed(2)
    cache, table, kv, starts, q, w = _score_case(dev, gen, "mxfp4", 16, 64, [40001, 300], [1, 1], 64)
    args = (q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev))
    s = ops.paged_index_scores(*args).cpu()
    got = ops.paged_indexer_topk(*args, 500).cpu().numpy()
    want = otk.topk_ascending(s.numpy(), 500, np.zeros(2, dtype=np.int64), np.array([40001, 300]))
    assert np.array_equal(got, want)


# ---------------------------------------------------------------- sparse attention


def _picks(gen, T, topk, lims):
    """Positions in any order, with repeats, -1, positions past the token's own and far outside."""
    idx = torch.randint(0, 1 << 20, (T, topk), generator=gen)
    lim = torch.tensor(lims).clamp(min=1)[:, None]
    idx = (idx % lim).to(I32)
    kind = torch.rand(T, topk, generator=gen)
    idx[kind < 0.1] = -1
    idx[(kind > 0.1) & (kind < 0.13)] = 1 << 30
    return torch.where((kind > 0.13) & (kind < 0.2), lim.expand(T, topk).to(I32), idx)


def _lims(kv, starts):
    return [int(kv[r]) - (int(starts[r + 1]) - t) + 1 for r in range(len(kv)) for t in range(int(starts[r]), int(starts[r + 1]))]


SPARSE = [
    # H, key lengths, new tokens, block, topk
    (16, [1], [1], 16, 1),
    (1, [33, 5, 200], [1, 1, 1], 16, 7),
    (128, [31, 32, 700, 1500], [1] * 4, 64, 256),
    (16, [90, 5, 300], [3, 5, 1], 16, 65),
    (40, [257, 64, 1024], [1, 1, 1], 7, 100),
    (20, [130, 40], [70, 33], 48, 33),
    (4, [3, 0, 50], [7, 2, 4], 16, 64),
    (64, [900, 400], [11, 6], 64, 512),
    (32, [5000], [1], 64, 2048),
    (33, [700], [40], 16, 96),                  # two units of 32 rows a token
    (128, [1500], [60], 16, 128),               # many tokens: units that nearly fill the card, none of them cut
    (128, [700], [70], 16, 192),
    (80, [600], [130], 16, 96),
    (64, [600], [200], 16, 96),
    (16, [900], [300], 16, 160),
]


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H,lens,news,bs,topk", SPARSE)
def test_sparse(dev, d_qk, d_v, fmt, H, lens, news, bs, topk):
    gen = torch.Generator().manual_seed(H + bs + topk)
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, bs)
    idx = _picks(gen, len(q), topk, _lims(kv, starts))
    ref = orc.sparse(q, _cache_rows(cache), idx, table, starts, kv, bs, d_v, d_qk ** -0.5)
    args = (q.to(dev), cache, idx.to(dev), table.to(dev), kv.to(dev))
    got = ops.paged_sparse_mla_fwd(*args, starts.to(dev))
    _check(got, ref)
    again = ops.paged_sparse_mla_fwd(*args, starts.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    if all(n == 1 for n in news):
        _check(ops.paged_sparse_mla_fwd(*args), ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H", [16, 128])
def test_every_position_is_dense_attention(dev, d_qk, d_v, fmt, H):
    gen = torch.Generator().manual_seed(H)
    lens, news, bs = [120, 333, 64], [4, 1, 9], 16
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, bs)
    idx = torch.arange(340, dtype=I32).expand(len(q), 340).contiguous()
    args = (table.to(dev), kv.to(dev), starts.to(dev))
    from oracle import latent_cache as oc
    _check(ops.paged_sparse_mla_fwd(q.to(dev), cache, idx.to(dev), *args), oc.paged(q, _cache_rows(cache), table, starts, kv, bs, d_v, d_qk ** -0.5))


@pytest.mark.parametrize("d_qk,d_v", DIMS)
def test_as_sparse_mla(dev, d_qk, d_v):
    """The dense SparseMLA over the same rows: what a model trained with it serves."""
    gen = torch.Generator().manual_seed(1)
    S, H, topk, bs = 200, 32, 64, 16
    q, kv_rows = _normal(gen, S, H, d_qk), _normal(gen, S, d_qk)
    idx = torch.full((S, topk), -1, dtype=I32)
    for t in range(S):
        n = min(t + 1, topk)
        idx[t, :n] = torch.randperm(t + 1, generator=gen)[:n].sort().values.to(I32)
    out, lse = sparse_mla_fwd_interface(q[None].to(dev), kv_rows[None, :, None].to(dev), idx[None, :, None].to(dev), sm_scale=0.1, d_v=d_v)
    cache = lat.LatentCache.empty(14, bs, d_qk, d_v, "bf16", dev)
    table = torch.randperm(14, generator=gen)[None, :13].to(I32)
    pos = torch.arange(S)
    lat.latent_cache_append(cache, kv_rows[:, :d_v].to(dev), kv_rows[:, d_v:].to(dev), (table[0].long()[pos // bs] * bs + pos % bs).to(dev))
    one = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    got = ops.paged_sparse_mla_fwd(q.to(dev), cache, idx.to(dev), table.to(dev), one([S]), one([0, S]), sm_scale=0.1)
    ref = orc.sparse(q, _cache_rows(cache), idx, table, [0, S], [S], bs, d_v, 0.1)
    _check(got, ref)
    _check((out[0], lse[0]), ref)


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("d_qk,d_v", DIMS)
def test_rows_that_are_not_picked(dev, d_qk, d_v, what):
    gen = torch.Generator().manual_seed(6)
    H, lens, news, bs = 24, [150, 90], [6, 1], 16
    cache, table, kv, starts, q = _paged_case(dev, gen, "bf16", d_qk, d_v, H, lens, news, bs)
    idx = _picks(gen, len(q), 48, _lims(kv, starts))
    idx[idx == 17] = 16
    idx[2] = -1                                                       # nothing picked
    table[1, 2] = -1                                                  # a hidden page
    ref = orc.sparse(q, _cache_rows(cache), idx, table, starts, kv, bs, d_v, 0.1)
    flat = cache.data.flatten(0, 1)
    for r in range(2):
        flat[int(table[r, 1]) * bs + 1] = what                        # position 17
    used = {int(table[r, p]) for r in range(2) for p in range(-(-lens[r] // bs))}
    for p in set(range(cache.num_blocks)) - used:
        flat[p * bs:(p + 1) * bs] = what
    q[2] = what
    got = ops.paged_sparse_mla_fwd(q.to(dev), cache, idx.to(dev), table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.1)
    assert (got[0][2] == 0).all() and (got[1][2] == -INF).all()
    _check(got, ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H", [16, 64, 200])
def test_sparse_rows_of_no_request_are_left(dev, d_qk, d_v, fmt, H):
    gen = torch.Generator().manual_seed(8)
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, [60, 40], [2, 3], 16)
    idx = _picks(gen, 5, 32, _lims(kv, starts))
    ref = orc.sparse(q, _cache_rows(cache), idx, table, starts, kv, 16, d_v, d_qk ** -0.5)
    pad = lambda x: torch.cat([x[:1], x, x[:4]]).to(dev)  # noqa: E731
    out, lse = torch.full((10, H, d_v), 1.5, dtype=BF, device=dev), torch.full((10, H), 2.5, device=dev)
    ops.paged_sparse_mla_fwd(pad(q), cache, pad(idx), table.to(dev), kv.to(dev), (starts + 1).to(dev), out=out, lse=lse)
    rest = [0, 6, 7, 8, 9]
    assert (out[rest] == 1.5).all() and (lse[rest] == 2.5).all()
    _check((out[1:6], lse[1:6]), ref)


def test_many_tokens(dev):
    """More tokens than workgroups, cut and whole ones, early tokens with fewer keys than picks."""
    gen = torch.Generator().manual_seed(12)
    S, H, topk, bs, d_qk, d_v = 900, 8, 96, 16, 128, 64
    cache, table, kv, starts, q = _paged_case(dev, gen, "mxfp4", d_qk, d_v, H, [S], [S], bs)
    idx = torch.full((S, topk), -1, dtype=I32)
    for t in range(S):
        n = min(t + 1, topk)
        idx[t, :n] = torch.randperm(t + 1, generator=gen)[:n].sort().values.to(I32)
    ref = orc.sparse(q, _cache_rows(cache), idx, table, starts, kv, bs, d_v, d_qk ** -0.5)
    _check(ops.paged_sparse_mla_fwd(q.to(dev), cache, idx.to(dev), table.to(dev), kv.to(dev), starts.to(dev)), ref)


# ---------------------------------------------------------------- a served layer


def test_serving_steps(dev):
    """Prompts, then single tokens, of three requests, one of which ends: norm, append, top-k and attention as a server runs
    them, each step against the 64-bit results; then a decode step captured once and replayed on new data."""
    gen = torch.Generator().manual_seed(21)
    H, Hi, d, d_qk, d_v, bs, topk, R, F = 16, 32, 128, 128, 64, 16, 40, 3, 40
    keys = ops.IndexKeyCache.empty(F, bs, d, "mxfp8", dev)
    cache = lat.LatentCache.empty(F, bs, d_qk, d_v, "mxfp4", dev)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    nw, nb = (1 + 0.1 * torch.randn(d, generator=gen)).to(dev), (0.1 * torch.randn(d, generator=gen)).to(dev)
    table, free, count, ctx = i32([[-1] * 14] * R), i32(list(range(F))), i32([F]), i32([0] * R)

    def data(T):
        return dict(kx=_normal(gen, T, d).to(dev), lat=_normal(gen, T, d_qk).to(dev), qi=_normal(gen, T, Hi, d).to(dev),
                    w=torch.randn(T, Hi, generator=gen).to(dev), q=_normal(gen, T, H, d_qk).to(dev))

    def step(x, plan, starts):
        lat.latent_cache_append(cache, x["lat"][:, :d_v], x["lat"][:, d_v:], plan.slots)
        ops.index_key_append(keys, layer_norm(x["kx"], nw, nb, 1e-6), plan.slots)
        picks = ops.paged_indexer_topk(x["qi"], x["w"], keys, plan.block_table, plan.kv_lens, topk, starts)
        return picks, *ops.paged_sparse_mla_fwd(x["q"], cache, picks, plan.block_table, plan.kv_lens, starts, sm_scale=0.1)

    def verify(x, plan, got):
        picks, out, lse = got
        tb, st, kv = plan.block_table.cpu(), plan.query_starts.cpu(), plan.kv_lens.cpu()
        rows = orc.unpack_pages(keys.data.cpu(), d)
        s, tol, lim = orc.scores(x["qi"].cpu(), x["w"].cpu(), rows, tb, st, kv, bs, 14 * bs)
        for t in range(int(st[-1])):
            n = int(lim[t])
            mine = picks[t][picks[t] >= 0].cpu().long()
            assert mine.numel() == min(topk, n) and (mine.diff() > 0).all() and (mine < n).all()
            if n > topk:                                          # no key left out beats one that was picked by more than the bounds
                rest = torch.ones(n, dtype=torch.bool)
                rest[mine] = False
                assert (s[t, :n][rest] - tol[t, :n][rest]).max() <= (s[t, mine] + tol[t, mine]).min()
        _check((out, lse), orc.sparse(x["q"].cpu(), _cache_rows(cache), picks.cpu(), tb, st, kv, bs, d_v, 0.1))

    # new normed keys are the norm's
    x = data(70)
    _ = LayerNorm
    y = layer_norm(x["kx"], nw, nb, 1e-6)
    ref = oln.layer_norm(x["kx"].cpu(), nw.cpu(), nb.cpu(), 1e-6)
    assert ((y.double().cpu() - ref["y"]).abs() <= ref["e_y"]).all()
    for new in ([30, 25, 15], [1, 1, 1], [1, 1, 1], [64, -1, 1], [1, 9, 1]):
        T = 70
        plan = lat.plan_latent_step(ctx, i32(new), table, free, count, T, bs)
        x = data(T)
        got = step(x, plan, plan.query_starts)
        verify(x, plan, got)
        table, free, count, ctx = plan.block_table, plan.free_blocks, plan.free_count, plan.context_lens
    # a decode step in a graph: its inputs are copied in
    x, one = data(R), i32([1] * R)
    state = [t.clone() for t in (ctx, table, free, count)]
    def decode():
        plan = lat.plan_latent_step(state[0], one, state[1], state[2], state[3], R, bs)
        return plan, step(x, plan, None)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        plan, got = decode()
    for _ in range(4):
        fresh = data(R)
        for k in x:
            x[k].copy_(fresh[k])
        graph.replay()
        torch.cuda.synchronize()
        verify(x, plan, got)
        for a, b in zip(state, (plan.context_lens, plan.block_table, plan.free_blocks, plan.free_count)):
            a.copy_(b)


def test_on_another_stream(dev):
    gen = torch.Generator().manual_seed(14)
    cache, table, kv, starts, q, w = _score_case(dev, gen, "mxfp8", 64, 128, [200, 500], [1, 1], 16)
    args = (q.to(dev), w.to(dev), cache, table.to(dev), kv.to(dev))
    a, b = ops.paged_index_scores(*args), ops.paged_indexer_topk(*args, 30)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c, d = ops.paged_index_scores(*args), ops.paged_indexer_topk(*args, 30)
    side.synchronize()
    assert torch.equal(a, c) and torch.equal(b, d)
