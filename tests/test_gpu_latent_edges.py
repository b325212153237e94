"""Latent attention where it can go wrong: what masked places hold, empty sizes, views, streams, graphs, every unit
size of the paged kernels, far offsets, and the operators together as a server and a trainer use them."""
import pytest
import torch

from cppmega_amd import latent_mla_ops as ops
from oracle import latent_cache as oc
from oracle import latent_mla as om
from tests.test_gpu_latent_mla import _docs, _mask, _normal, check, run_absorbed, run_expanded
from tests.test_gpu_latent_paged import DIMS, _cache_rows, _check, _paged_case

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


# ---------------------------------------------------------------- dense: masked places


@pytest.mark.parametrize("what", [NAN, INF, -INF, 3.0e38])
@pytest.mark.parametrize("d_qk,d_v", [(128, 64), (128, 128), (192, 128)])
def test_absorbed_keys_that_no_row_admits(dev, d_qk, d_v, what):
    """Padding may hold anything: every result as without it, its own gradients zero."""
    gen = torch.Generator().manual_seed(d_qk + d_v)
    B, S, H = 2, 150, 4
    q, kv, do = _normal(gen, B, S, H, d_qk), _normal(gen, B, S, 1, d_qk), _normal(gen, B, S, H, d_v)
    m = _mask(gen, "docs", B, S, S)
    lo, hi = om.windows(B, S, S, **m)
    ref = om.absorbed(q, kv, d_v, 0.1, lo, hi, do)
    for b in range(B):
        pad = ~((torch.arange(S) >= lo[b, :, None]) & (torch.arange(S) < hi[b, :, None])).any(0)
        assert pad.any()
        kv[b, pad] = what
        q[b, (hi <= lo)[b]] = what           # rows without keys as well
        do[b, (hi <= lo)[b]] = what
    check(run_absorbed(dev, q, kv, d_v, do, 0.1, m), ref, ("out", "lse", "dq", "dkv"))


@pytest.mark.parametrize("what", [NAN, INF])
def test_expanded_keys_that_no_row_admits(dev, what):
    gen = torch.Generator().manual_seed(5)
    B, S, S_kv, H = 1, 140, 200, 3
    q, do = _normal(gen, B, S, H, 192), _normal(gen, B, S, H, 128)
    kn, pe, v = _normal(gen, B, S_kv, H, 128), _normal(gen, B, S_kv, 64), _normal(gen, B, S_kv, H, 128)
    t = torch.arange(S).expand(B, S)
    m = dict(starts=(t + 5).to(torch.int32).contiguous(), ends=(t + 45).to(torch.int32).contiguous())
    ref = om.expanded(q, kn, pe, v, 0.07, *om.windows(B, S, S_kv, **m), do)
    for x in (kn, pe, v):
        x[:, :5] = what
        x[:, 185:] = what
    check(run_expanded(dev, q, kn, pe, v, do, 0.07, m), ref, ("out", "lse", "dq", "dk_nope", "dk_pe", "dv"))


@pytest.mark.parametrize("what", [NAN, INF])
@pytest.mark.parametrize("expanded", [False, True])
def test_a_document_is_not_reached_by_another(dev, what, expanded):
    """A key, a query row and a gradient row that are not finite stay within their own document."""
    gen = torch.Generator().manual_seed(9)
    S, H = 192, 4
    starts = torch.tensor([[0] * 70 + [70] * 50 + [120] * 72], dtype=torch.int32)
    ends = torch.arange(1, S + 1, dtype=torch.int32)[None].contiguous()
    m = dict(starts=starts, ends=ends)
    w = om.windows(1, S, S, **m)
    mine = torch.ones(S, dtype=torch.bool)
    mine[70:120] = False
    if expanded:
        x = [_normal(gen, 1, S, H, 128), _normal(gen, 1, S, H, 64), _normal(gen, 1, S, 64), _normal(gen, 1, S, H, 64)]
        do, names = _normal(gen, 1, S, H, 64), ("out", "lse", "dq", "dk_nope", "dk_pe", "dv")
        ref, run = om.expanded(*x, 0.1, *w, do), lambda: run_expanded(dev, *x, do, 0.1, m)
    else:
        x = [_normal(gen, 1, S, H, 128), _normal(gen, 1, S, 1, 128)]
        do, names = _normal(gen, 1, S, H, 64), ("out", "lse", "dq", "dkv")
        ref, run = om.absorbed(*x, 64, 0.1, *w, do), lambda: run_absorbed(dev, *x, 64, do, 0.1, m)
    for t in (*x, do):
        t[:, 90] = what
    got = run()
    check({n: got[n][:, mine.to(dev)] for n in names}, {k: v[:, mine] for k, v in ref.items()}, names)
    assert not torch.isfinite(got["out"][:, 90:120].float()).all()


@pytest.mark.parametrize("q_at,k_at", [(1.0, -INF), (3.0e38, -3.0e38)])
@pytest.mark.parametrize("form", ["absorbed", "expanded", "paged"])
def test_scores_of_minus_infinity(dev, q_at, k_at, form):
    """A document whose every score is -Inf (an Inf in its keys' rope part, or a product past fp32's range) has no weights:
    out 0, lse -Inf and no gradient, in every form; its neighbours are as without it."""
    gen = torch.Generator().manual_seed(19)
    S, H, D, V = 150, 4, 128, 64
    starts = torch.tensor([[0] * 60 + [60] * 50 + [110] * 40], dtype=torch.int32)
    m = dict(starts=starts, ends=torch.arange(1, S + 1, dtype=torch.int32)[None].contiguous())
    lo, hi = om.windows(1, S, S, **m)
    hi_ref = torch.where(starts == 60, lo, hi)      # the reference: that document sees no key
    q, do = _normal(gen, 1, S, H, D), _normal(gen, 1, S, H, V)
    q[:, 60:110, :, D - 1] = q_at
    if form == "expanded":
        x = [_normal(gen, 1, S, H, 64), _normal(gen, 1, S, 64), _normal(gen, 1, S, H, V)]
        ref, names = om.expanded(q, *x, 0.1, lo, hi_ref, do), ("out", "lse", "dq", "dk_nope", "dk_pe", "dv")
        x[1][:, 60:110, 63] = k_at
        got = run_expanded(dev, q, *x, do, 0.1, m)
    else:
        kv = _normal(gen, 1, S, 1, D)
        ref, names = om.absorbed(q, kv, V, 0.1, lo, hi_ref, do), ("out", "lse", "dq", "dkv")
        kv[:, 60:110, :, D - 1] = k_at
        if form == "absorbed":
            got = run_absorbed(dev, q, kv, V, do, 0.1, m)
        else:                                       # a document is a request, its tokens new
            cache = ops.LatentCache(kv.to(dev).view(15, 10, D), D, V)
            table = torch.tensor([[0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, -1], [11, 12, 13, 14, -1, -1]], dtype=torch.int32)
            lens, at = torch.tensor([60, 50, 40], dtype=torch.int32), torch.tensor([0, 60, 110, 150], dtype=torch.int32)
            out, lse = ops.paged_latent_mla_fwd(q[0].to(dev), cache, table.to(dev), lens.to(dev), at.to(dev), 0.1)
            got, names = dict(out=out[None], lse=lse[None]), ("out", "lse")
    check({n: got[n] for n in names}, ref, names)


@pytest.mark.parametrize("k_at", [-1.0e11, -1.0e14, -1.0e20, -1.0e29, -3.0e38])
@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_scores_far_below_the_others(dev, k_at, form):
    """Finite keys whose scores lie below -2^31 have no weight beside keys that come after them, and none by themselves."""
    gen = torch.Generator().manual_seed(29)
    S, H, D, V, n = 150, 4, 128, 64, 40
    t = torch.arange(1, S + 1)[None]
    lo, hi = torch.full((1, S), n), torch.where(t > n, t, n)     # the reference: the first n keys are not there
    lo[:, :n] = hi[:, :n] = 0
    q, do = _normal(gen, 1, S, H, D), _normal(gen, 1, S, H, V)
    q[..., D - 1] = 1.0
    if form == "expanded":
        x = [_normal(gen, 1, S, H, 64), _normal(gen, 1, S, 64), _normal(gen, 1, S, H, V)]
        ref, names = om.expanded(q, *x, 0.1, lo, hi, do), ("out", "lse", "dq", "dk_nope", "dk_pe", "dv")
        x[1][:, :n, 63] = k_at
        got = run_expanded(dev, q, *x, do, 0.1, dict(causal=True))
    else:
        kv = _normal(gen, 1, S, 1, D)
        ref, names = om.absorbed(q, kv, V, 0.1, lo, hi, do), ("out", "lse", "dq", "dkv")
        kv[:, :n, :, D - 1] = k_at
        got = run_absorbed(dev, q, kv, V, do, 0.1, dict(causal=True))
    check(got, ref, names)


@pytest.mark.parametrize("k_at", [-1.0e11, -1.0e20, -3.0e38])
@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H", [4, 40, 128])
def test_paged_scores_far_below_the_others(dev, k_at, d_qk, d_v, fmt, H):
    """The same over pages, in one piece and in several, for every kernel: the first pages' rows carry such a value in their
    rope part; the reference sees those pages as none."""
    gen = torch.Generator().manual_seed(H)
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, [4100, 90], [1, 2], 16)
    q[..., d_qk - 1] = 1.0
    rows = _cache_rows(cache)
    hidden = table.clone()
    hidden[0, :130], hidden[1, :2] = -1, -1
    ref = oc.paged(q, rows, hidden, starts, kv, 16, d_v, 0.1)
    pages = torch.cat([table[0, :130], table[1, :2]]).long()
    at = 2 * d_qk - 2 if fmt == "bf16" else d_v // 2 + 2 * (d_qk - d_v) - 2       # the last rope channel's bytes
    cache.data.view(torch.uint8)[pages.to(dev), :, at:at + 2] = torch.tensor([k_at], dtype=torch.bfloat16).view(torch.uint8).to(dev)
    _check(ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.1), ref)


@pytest.mark.parametrize("expanded", [False, True])
def test_a_row_of_nan_has_nan_results(dev, expanded):
    """A query row, or one key that rows admit, with NaN: out and lse of the rows that it reaches are NaN, of the others as
    without it."""
    gen = torch.Generator().manual_seed(27)
    S, H = 130, 2
    x = [_normal(gen, 1, S, H, 128), *((_normal(gen, 1, S, H, 64), _normal(gen, 1, S, 64), _normal(gen, 1, S, H, 64)) if expanded
                                       else (_normal(gen, 1, S, 1, 128),))]
    w = om.windows(1, S, S)
    ref = om.expanded(*x, 0.1, *w) if expanded else om.absorbed(*x, 64, 0.1, *w)
    x[0][:, 7, 1] = NAN
    x[1][:, 100:101, 0, 0] = NAN                    # expanded: of head 0 alone
    on = [t.to(dev) for t in x]
    out, lse = ops.latent_mla_expanded_fwd(*on, 0.1) if expanded else ops.latent_mla_fwd_interface(*on, 0.1, 64)
    hit = torch.zeros(1, S, H, dtype=torch.bool)
    hit[:, 7, 1] = True
    hit[:, 100:, :1 if expanded else H] = True
    assert out[hit.to(dev)].isnan().all() and lse[hit.to(dev)].isnan().all()
    check(dict(out=out[~hit.to(dev)], lse=lse[~hit.to(dev)]), {k: v[~hit] for k, v in ref.items()}, ("out", "lse"))


@pytest.mark.parametrize("S,S_kv", [(0, 5), (5, 0), (0, 0), (3, 1)])
@pytest.mark.parametrize("expanded", [False, True])
def test_empty_and_single(dev, S, S_kv, expanded):
    """No queries: the key gradients are zeros.  No keys: out 0, lse -inf, gradients 0.  More queries than keys."""
    gen = torch.Generator().manual_seed(S + S_kv)
    w = om.windows(2, S, S_kv)
    if expanded:
        x, do = [_normal(gen, 2, S, 3, 192), _normal(gen, 2, S_kv, 3, 128), _normal(gen, 2, S_kv, 64), _normal(gen, 2, S_kv, 3, 128)], _normal(gen, 2, S, 3, 128)
        check(run_expanded(dev, *x, do, None, dict(causal=True)), om.expanded(*x, 192 ** -0.5, *w, do),
              ("out", "lse", "dq", "dk_nope", "dk_pe", "dv"))
    else:
        x, do = [_normal(gen, 2, S, 6, 128), _normal(gen, 2, S_kv, 3, 128)], _normal(gen, 2, S, 6, 64)
        check(run_absorbed(dev, *x, 64, do, None, dict(causal=True)), om.absorbed(*x, 64, 128 ** -0.5, *w, do),
              ("out", "lse", "dq", "dkv"))


@pytest.mark.parametrize("poison", [False, True])
def test_more_row_tiles_than_a_search_holds(dev, poison):
    """Key gradients from 68 row tiles in one workgroup (128 heads: unsplit), few of which admit its keys: the search passes
    its 64 tiles, and with NaN in rows without keys it begins anew for the careful pass."""
    gen = torch.Generator().manual_seed(65)
    S, S_kv, H, heads = 4300, 256, 128, [0, 77, 127]
    starts, ends = torch.zeros(1, S, dtype=torch.int32), torch.zeros(1, S, dtype=torch.int32)
    for a, b, lo, hi in ((10, 150, 0, 100), (4170, 4200, 128, 250), (4230, 4290, 30, 120)):
        starts[:, a:b], ends[:, a:b] = lo, hi
    m = dict(starts=starts, ends=ends)
    q, do = _normal(gen, 1, S, H, 128), _normal(gen, 1, S, H, 64)
    x = [_normal(gen, 1, S_kv, H, 64), _normal(gen, 1, S_kv, 64), _normal(gen, 1, S_kv, H, 64)]
    some = lambda t: t[:, :, heads] if t.ndim == 4 else t  # noqa: E731
    ref = om.expanded(some(q), *(some(t) for t in x), 0.1, *om.windows(1, S, S_kv, **m), some(do))
    if poison:
        for t in (q, do):
            t[:, [0, 151, 4169, 4201, 4229, 4299]] = NAN
    got = run_expanded(dev, q, *x, do, 0.1, m)
    names = ("dq", "dk_nope", "dv")
    check({n: got[n][:, :, heads] for n in names}, ref, names)
    assert torch.isfinite(got["dk_pe"].float()).all()


def test_large_scores(dev):
    """Scores of hundreds: the running maximum moves, weights underflow, lse stays exact to its bound."""
    gen = torch.Generator().manual_seed(2)
    q, kv, do = 16 * _normal(gen, 1, 260, 2, 128), 16 * _normal(gen, 1, 260, 1, 128), _normal(gen, 1, 260, 2, 64)
    ref = om.absorbed(q, kv, 64, 0.3, *om.windows(1, 260, 260), do)
    got = run_absorbed(dev, q, kv, 64, do, 0.3, dict(causal=True))
    check(got, ref, ("lse",))
    assert all(torch.isfinite(got[n].float()).all() for n in got)


# ---------------------------------------------------------------- dense: views, order, streams, graphs


def test_broadcast_and_misaligned_views(dev):
    """Heads that share one key head by a stride of zero, batches that share a rope part, and views 2 bytes off."""
    gen = torch.Generator().manual_seed(12)
    B, S, S_kv, H = 2, 70, 90, 4
    q, do = _normal(gen, B, S, H, 192), _normal(gen, B, S, H, 128)
    kn, v = _normal(gen, B, S_kv, 1, 128), _normal(gen, 1, S_kv, H, 128)
    pe = _normal(gen, 1, S_kv, 65)
    big = pe.to(dev)
    views = (kn.to(dev).expand(B, S_kv, H, 128), big[..., 1:].expand(B, S_kv, 64), v.to(dev).expand(B, S_kv, H, 128))
    full = (kn.expand(B, S_kv, H, 128), pe[..., 1:].expand(B, S_kv, 64), v.expand(B, S_kv, H, 128))
    ref = om.expanded(q, *full, 0.1, *om.windows(B, S, S_kv), do)
    out, lse = ops.latent_mla_expanded_fwd(q.to(dev), *views, 0.1)
    got = ops.latent_mla_expanded_bwd(q.to(dev), *views, out, do.to(dev), lse, 0.1)
    check(dict(zip(("out", "lse", "dq", "dk_nope", "dk_pe", "dv"), (out, lse, *got))), ref,
          ("out", "lse", "dq", "dk_nope", "dk_pe", "dv"))
    # through autograd the shared head's gradient is the sum over the heads and batches, rounded once more
    leaf = kn.to(dev).requires_grad_()
    o, _ = ops.LatentMLAExpanded.apply(q.to(dev), leaf.expand(B, S_kv, H, 128), *views[1:], 0.1, None, None, None)
    (g,) = torch.autograd.grad(o, leaf, do.to(dev))
    want = ref["dk_nope"].sum(2, keepdim=True)
    tol = ref["e_dk_nope"].sum(2, keepdim=True)
    tol = tol + 2.0 ** -7 * (want.abs() + tol)     # the sum's own rounding, of a tree of bf16 or fp32 partial sums at most
    assert ((g.double().cpu() - want).abs() <= tol + 2.0 ** -8 * ref["dk_nope"].abs().sum(2, keepdim=True)).all()


def _off(t, dev):
    """``t`` on the device, contiguous, 2 bytes past an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)[1:]
    got = flat.view(t.shape).copy_(t)
    assert got.is_contiguous() and got.data_ptr() % 16 == 2
    return got


@pytest.mark.parametrize("expanded", [False, True])
def test_contiguous_but_misaligned(dev, expanded):
    """Leaves, and an upstream gradient (that of a concatenation behind an odd number of values), 2 bytes off."""
    gen = torch.Generator().manual_seed(61)
    S, H = 66, 2
    q, do = _normal(gen, 1, S, H, 128), _normal(gen, 1, S, H, 64)
    x = [_normal(gen, 1, S, H, 64), _normal(gen, 1, S, 64), _normal(gen, 1, S, H, 64)] if expanded else [_normal(gen, 1, S, 1, 128)]
    w = om.windows(1, S, S)
    ref = om.expanded(q, *x, 0.1, *w, do) if expanded else om.absorbed(q, *x, 64, 0.1, *w, do)
    leaves = [_off(t, dev).requires_grad_() for t in (q, *x)]
    out, lse = ops.LatentMLAExpanded.apply(*leaves, 0.1) if expanded else ops.LatentMLA.apply(*leaves, 0.1, 64)
    odd = torch.zeros(3, dtype=torch.bfloat16, device=dev, requires_grad=True)
    both = torch.cat([odd, out.flatten()])
    grads = torch.autograd.grad(both, leaves, torch.cat([torch.zeros(3, dtype=torch.bfloat16), do.flatten()]).to(dev))
    names = ("dq", "dk_nope", "dk_pe", "dv") if expanded else ("dq", "dkv")
    check(dict(zip(names, grads)) | dict(out=out, lse=lse), ref, ("out", "lse", *names))


def test_strides_of_axes_of_one(dev):
    """One key, one token: the stride of an axis of one says nothing, whatever it is."""
    gen = torch.Generator().manual_seed(62)
    q, do = _normal(gen, 1, 1, 2, 128), _normal(gen, 1, 1, 2, 64)
    x = [_normal(gen, 1, 1, 2, 64), _normal(gen, 1, 1, 64), _normal(gen, 1, 1, 2, 64)]
    odd = [t.to(dev).as_strided(t.shape, (5, 1 << 24, *t.stride()[2:])) for t in x]
    ref = om.expanded(q, *x, 0.1, *om.windows(1, 1, 1), do)
    out, lse = ops.latent_mla_expanded_fwd(q.to(dev), *odd, 0.1)
    got = ops.latent_mla_expanded_bwd(q.to(dev), *odd, out, do.to(dev), lse, 0.1)
    names = ("out", "lse", "dq", "dk_nope", "dk_pe", "dv")
    check(dict(zip(names, (out, lse, *got))), ref, names)
    for d_qk, d_v in DIMS:       # one token's row of a wider projection, at an odd place; then several, packed but off
        cache = ops.LatentCache.empty(1, 16, d_qk, d_v, "bf16", dev)
        row = _normal(gen, 1, d_qk + 3)
        on = row.to(dev)
        ops.latent_cache_append(cache, on[:, 3:3 + d_v], on[:, 3 + d_v:], torch.tensor([4], device=dev))
        assert torch.equal(cache.data[0, 4].cpu(), row[0, 3:])
        rows = _normal(gen, 5, d_qk)
        ops.latent_cache_append(cache, _off(rows[:, :d_v], dev), _off(rows[:, d_v:], dev), torch.arange(5, 10, device=dev))
        assert torch.equal(cache.data[0, 5:10].cpu(), rows)


def test_default_value_channels(dev):
    gen = torch.Generator().manual_seed(63)
    q, kv = _normal(gen, 1, 40, 2, 128).to(dev), _normal(gen, 1, 40, 1, 128).to(dev)
    want = ops.latent_mla_fwd_interface(q, kv, d_v=128)
    for got in (ops.latent_mla_fwd_interface(q, kv), ops.LatentMLA.apply(q, kv)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_three_axes_are_a_batch_of_one(dev):
    gen = torch.Generator().manual_seed(3)
    q, kv, do = (_normal(gen, 60, 4, 128).to(dev), _normal(gen, 60, 1, 128).to(dev), _normal(gen, 60, 4, 64).to(dev))
    starts, ends = (x[0].to(dev) for x in _docs(gen, 1, 60))
    out, lse = ops.latent_mla_fwd_interface(q, kv, None, 64, None, starts, ends)
    out4, lse4 = ops.latent_mla_fwd_interface(q[None], kv[None], None, 64, None, starts[None], ends[None])
    assert torch.equal(out, out4[0]) and torch.equal(lse, lse4[0])
    a = ops.latent_mla_bwd(q, kv, out, do, lse, None, None, starts, ends)
    b = ops.latent_mla_bwd(q[None], kv[None], out4, do[None], lse4, None, None, starts[None], ends[None])
    assert all(torch.equal(x, y[0]) for x, y in zip(a, b))


@pytest.mark.parametrize("expanded", [False, True])
def test_gradients_are_differences(dev, expanded):
    """The kernels' gradients along a random direction against the 64-bit difference quotient of the loss."""
    gen = torch.Generator().manual_seed(21)
    S, H = 90, 3
    lo, hi = om.windows(1, S, S)
    if expanded:
        x, do = [_normal(gen, 1, S, H, 128), _normal(gen, 1, S, H, 64), _normal(gen, 1, S, 64), _normal(gen, 1, S, H, 64)], _normal(gen, 1, S, H, 64)
        names, f = ("dq", "dk_nope", "dk_pe", "dv"), lambda *a: om.expanded(*a, 0.1, lo, hi)["out"]
        ref, got = om.expanded(*x, 0.1, lo, hi, do), run_expanded(dev, *x, do, 0.1, dict(causal=True))
    else:
        x, do = [_normal(gen, 1, S, H, 128), _normal(gen, 1, S, 1, 128)], _normal(gen, 1, S, H, 64)
        names, f = ("dq", "dkv"), lambda *a: om.absorbed(*a, 64, 0.1, lo, hi)["out"]
        ref, got = om.absorbed(*x, 64, 0.1, lo, hi, do), run_absorbed(dev, *x, 64, do, 0.1, dict(causal=True))
    x = [t.double() for t in x]
    for i, n in enumerate(names):
        d = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        side = lambda s: (f(*(t + s * h * d if j == i else t for j, t in enumerate(x))) * do.double()).sum()  # noqa: E731
        num = (side(1) - side(-1)) / (2 * h)
        tol = (ref["e_" + n] * d.abs()).sum() + 1e-6 * (1 + num.abs())
        assert (got[n].double().cpu() * d).sum().sub(num).abs() <= tol, n


def _train(gen, dev, S=300):
    q, kv = _normal(gen, 1, S, 8, 128).to(dev), _normal(gen, 1, S, 1, 128).to(dev)
    up, pe, do = _normal(gen, 1, S, 8, 128).to(dev), _normal(gen, 1, S, 64).to(dev), _normal(gen, 1, S, 8, 64).to(dev)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, kv, up, pe)]
        a, lse = ops.LatentMLA.apply(leaves[0], leaves[1], None, 64, True, None, None)
        b, lse2 = ops.LatentMLAExpanded.apply(leaves[0], leaves[2][..., :64], leaves[3], leaves[2][..., 64:], None, True, None, None)
        return [a, lse, b, lse2, *torch.autograd.grad((a, b), leaves, (do, do))]
    return (q, kv, up, pe, do), step


def test_repeats_and_streams(dev):
    """The same bits again, and on two streams at once."""
    _, step = _train(torch.Generator().manual_seed(4), dev)
    want = step()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    got = []
    for _ in range(3):
        for s in (a, b):
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for g in got for x, y in zip(g, want))


def test_graph_of_a_training_step(dev):
    """Both forms, forward and backward, captured on a side stream: replays after changed inputs and eager work."""
    ins, step = _train(torch.Generator().manual_seed(6), dev, 190)
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        held = step()
    for i in range(4):
        gen = torch.Generator().manual_seed(100 + i)
        for t in ins:
            t.copy_(_normal(gen, *t.shape))
        want = step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want)), i


# ---------------------------------------------------------------- paged: unit sizes, pieces, pages


UNITS = [
    # H, new tokens: every unit size of both widths, alone and as several units
    (5, [1, 1, 1]), (16, [1, 1, 1]), (24, [1, 1, 1]), (48, [1, 1, 1]), (80, [1, 1, 1]), (33, [4, 2, 4]), (128, [2, 2, 1]),
]


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H,news", UNITS)
def test_every_unit_size_in_pieces(dev, d_qk, d_v, fmt, H, news):
    """Lengths of thousands beside one key: units are cut into pieces over the workgroups and joined; a page that ends
    inside a tile, bad pages amid a request, lengths past the table."""
    gen = torch.Generator().manual_seed(H)
    lens = [4100, 9, 1555]
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, 24)
    table[0, 3], table[0, 77], table[2, 0] = -1, cache.num_blocks, -7
    kv[1] = 10 ** 6     # cut at the table's end, whose last entries are no pages
    ref = oc.paged(q, _cache_rows(cache), table, starts, kv, 24, d_v, 0.06)
    got = ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.06)
    _check(got, ref)
    again = ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.06)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("H", [16, 80])
def test_pages_of_one_row(dev, d_qk, d_v, H):
    """More pages than a workgroup's window of the table holds at once."""
    gen = torch.Generator().manual_seed(H)
    for fmt in ("bf16", "mxfp4"):
        cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, [2700], [1], 1)
        table[0, 1500] = -1
        ref = oc.paged(q, _cache_rows(cache), table, starts, kv, 1, d_v, 0.05)
        _check(ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), sm_scale=0.05), ref)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H", [4, 12, 40])
def test_keys_that_a_token_does_not_see(dev, d_qk, d_v, fmt, H):
    """Later tokens' keys, rows behind a request's last and pages of nobody hold NaN (bf16: Inf as well)."""
    gen = torch.Generator().manual_seed(H + d_qk)
    lens, news, bs = [70, 333], [4, 3], 16
    cache, table, kv, starts, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, lens, news, bs)
    used = torch.zeros(cache.num_blocks * bs, dtype=torch.bool)
    for r, n in enumerate(lens):
        k = torch.arange(n)
        used[table[r].long()[k // bs] * bs + k % bs] = True
    poison = torch.nonzero(~used)[:, 0]
    last = torch.stack([table[r, (n - 1) // bs].long() * bs + (n - 1) % bs for r, n in enumerate(lens)])  # the last token's own key
    clean = _cache_rows(cache)
    ref = oc.paged(q, clean, table, starts, kv, bs, d_v, 0.08)
    bad = torch.full((len(poison) + 2, d_qk), NAN, dtype=torch.bfloat16, device=dev)
    if fmt == "bf16":
        bad[::2] = INF
    ops.latent_cache_append(cache, bad[:, :d_v], bad[:, d_v:], torch.cat([poison, last]).to(dev))
    out, lse = ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.08)
    see = torch.ones(q.shape[0], dtype=torch.bool)
    see[[3, 6]] = False          # the last tokens see their own key
    _check((out[see.to(dev)], lse[see.to(dev)]), {k: v[see] for k, v in ref.items()})
    assert not torch.isfinite(out[~see.to(dev)].float()).all()


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("H", [16, 100])
def test_a_row_that_is_not_finite_stays_alone(dev, d_qk, d_v, H):
    gen = torch.Generator().manual_seed(8)
    cache, table, kv, starts, q = _paged_case(dev, gen, "bf16", d_qk, d_v, H, [900, 40], [2, 1], 32)
    ref = oc.paged(q, _cache_rows(cache), table, starts, kv, 32, d_v, 0.08)
    q[0, 3], q[1, 5] = NAN, INF
    out, lse = ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.08)
    ok = torch.ones(3, H, dtype=torch.bool)
    ok[0, 3] = ok[1, 5] = False
    _check((out[ok.to(dev)], lse[ok.to(dev)]), {k: v[ok] for k, v in ref.items()})
    assert out[0, 3].isnan().all() and lse[0, 3].isnan()


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("H", [8, 64, 128])
def test_rows_of_no_request_are_left(dev, d_qk, d_v, H):
    """A padded batch, shared pages, a strided-table neighbour: rows behind the last sequence keep what they held."""
    gen = torch.Generator().manual_seed(H)
    cache, table, kv, starts, q = _paged_case(dev, gen, "bf16", d_qk, d_v, H, [100, 0, 260], [3, 1, 2], 16)
    table[1] = table[2]                         # the prefix of another
    kv[1] = 130
    ref = oc.paged(q, _cache_rows(cache), table, starts, kv, 16, d_v, 0.1)
    pad = torch.cat([q, _normal(gen, 5, H, d_qk)])
    out = torch.full((11, H, d_v), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((11, H), -7.0, device=dev)
    got = ops.paged_latent_mla_fwd(pad.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), 0.1, out, lse)
    assert got[0] is out and got[1] is lse
    _check((out[:6], lse[:6]), ref)
    assert (out[6:] == 7).all() and (lse[6:] == -7).all()
    none = ops.paged_latent_mla_fwd(q[:0].to(dev), cache, table[:0].to(dev), kv[:0].to(dev))
    assert none[0].shape == (0, H, d_v) and none[1].shape == (0, H)


def test_starts_out_of_order_stay_in_bounds(dev):
    """Starts that fall, pass the batch or are negative: results of sound requests hold, nothing else is promised."""
    gen = torch.Generator().manual_seed(1)
    cache, table, kv, _, q = _paged_case(dev, gen, "bf16", 128, 64, 4, [50, 60, 70], [2, 2, 2], 16)
    starts = torch.tensor([0, 2, -5, 900], dtype=torch.int32)
    out, lse = ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), sm_scale=0.1)
    torch.cuda.synchronize()
    assert out.shape == (6, 4, 64)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("H", [4, 100])
def test_sound_requests_beside_bad_starts(dev, d_qk, d_v, fmt, H):
    """Negative starts, starts past the batch and one that falls claim no token: the two sound requests have their results,
    and nothing is written around them."""
    gen = torch.Generator().manual_seed(H)
    cache, table, kv, _, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, [50, 60, 170, 40, 30], [1, 3, 4, 1, 1], 16)
    T = 7
    q = q[:T].contiguous()
    starts = torch.tensor([-9, 0, 3, T, 900, -3], dtype=torch.int32)
    ref = oc.paged(q, _cache_rows(cache), table[1:3], torch.tensor([0, 3, T]), kv[1:3], 16, d_v, 0.1)
    out = torch.full((T + 16, H, d_v), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((T + 16, H), -7.0, device=dev)
    ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), kv.to(dev), starts.to(dev), 0.1, out[8:8 + T], lse[8:8 + T])
    _check((out[8:8 + T], lse[8:8 + T]), ref)
    for x, held in ((out, 7.0), (lse, -7.0)):
        assert (x[:8] == held).all() and (x[8 + T:] == held).all()


def test_many_starts_out_of_order(dev):
    """Row groups asked for pass 31 bits (512 requests that each claim nearly the whole batch of 2^29 rows: 512 * (2^22 + 11)
    groups of 128): the plan stays within its buffers, and the one sound request has its results."""
    T, H, R, bs = (1 << 22) + 16, 128, 1030, 16
    if torch.cuda.get_device_properties(dev).total_memory < 260 << 30:
        pytest.skip("208 GB of queries and results")
    gen = torch.Generator().manual_seed(77)
    cache = ops.LatentCache.empty(4, bs, 128, 64, "bf16", dev)
    rows = _normal(gen, 64, 128).to(dev)
    ops.latent_cache_append(cache, rows[:, :64], rows[:, 64:], torch.arange(64, device=dev))
    starts = torch.full((R + 1,), T, dtype=torch.int32)
    starts[0], starts[1:1026:2] = 0, 5              # request 0: five tokens; then every other one from token 5 to the end
    kv = torch.zeros(R, dtype=torch.int32)
    kv[0] = 60
    table = torch.arange(4, dtype=torch.int32)[None].expand(R, 4).contiguous()
    torch.cuda.empty_cache()
    try:
        q = torch.empty(T, H, 128, dtype=torch.bfloat16, device=dev)
        out, lse = torch.empty(T, H, 64, dtype=torch.bfloat16, device=dev), torch.empty(T, H, device=dev)
    except torch.OutOfMemoryError:
        pytest.skip("208 GB of queries and results")
    q[:5] = _normal(gen, 5, H, 128).to(dev)
    ops.paged_latent_mla_fwd(q, cache, table.to(dev), kv.to(dev), starts.to(dev), 0.1, out, lse)
    got, few = (out[:5].clone(), lse[:5].clone()), q[:5].cpu()
    torch.cuda.synchronize()
    del q, out, lse
    torch.cuda.empty_cache()
    ref = oc.paged(few, _cache_rows(cache), table[:1], starts[:2], kv[:1], bs, 64, 0.1)
    _check(got, ref)


@pytest.mark.parametrize("fmt,blocks", [("bf16", 60000), ("mxfp4", 176000)])
def test_offsets_past_32_bits(dev, fmt, blocks):
    """Rows behind 4 GiB of cache: append, gather and attention."""
    gen = torch.Generator().manual_seed(7)
    cache = ops.LatentCache.empty(blocks, 64, 576, 512, fmt, dev)
    assert cache.data[-3:].data_ptr() - cache.data.data_ptr() > 2 ** 32
    table = torch.tensor([[blocks - 1, 0, blocks - 3, 17, blocks // 2]], dtype=torch.int32)
    key = torch.arange(300)
    slots = table[0].long()[key // 64] * 64 + key % 64
    rows = _normal(gen, 300, 576)
    ops.latent_cache_append(cache, rows[:, :512].to(dev), rows[:, 512:].to(dev), slots.to(dev))
    back = ops.latent_cache_gather(cache, slots.to(dev)).cpu()
    if fmt == "bf16":
        assert torch.equal(back, rows)
    small = torch.arange(5, dtype=torch.int32)[None]
    for H in (16, 128):
        q = _normal(gen, 1, H, 576)
        ref = oc.paged(q, torch.cat([back, torch.zeros(20, 576)]).double(), small, [0, 1], [300], 64, 512, 0.05)
        _check(ops.paged_latent_mla_fwd(q.to(dev), cache, table.to(dev), torch.tensor([300], dtype=torch.int32, device=dev), sm_scale=0.05), ref)


# ---------------------------------------------------------------- together


def _serve(dev, fmt, H, S, bs, prompts, steps, captured):
    """Requests from their prompts on, token by token, as a server runs them: -> rows, queries and results per request."""
    gen = torch.Generator().manual_seed(31)
    R, W = len(prompts), -(-(max(prompts) + steps) // bs)
    F = R * W
    data = [(_normal(gen, p + steps, 128), _normal(gen, p + steps, H, 128)) for p in prompts]
    cache = ops.LatentCache.empty(F, bs, 128, 64, fmt, dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    state = [i32([0] * R), torch.full((R, W), -1, dtype=torch.int32, device=dev),
             torch.randperm(F, generator=gen).to(torch.int32).to(dev), i32([F])]
    results = [[] for _ in prompts]

    def step(ctx, table, free, count, new, rows, q):
        plan = ops.plan_latent_step(ctx, new, table, free, count, rows.shape[0], bs)
        ops.latent_cache_append(cache, rows[:, :64], rows[:, 64:], plan.slots)
        out, lse = ops.paged_latent_mla_fwd(q, cache, plan.block_table, plan.kv_lens, plan.query_starts)
        return out, lse, [plan.context_lens, plan.block_table, plan.free_blocks, plan.free_count], plan.granted

    n = sum(prompts) + 3                      # a padded batch
    rows, q = torch.zeros(n, 128, dtype=torch.bfloat16), torch.zeros(n, H, 128, dtype=torch.bfloat16)
    rows[:n - 3], q[:n - 3] = torch.cat([d[0][:p] for d, p in zip(data, prompts)]), torch.cat([d[1][:p] for d, p in zip(data, prompts)])
    out, lse, state, ok = step(*state, i32(prompts), rows.to(dev), q.to(dev))
    assert ok.all()
    at = 0
    for r, p in enumerate(prompts):
        results[r].append((out[at:at + p].cpu(), lse[at:at + p].cpu()))
        at += p
    one, held = i32([1] * R), [t.clone() for t in state]
    rows, q = torch.zeros(R, 128, dtype=torch.bfloat16, device=dev), torch.zeros(R, H, 128, dtype=torch.bfloat16, device=dev)
    graph = torch.cuda.CUDAGraph() if captured else None
    if captured:
        s = torch.cuda.Stream(dev)
        with torch.cuda.stream(s):
            step(*[t.clone() for t in held], i32([0] * R), rows, q)      # (no tokens: the cache stays)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            gout, glse, after, gok = step(*held, one, rows, q)
            for a, b in zip(held, after):
                a.copy_(b)
    for k in range(steps):
        rows.copy_(torch.stack([d[0][p + k] for d, p in zip(data, prompts)]))
        q.copy_(torch.stack([d[1][p + k] for d, p in zip(data, prompts)]))
        if captured:
            graph.replay()
            out, lse, ok = gout, glse, gok
        else:
            out, lse, state, ok = step(*state, one, rows, q)
        torch.cuda.synchronize()
        assert ok.all()
        for r in range(R):
            results[r].append((out[r:r + 1].cpu(), lse[r:r + 1].cpu()))
    return data, results


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("H", [4, 40])
def test_serving_is_training(dev, fmt, captured, H):
    """Plan, append and attention over prompts and decode steps give what the dense attention gives over the whole
    sequence at once: each within its bound of the 64-bit result over the cached rows."""
    prompts, steps = [37, 1, 130], 6
    data, results = _serve(dev, fmt, H, 0, 16, prompts, steps, captured)
    for (rows, q), got in zip(data, results):
        if fmt == "mxfp4":   # the rows as the cache holds them
            c = ops.LatentCache.empty(1, len(rows), 128, 64, fmt, dev)
            slots = torch.arange(len(rows), device=dev)
            ops.latent_cache_append(c, rows[:, :64].to(dev), rows[:, 64:].to(dev), slots)
            rows = ops.latent_cache_gather(c, slots).cpu()
        S = len(rows)
        ref = om.absorbed(q[None], rows[None, :, None], 64, 128 ** -0.5, *om.windows(1, S, S))
        ref = {k: v[0] for k, v in ref.items() if k in ("out", "e_out", "lse", "e_lse")}
        out, lse = (torch.cat(x) for x in zip(*got))
        check(dict(out=out, lse=lse), ref, ("out", "lse"))
        dense = ops.latent_mla_fwd_interface(q.to(dev), rows[:, None].contiguous().to(dev), d_v=64)
        check(dict(zip(("out", "lse"), dense)), ref, ("out", "lse"))
        assert ((out.double() - dense[0].double().cpu()).abs() <= 2 * ref["e_out"]).all()


def test_both_forms_are_one_attention(dev):
    """Expanded keys made from latent rows by an up-projection, and the same attention absorbed: q's nope part through
    the projection's transpose.  The absorbed query and the expanded keys are each rounded to bf16 once."""
    gen = torch.Generator().manual_seed(17)
    S, H, r, dn, dr = 96, 3, 64, 128, 64
    lat, pe, q = _normal(gen, 1, S, r), _normal(gen, 1, S, dr), _normal(gen, 1, S, H, dn + dr)
    wk = (torch.randn(H, dn, r, generator=gen) / 16).to(torch.bfloat16)
    kn = torch.einsum("bsr,hdr->bshd", lat.double(), wk.double()).to(torch.bfloat16)
    qa = torch.einsum("bshd,hdr->bshr", q[..., :dn].double(), wk.double()).to(torch.bfloat16)
    absorbed, kv = torch.cat([qa, q[..., dn:]], -1), torch.cat([lat, pe], -1)[:, :, None]
    v = lat[:, :, None].expand(1, S, H, r).contiguous()
    pad = torch.cat([v, torch.zeros(1, S, H, 128 - r, dtype=torch.bfloat16)], -1)   # (the expanded kernel's 128 value channels)
    scale = 192 ** -0.5
    a, lse_a = ops.LatentMLA.apply(absorbed.to(dev), kv.contiguous().to(dev), scale, 64, True, None, None)
    b, lse_b = ops.LatentMLAExpanded.apply(q.to(dev), kn.to(dev), pe.to(dev), pad.to(dev), scale, True, None, None)
    # either rounding moves a score by at most 2^-8 of sum |q| |k| (expanded: of q_nope and the keys; absorbed: of qa and the rows)
    s_e = torch.einsum("bshd,bthd->bhst", q[..., :dn].double().abs(), kn.double().abs()) * 2.0 ** -8 * scale
    s_a = torch.einsum("bshr,btr->bhst", qa.double().abs(), lat.double().abs()) * 2.0 ** -8 * scale
    seen = torch.ones(S, S).tril().bool()
    eps = (s_e + s_a).masked_fill(~seen, 0).amax(-1).transpose(1, 2) * 1.01      # [1, S, H], largest shift of a row's scores
    ref = om.absorbed(absorbed, kv, 64, scale, *om.windows(1, S, S))
    big = lat.double().abs().amax()
    move = torch.expm1(2 * eps)[..., None] * big                                  # |sum (p' - p) v| <= (e^(2 eps) - 1) max |v|
    assert ((a.double().cpu() - b[..., :64].double().cpu()).abs() <= move + 2 * ref["e_out"] + 2.0 ** -8 * big).all()
    assert ((lse_a.double().cpu() - lse_b.double().cpu()).abs() <= eps / 0.6931 + 2 * ref["e_lse"] + 1e-5).all()
    assert (b[..., 64:] == 0).all()


def test_trained_expanded_served_absorbed(dev):
    """A layer in its expanded form at the default scale, and served from the cache at that scale: one attention.  (The cached
    row's own width would give another scale.)"""
    gen = torch.Generator().manual_seed(18)
    S, H, r, dn, dr = 50, 3, 64, 128, 64
    lat, pe, q = _normal(gen, S, r), _normal(gen, S, dr), _normal(gen, S, H, dn + dr)
    wk = (torch.randn(H, dn, r, generator=gen) / 16).to(torch.bfloat16)
    kn = torch.einsum("sr,hdr->shd", lat.double(), wk.double()).to(torch.bfloat16)
    qa = torch.einsum("shd,hdr->shr", q[..., :dn].double(), wk.double()).to(torch.bfloat16)
    v = torch.cat([lat[:, None].expand(S, H, r), torch.zeros(S, H, 128 - r, dtype=torch.bfloat16)], -1)
    b, lse_b = (t[0] for t in ops.LatentMLAExpanded.apply(q[None].to(dev), kn[None].to(dev), pe[None].to(dev), v[None].to(dev)))
    cache = ops.LatentCache.empty(4, 16, 128, 64, "bf16", dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    plan = ops.plan_latent_step(i32([0]), i32([S]), i32([[-1] * 4]), i32([2, 0, 3, 1]), i32([4]), S, 16)
    ops.latent_cache_append(cache, lat.to(dev), pe.to(dev), plan.slots)
    scale = (dn + dr) ** -0.5
    a, lse_a = ops.paged_latent_mla_fwd(torch.cat([qa, q[..., dn:]], -1).to(dev), cache, plan.block_table, plan.kv_lens,
                                        plan.query_starts, sm_scale=scale)
    # qa and kn are each rounded once: a score moves by at most 2^-8 of sum |q| |k| on either side
    seen = torch.ones(S, S).tril().bool()
    move = (torch.einsum("shd,thd->hst", q[..., :dn].double().abs(), kn.double().abs())
            + torch.einsum("shr,tr->hst", qa.double().abs(), lat.double().abs())) * 2.0 ** -8 * scale
    eps = move.masked_fill(~seen, 0).amax(-1).T * 1.01
    ref = om.absorbed(torch.cat([qa, q[..., dn:]], -1)[None], torch.cat([lat, pe], -1)[None, :, None], 64, scale, *om.windows(1, S, S))
    big = lat.double().abs().amax()
    assert ((lse_a.double().cpu() - lse_b.double().cpu()).abs() <= eps / 0.6931 + 2 * ref["e_lse"][0] + 1e-5).all()
    assert ((a.double().cpu() - b[..., :64].double().cpu()).abs()
            <= torch.expm1(2 * eps)[..., None] * big + 2 * ref["e_out"][0] + 2.0 ** -8 * big).all()


def test_residual_is_what_rounding_took(dev):
    """out + residual is the output to 2^-17 beyond the products' own error, and with it the gradients' error falls to that
    of the weights' and the results' rounding (two of them, each at most half a step)."""
    gen = torch.Generator().manual_seed(23)
    S, H = 400, 4
    q, kv, do = _normal(gen, 1, S, H, 128), _normal(gen, 1, S, 1, 128), _normal(gen, 1, S, H, 64)
    m = dict(zip(("starts", "ends"), _docs(gen, 1, S)))
    ref = om.absorbed(q, kv, 64, 0.1, *om.windows(1, S, S, **m), do)
    w = {k: v.to(dev) for k, v in m.items()}
    plain = ops.latent_mla_fwd_interface(q.to(dev), kv.to(dev), 0.1, 64, **w)
    out, lse, low = ops.latent_mla_fwd_interface(q.to(dev), kv.to(dev), 0.1, 64, **w, residual=True)
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    assert (low.float().abs() <= 2.0 ** -8 * out.float().abs() + 1e-30).all()
    both = [ops.latent_mla_bwd(q.to(dev), kv.to(dev), out, do.to(dev), lse, 0.1, **w, residual=r) for r in (low, None)]
    off = [[float((g.double().cpu() - ref[n]).norm() / ref[n].norm()) for n, g in zip(("dq", "dkv"), x)] for x in both]
    assert all(a <= b for a, b in zip(*off)), off
    got = run_absorbed(dev, q, kv, 64, do, 0.1, m)
    assert torch.equal(got["dq"], both[0][0]) and torch.equal(got["dkv"], both[0][1])


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("fmt,H", [("bf16", 16), ("bf16", 100), ("mxfp4", 16), ("mxfp4", 100)])
def test_graph_of_paged_attention(dev, d_qk, d_v, fmt, H):
    """Captured on a side stream and replayed with other queries, lengths and tables, eager work between."""
    gen = torch.Generator().manual_seed(H)
    cache, table, kv, _, q = _paged_case(dev, gen, fmt, d_qk, d_v, H, [700, 64, 1], [1, 1, 1], 16)
    q, table, kv = q.to(dev), table.to(dev), kv.to(dev)
    s = torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        ops.paged_latent_mla_fwd(q, cache, table, kv, sm_scale=0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = ops.paged_latent_mla_fwd(q, cache, table, kv, sm_scale=0.1)
    for i, lens in enumerate(([700, 64, 1], [13, 700, 0], [1, 33, 650], [300, 300, 300])):
        q.copy_(_normal(gen, *q.shape))
        kv.copy_(torch.tensor(lens))
        table.copy_(table.roll(1, 0))
        want = ops.paged_latent_mla_fwd(q, cache, table, kv, sm_scale=0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]), i


def test_plan_keeps_its_inputs_and_results_apart(dev):
    """The inputs are not written, results of two calls share nothing, and a step repeated from the same state is the same."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    a = [i32([5, 0, 30]), i32([1, 20, -1]), i32([[3, -1, -1], [-1, -1, -1], [0, 1, -1]]), i32([2, 4, 5, 6, 7, 8]), i32([5])]
    before = [t.clone() for t in a]
    one = ops.plan_latent_step(*a, 24, 16)
    kept = [t.clone() for t in one]
    two = ops.plan_latent_step(*a, 24, 16)
    assert all(torch.equal(x, y) for x, y in zip(a, before))
    for t in two:
        t.fill_(-9)
    assert all(torch.equal(x, y) for x, y in zip(one, kept))
    for i, t in enumerate(one):      # nor do a call's own results overlap
        t.fill_(100 + i)
    assert all((t == 100 + i).all() for i, t in enumerate(one))


def test_gradient_of_a_sum(dev):
    """An upstream gradient that is a broadcast scalar, into leaves of which one takes none."""
    gen = torch.Generator().manual_seed(41)
    q, kv = _normal(gen, 1, 65, 4, 128), _normal(gen, 1, 65, 1, 128)
    ref = om.absorbed(q, kv, 64, 0.1, *om.windows(1, 65, 65), torch.ones(1, 65, 4, 64))
    a, b = q.to(dev), kv.to(dev).requires_grad_()
    out, lse = ops.LatentMLA.apply(a, b, 0.1, 64, None, None, None)
    out.sum().backward()
    check(dict(dkv=b.grad), ref, ("dkv",))
    assert not lse.requires_grad
    with torch.no_grad():
        assert torch.equal(ops.LatentMLA.apply(a, b, 0.1, 64, None, None, None)[0], out)


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -40, 4.0])
def test_scales(dev, scale):
    """From the least that is served (every weight 1 / n) to one where a row sees one key."""
    gen = torch.Generator().manual_seed(50)
    q, kv, do = _normal(gen, 1, 100, 4, 128), _normal(gen, 1, 100, 1, 128), _normal(gen, 1, 100, 4, 64)
    ref = om.absorbed(q, kv, 64, scale, *om.windows(1, 100, 100), do)
    if scale < 1:
        check(run_absorbed(dev, q, kv, 64, do, scale, dict(causal=True)), ref, ("out", "lse", "dkv"))
    else:
        got = run_absorbed(dev, q, kv, 64, do, scale, dict(causal=True))
        check(got, ref, ("lse",))
        assert all(torch.isfinite(t.float()).all() for t in got.values())
