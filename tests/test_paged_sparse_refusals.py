"""What the index-key cache, the paged scores, paged sparse attention and the layer norm refuse, on the CPU: every check comes
before the device's."""
import pytest
import torch

from cppmega_amd import LayerNorm, _lib, layer_norm, layer_norm_backward
from cppmega_amd import paged_sparse_ops as ops
from cppmega_amd._lib import DTYPE_BF16, DTYPE_E4M3, DTYPE_F32, DTYPE_MXFP4, DTYPE_MXFP8
from cppmega_amd.latent_mla_ops import LatentCache

BF = torch.bfloat16
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, -1, -2, -4
P = 1 << 20  # a pointer that is aligned and never read: each call ends at its check


def _t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _i32(*shape):
    return _t(*shape, dtype=torch.int32)


def _f32(*shape):
    return _t(*shape, dtype=torch.float32)


def _refused(error, f, *a, **k):
    with pytest.raises(error):
        f(*a, **k)


def test_cache_arguments():
    for data, d in ((_t(2, 16, 96), 96), (_t(2, 16, 64), 128), (_t(2, 16, 128).half(), 128), (_t(2, 16 * 128), 128), (_t(0, 16, 128), 128),
                    (_t(2, 16, 129)[..., :128], 128), (_t(2, 16, 133, dtype=torch.uint8), 128), (_t(2, 6, 132, dtype=torch.uint8), 128),
                    (_t(1, 65537, 64), 64), (_t(2, 16, 36, dtype=torch.uint8), 128)):
        _refused(AssertionError, ops.IndexKeyCache, data, d)
    _refused(AssertionError, ops.IndexKeyCache.empty, 2, 16, 128, "fp8", "cpu")
    _refused(AssertionError, ops.index_key_row_bytes, 128, "e4m3")
    for d, fmt, n in ((128, "bf16", 256), (128, "mxfp8", 132), (128, "mxfp4", 68), (64, "mxfp8", 68), (64, "mxfp4", 36)):
        assert ops.index_key_row_bytes(d, fmt) == n == _lib.load().dsa_index_key_row_bytes(d, ops.index_keys._CODES[fmt])
        assert ops.IndexKeyCache.empty(2, 16, d, fmt, "cpu").fmt == fmt
    c = ops.IndexKeyCache(_t(2, 16, 128))
    slots = _t(3, dtype=torch.int64)
    for a in ((_t(3, 64), slots), (_t(3, 128), slots[:2]), (_t(3, 128), slots.int()), (_t(3, 128).half(), slots), (_t(3, 1, 128), slots)):
        _refused(AssertionError, ops.index_key_append, c, *a)
    _refused(RuntimeError, ops.index_key_append, c, _t(3, 128), slots)
    _refused(AssertionError, ops.index_key_gather, c, slots.int())
    _refused(RuntimeError, ops.index_key_gather, c, slots)


def test_score_arguments():
    c = ops.IndexKeyCache(_t(2, 16, 128))
    q, w, table, kv = _t(3, 16, 128), _f32(3, 16), _i32(3, 4), _i32(3)
    for f, more in ((ops.paged_index_scores, ()), (ops.paged_indexer_topk, (8,))):
        for a, k in (((q[0], w, c, table, kv), {}), ((_t(3, 16, 64), w, c, table, kv), {}), ((q.half(), w, c, table, kv), {}),
                     ((q, w[:2], c, table, kv), {}), ((q, w.double(), c, table, kv), {}), ((q, w.t().contiguous().t(), c, table, kv), {}),
                     ((q, w, c, table[:2], kv), {}), ((q, w, c, table.long(), kv), {}), ((q, w, c, table, kv.long()), {}),
                     ((q, w, c, _i32(3, 8)[:, ::2], kv), {}), ((_t(4, 16, 128), _f32(4, 16), c, table, kv), {}),
                     ((q, w, c, table, kv), dict(query_starts=_i32(3))), ((q, w, c, table, kv), dict(num_keys=65)),
                     ((q, w, c, table, kv), dict(num_keys=-1))):
            _refused(AssertionError, f, *a, *more, **k)
        _refused(RuntimeError, f, q, w, c, table, kv, *more)
    _refused(AssertionError, ops.paged_indexer_topk, q, w, c, table, kv, 0)


def test_sparse_arguments():
    c = LatentCache(_t(2, 16, 128), 128, 64)
    q, idx, table, kv = _t(3, 2, 128), _i32(3, 8), _i32(3, 4), _i32(3)
    f = ops.paged_sparse_mla_fwd
    for a, k in (((q[0], c, idx, table, kv), {}), ((_t(3, 2, 192), c, idx, table, kv), {}), ((q.half(), c, idx, table, kv), {}),
                 ((q, c, idx[:2], table, kv), {}), ((q, c, idx.long(), table, kv), {}), ((q, c, _i32(3, 0), table, kv), {}),
                 ((q, c, _i32(3, 16)[:, ::2], table, kv), {}), ((q, c, _i32(3, 1, 8), table, kv), {}),
                 ((q, c, idx, table[:2], kv), {}), ((q, c, idx, table, kv.long()), {}), ((_t(4, 2, 128), c, _i32(4, 8), table, kv), {}),
                 ((q, c, idx, table, kv), dict(query_starts=_i32(3)))):
        _refused(AssertionError, f, *a, **k)
    for scale in (0.0, -1.0, 1e-38, float("inf"), float("nan")):
        _refused(ValueError, f, q, c, idx, table, kv, sm_scale=scale)
    _refused(RuntimeError, f, q, c, idx, table, kv)


def test_layer_norm_arguments():
    x, w, b = _t(3, 64), _t(64), _t(64)
    for a in ((x.half(), w, b), (x, w[:63], b), (x, w, b.float()), (x, w.half(), None), (x, w, _t(1, 64)), (_t(3, 0), None, None), (_t(), None, None)):
        _refused(AssertionError, layer_norm, *a)
        _refused(AssertionError, LayerNorm.apply, *a)
    for eps in (-1.0, float("inf"), float("nan")):
        _refused(ValueError, layer_norm, x, w, b, eps)
    _refused(RuntimeError, layer_norm, x, w, b)
    mean, rstd = _f32(3), _f32(3)
    for a in ((x[:2], x, w, mean, rstd), (x.float(), x, w, mean, rstd), (x, x, w, mean[:2], rstd), (x, x, w, mean, rstd.double()),
              (x, x, w[:3], mean, rstd)):
        _refused(AssertionError, layer_norm_backward, *a)
    _refused(RuntimeError, layer_norm_backward, x, x, w, mean, rstd)


# ---------------------------------------------------------------- the C entry points (nothing is launched)


def test_c_index_keys():
    L = _lib.load()
    add = lambda **k: L.dsa_index_key_append(*({**dict(c=P, k=P, ks=128, s=P, T=3, nb=2, bs=16, D=128, dt=DTYPE_MXFP8, st=None), **k}).values())  # noqa: E731
    get = lambda **k: L.dsa_index_key_gather(*({**dict(c=P, s=P, o=P, T=3, nb=2, bs=16, D=128, dt=DTYPE_MXFP4, st=None), **k}).values())  # noqa: E731
    for f in (add, get):
        for k in (dict(nb=0), dict(nb=1 << 31), dict(bs=0), dict(bs=65537), dict(bs=6), dict(dt=DTYPE_E4M3), dict(T=-1), dict(T=1 << 31), dict(c=None),
                  dict(c=P + 8), dict(s=None)):
            assert f(**k) == INVALID, k
        assert f(D=96) == UNSUPPORTED and f(T=0, c=None) == OK
    assert add(k=P + 2) == add(ks=-8) == add(ks=12) == get(o=None) == get(o=P + 4) == INVALID
    assert L.dsa_index_key_row_bytes(96, DTYPE_BF16) == L.dsa_index_key_row_bytes(64, DTYPE_F32) == 0


def test_c_scores():
    L = _lib.load()
    f = lambda **k: L.dsa_paged_index_scores(*({**dict(q=P, w=P, c=P, t=P, qs=P, kv=P, s=P, lim=None, T=5, R=3, W=4, first=0, n=5, L=64, H=16, D=128,  # noqa: E731
                                                       nb=2, bs=16, dt=DTYPE_MXFP8, wd=DTYPE_F32, relu=1, st=None), **k}).values())
    for k in (dict(T=-1), dict(R=-1), dict(W=0), dict(H=0), dict(L=-1), dict(L=65), dict(first=-1), dict(n=-1), dict(first=1), dict(R=1 << 20), dict(T=1 << 30, n=0),
              dict(W=1 << 27), dict(wd=DTYPE_E4M3), dict(dt=DTYPE_F32), dict(bs=10), dict(qs=None), dict(q=None), dict(w=None), dict(c=P + 8), dict(q=P + 2),
              dict(t=None), dict(kv=None), dict(s=None)):
        assert f(**k) == INVALID, k
    for k in (dict(H=8), dict(H=128), dict(D=32)):
        assert f(**k) == UNSUPPORTED, k
    assert f(n=0, q=None) == f(T=0, n=0) == f(L=0, s=None) == OK


def test_c_sparse():
    L = _lib.load()
    f = lambda **k: L.dsa_paged_sparse_mla_fwd(*({**dict(q=P, c=P, i=P, t=P, qs=P, kv=P, o=P, l=P, ws=P, n=0, T=5, R=3, W=4, H=16, k=8, D=128, V=64, nb=2,  # noqa: E731
                                                         bs=16, dt=DTYPE_MXFP4, scale=0.1, st=None), **k}).values())
    for k in (dict(T=-1), dict(R=-1), dict(W=0), dict(H=0), dict(H=8192), dict(k=0), dict(k=1 << 31), dict(T=1 << 29), dict(R=1 << 20), dict(W=1 << 28),
              dict(nb=1 << 28), dict(qs=None), dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e-38), dict(i=None), dict(t=None), dict(kv=None), dict(l=None),
              dict(q=P + 2), dict(c=P + 8), dict(o=P + 8), dict(dt=DTYPE_MXFP8), dict(T=1 << 20, k=1 << 30)):
        assert f(**k) == INVALID, k
    assert f(D=192, V=128) == UNSUPPORTED
    size = L.dsa_paged_sparse_mla_workspace_size
    for D, V in ((128, 64), (576, 512)):
        a = dict(T=5, H=16, k=2048, D=D, V=V)
        need = size(5, 16, 2048, D, V)
        assert need > 0 and f(**a, n=need - 1) == f(**a, ws=None, n=need) == f(**a, ws=P + 16, n=need) == WORKSPACE
    assert f(T=0, R=0, q=None) == f(T=3, R=0, qs=P, q=None) == OK and size(0, 16, 8, 128, 64) == 0
    assert size(5, 16, 8, 192, 128) == size(5, 0, 8, 128, 64) == size(5, 16, 0, 128, 64) == 0


def test_c_calls_too_large_for_their_numbering():
    L = _lib.load()
    keys = lambda T: L.dsa_index_key_append(P, P, 64, P, T, 2, 16, 64, DTYPE_BF16, None)  # noqa: E731
    assert keys(1 << 28) == INVALID
    size = L.dsa_paged_sparse_mla_workspace_size
    assert size(5, 16, 1 << 27, 128, 64) > 0 and size(5, 16, 1 << 27, 576, 512) > 0
    for D, V in ((128, 64), (576, 512)):
        for T, H, topk in ((5, 16, (1 << 27) + 1), (1 << 26, 1, 8), (1 << 19, 4095, 8)):
            assert size(T, H, topk, D, V) == 0
            assert L.dsa_paged_sparse_mla_fwd(P, P, P, P, P, P, P, P, P, 1 << 60, T, 3, 4, H, topk, D, V, 2, 16, DTYPE_BF16, 0.1, None) == INVALID
    assert size(1 << 20, 64, 1 << 18, 576, 512) == 0                # blocks of picks past 2^31


def test_c_the_last_call_of_a_grid():
    """A grid's axis has fewer than 2^32 threads, its last workgroup's among them.  Admitted calls end at a later check."""
    L = _lib.load()
    why = lambda: L.dsa_last_error().decode()  # noqa: E731
    for D, most in ((128, (1 << 28) - 16), (64, (1 << 28) - 1)):
        for f, a in ((L.dsa_index_key_append, (P, None, 128, P)), (L.dsa_index_key_gather, (P, P, None))):
            assert f(*a, most, 2, 16, D, DTYPE_BF16, None) == INVALID and "pointer" in why()
            assert f(*a, most + 1, 2, 16, D, DTYPE_BF16, None) == INVALID and "T=" in why()
    sparse = lambda T, H, D, V: L.dsa_paged_sparse_mla_fwd(P, P, P, P, P, P, P, P, P, 1 << 60, T, 0, 4, H, 8, D, V, 2, 16, DTYPE_BF16, 0.1, None)  # noqa: E731
    for D, V, most in ((128, 64, (1 << 26) - 4), (576, 512, (1 << 26) - 1)):
        assert sparse(most, 1, D, V) == sparse(most // 2, 33, D, V) == OK                    # (no requests: nothing to do)
        assert sparse(most + 1, 1, D, V) == sparse(most // 2 + 1, 33, D, V) == INVALID and "out of range" in why()


def test_c_workspace_of_whole_units():
    """No workspace where no unit is cut: it would be two 32-bit pieces a workgroup that nobody writes."""
    L = _lib.load()
    size = lambda T, H, topk: L.dsa_paged_sparse_mla_workspace_size(T, H, topk, 576, 512)  # noqa: E731
    for whole in ((1537, 128, 64), (64, 128, 2048), (160, 16, 64), (1, 16, 64), (256, 16, 2048)):
        assert size(*whole) == 0, whole
    for cut in ((96, 16, 2048), (1, 128, 2048), (400, 16, 2048), (257, 64, 640)):            # (the last: MXFP4's)
        assert size(*cut) > 0, cut
    assert L.dsa_paged_sparse_mla_fwd(P, P, P, P, P, P, P, P, None, 0, 160, 0, 4, 16, 64, 576, 512, 2, 16, DTYPE_BF16, 0.1, None) == OK


def test_c_layer_norm():
    L = _lib.load()
    fwd = lambda **k: L.dsa_layer_norm_fwd(*({**dict(x=P, w=P, b=P, y=P, m=P, r=P, rows=4, n=64, xs=64, eps=1e-5, dt=DTYPE_BF16, wd=DTYPE_F32,  # noqa: E731
                                                     st=None), **k}).values())
    bwd = lambda **k: L.dsa_layer_norm_bwd(*({**dict(dy=P, x=P, w=P, m=P, r=P, dx=P, dw=P, db=P, ws=P, nws=0, rows=400, n=1000, dys=1000, xs=1000,  # noqa: E731
                                                     dt=DTYPE_BF16, wd=DTYPE_F32, st=None), **k}).values())
    for f in (fwd, bwd):
        for k in (dict(rows=-1), dict(rows=1 << 31), dict(n=0), dict(dt=DTYPE_E4M3), dict(wd=DTYPE_MXFP4), dict(xs=-1), dict(x=None), dict(x=P + 1), dict(w=P + 2),
                  dict(dt=DTYPE_F32, x=P + 2)):
            assert f(**k) == INVALID, k
        assert f(n=16385) == UNSUPPORTED
    for k in (dict(y=None), dict(m=None), dict(eps=-1.0), dict(eps=float("nan")), dict(y=P + 1)):
        assert fwd(**k) == INVALID, k
    assert fwd(rows=0, x=None) == OK
    for k in (dict(dy=None), dict(m=None), dict(r=None), dict(dys=-1), dict(dx=P + 1), dict(dw=P + 2)):
        assert bwd(**k) == INVALID, k
    need = L.dsa_layer_norm_bwd_workspace_size(400, 1000)
    assert need > 0 and bwd(nws=need - 1) == bwd(ws=None, nws=need) == bwd(ws=P + 2, nws=need) == WORKSPACE
    assert L.dsa_layer_norm_bwd_workspace_size(1, 64) == L.dsa_layer_norm_bwd_workspace_size(-1, 64) == 0
    assert bwd(dx=None, dw=None, db=None, ws=None) == OK
