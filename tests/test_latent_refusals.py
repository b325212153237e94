"""What the latent attention, cache and plan entry points refuse, on the CPU: every check comes before the device's."""
import ctypes

import pytest
import torch

from cppmega_amd import _lib
from cppmega_amd import latent_mla_ops as ops
from cppmega_amd._lib import DTYPE_BF16, DTYPE_MXFP4
from oracle import latent_cache as oc
from oracle import latent_mla as om

BF = torch.bfloat16
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, -1, -2, -4


def _t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _i32(*shape):
    return _t(*shape, dtype=torch.int32)


def _refused(error, f, *args, **kw):
    with pytest.raises(error):
        f(*args, **kw)


def test_dense_arguments():
    q, kv = _t(1, 4, 2, 128), _t(1, 4, 1, 128)
    fwd = ops.latent_mla_fwd_interface
    for a, k in (
        ((_t(4, 128), kv), {}),                                        # q's axes
        ((q, _t(2, 4, 1, 128)), {}),                                   # batches
        ((q, _t(1, 4, 1, 192)), {}),                                   # channels
        ((_t(1, 4, 3, 128), _t(1, 4, 2, 128)), {}),                    # heads over groups
        ((q, kv), dict(d_v=129)), ((q, kv), dict(d_v=0)),
        ((q.half(), kv), {}), ((q, kv.float()), {}),
        ((_t(1, 2, 4, 128).transpose(1, 2), kv), {}),
        ((_t(1 * 4 * 2 * 128 + 1)[1:].view(1, 4, 2, 128), kv), {}),    # 2 bytes past 16
        ((q, kv), dict(starts=_i32(1, 4))), ((q, kv), dict(starts=_i32(1, 4), ends=_i32(1, 3))),
        ((q, kv), dict(starts=_i32(1, 4), ends=_t(1, 4, dtype=torch.int64))),
        ((q, kv), dict(starts=_i32(1, 4), ends=_i32(1, 4), causal=True)),
    ):
        _refused(AssertionError, fwd, *a, **({"d_v": 64} | k))
    for scale in (0.0, -1.0, 1e-38, float("inf"), float("nan")):
        _refused(ValueError, fwd, q, kv, scale, 64)
    _refused(RuntimeError, fwd, q, kv, None, 64)                       # no GPU tensor
    out, lse = _t(1, 4, 2, 64), _t(1, 4, 2, dtype=torch.float32)
    _refused(AssertionError, ops.latent_mla_bwd, q, kv, out, out, lse, residual=out[:, :2])
    _refused(AssertionError, ops.latent_mla_bwd, q, kv, out, out, lse, residual=out.float())
    for a in ((q, kv, _t(1, 4, 2, 128)[..., :64], out, lse), (q, kv, out, _t(1, 3, 2, 64), lse), (q, kv, out, out, lse.double()),
              (q, kv, out, out.float(), lse), (q, kv, out, out, lse[:, :3])):
        _refused(AssertionError, ops.latent_mla_bwd, *a)


def test_default_value_channels():
    """Without d_v a row is its own value, in the functional form as in LatentMLA: no check before the device's refuses it."""
    q, kv = _t(1, 4, 2, 128), _t(1, 4, 1, 128)
    _refused(RuntimeError, ops.latent_mla_fwd_interface, q, kv)
    _refused(RuntimeError, ops.latent_mla_fwd_interface, q[0], kv[0])
    _refused(RuntimeError, ops.LatentMLA.apply, q, kv)


def test_expanded_arguments():
    q, kn, pe, v = _t(1, 4, 2, 192), _t(1, 4, 2, 128), _t(1, 4, 64), _t(1, 4, 2, 128)
    f = ops.latent_mla_expanded_fwd
    for a in ((q[0], kn, pe, v), (q, _t(1, 4, 1, 128), pe, v), (q, kn, _t(1, 5, 64), v), (q, kn, _t(1, 4, 32), v),
              (q, kn, pe, _t(1, 4, 3, 128)), (q, kn, pe[0], v), (q, kn, pe, v.half()), (q.transpose(1, 2), kn, pe, v)):
        _refused(AssertionError, f, *a)
    _refused(AssertionError, f, q, kn, pe, v, causal=True, starts=_i32(1, 4), ends=_i32(1, 4))
    _refused(ValueError, f, q, kn, pe, v, -0.5)
    _refused(RuntimeError, f, q, kn, pe, v)
    out, lse = _t(1, 4, 2, 128), _t(1, 4, 2, dtype=torch.float32)
    _refused(AssertionError, ops.latent_mla_expanded_bwd, q, kn, pe, v, out, out[:, :2], lse)
    _refused(AssertionError, ops.latent_mla_expanded_bwd, q, kn, pe, v, out, out, lse.double())


def test_cache_arguments():
    for data, dims in ((_t(2, 16, 128), (576, 512)), (_t(2, 16, 576, dtype=torch.float16), (576, 512)),
                       (_t(2, 16, 192), (192, 128)), (_t(2, 16 * 576), (576, 512)), (_t(0, 16, 576), (576, 512)),
                       (_t(2, 16, 577)[..., :576], (576, 512)), (_t(2, 16, 399, dtype=torch.uint8), (576, 512)),
                       (_t(1, 65537, 128), (128, 64))):
        _refused(AssertionError, ops.LatentCache, data, *dims)
    _refused(AssertionError, ops.LatentCache.empty, 2, 16, 576, 512, "fp8", "cpu")
    _refused(AssertionError, ops.latent_cache_row_bytes, 576, 512, "fp8")
    assert ops.latent_cache_row_bytes(576, 512, "mxfp4") == oc.row_bytes(576, 512) == 400
    assert ops.latent_cache_row_bytes(128, 64, "mxfp4") == oc.row_bytes(128, 64) == 176
    c = ops.LatentCache(_t(2, 16, 128), 128, 64)
    slots = _t(3, dtype=torch.int64)
    add = ops.latent_cache_append
    for a in ((_t(3, 63), _t(3, 64), slots), (_t(3, 64), _t(2, 64), slots), (_t(3, 64), _t(3, 64), slots[:2]),
              (_t(3, 64), _t(3, 64), slots.int()), (_t(3, 64).half(), _t(3, 64), slots), (_t(3, 64), _t(3, 1, 64), slots)):
        _refused(AssertionError, add, c, *a)
    _refused(RuntimeError, add, c, _t(3, 64), _t(3, 64), slots)
    _refused(AssertionError, ops.latent_cache_gather, c, slots.int())
    _refused(AssertionError, ops.latent_cache_gather, c, _t(6, dtype=torch.int64)[::2])


def test_paged_arguments():
    c = ops.LatentCache(_t(2, 16, 128), 128, 64)
    q, table, kv = _t(3, 2, 128), _i32(3, 4), _i32(3)
    f = ops.paged_latent_mla_fwd
    for a, k in (((q[0], c, table, kv), {}), ((_t(3, 2, 192), c, table, kv), {}), ((q.half(), c, table, kv), {}),
                 ((q, c, table[:2], kv), {}), ((q, c, table.long(), kv), {}), ((q, c, table, kv.long()), {}),
                 ((q, c, _i32(3, 8)[:, ::2], kv), {}), ((q, c, _i32(3, 0), kv), {}), ((_t(4, 2, 128), c, table, kv), {}),
                 ((q, c, table, kv), dict(query_starts=_i32(3))), ((q, c, table, kv), dict(query_starts=_t(4)))):
        _refused(AssertionError, f, *a, **k)
    _refused(ValueError, f, q, c, table, kv, sm_scale=0.0)
    _refused(RuntimeError, f, q, c, table, kv)


def test_plan_arguments():
    a = dict(context_lens=_i32(3), query_lens=_i32(3), block_table=_i32(3, 4), free_blocks=_i32(5), free_count=_i32(1), num_tokens=3,
             block_size=16)
    for bad in (dict(context_lens=_i32(3).long()), dict(query_lens=_i32(4)), dict(block_table=_i32(2, 4)), dict(block_table=_i32(3, 0)),
                dict(free_count=_i32(2)), dict(free_blocks=_i32(0)), dict(num_tokens=-1), dict(block_size=0),
                dict(free_blocks=_i32(10)[::2])):
        _refused(AssertionError, ops.plan_latent_step, **(a | bad))
    _refused(RuntimeError, ops.plan_latent_step, **a)


# ---------------------------------------------------------------- the C entry points (nothing is launched)

P = 1 << 20  # a pointer that is aligned and never read: each call ends at its check


def test_c_dense():
    L = _lib.load()
    fwd = lambda **k: L.dsa_latent_mla_fwd(*({**dict(q=P, kv=P, s=None, e=None, o=P, lo=None, l=P, B=1, S=4, Sk=4, H=2, G=1, D=128, V=64, scale=0.1,  # noqa: E731
                                                     causal=1, st=None), **k}).values())
    for k in (dict(B=-1), dict(S=-1), dict(H=0), dict(G=3), dict(H=8192), dict(S=1 << 30), dict(Sk=1 << 30), dict(scale=0.0),
              dict(scale=1e-38), dict(scale=float("nan")), dict(causal=2), dict(s=P), dict(s=P, e=P), dict(q=None), dict(kv=P + 2), dict(o=P + 8),
              dict(l=None), dict(lo=P + 2), dict(S=1 << 29, H=4096)):
        assert fwd(**k) == INVALID, k
    for k in (dict(D=576, V=512), dict(D=192, V=64), dict(V=32)):
        assert fwd(**k) == UNSUPPORTED, k
    assert fwd(B=0, q=None) == OK and fwd(S=0, q=None, o=None, l=None) == OK
    st = (ctypes.c_int64 * 8)(1024, 256, 128, 256, 64, 1024, 256, 128)
    ex = lambda **k: L.dsa_latent_mla_expanded_fwd(*({**dict(q=P, kn=P, pe=P, v=P, s=None, e=None, o=P, lo=None, l=P, B=1, S=4, Sk=4, H=2, dn=128,  # noqa: E731
                                                             dr=64, V=128, strides=st, scale=0.1, causal=1, stream=None), **k}).values())
    for k in (dict(strides=None), dict(strides=(ctypes.c_int64 * 8)(4, *st[1:])), dict(strides=(ctypes.c_int64 * 8)(*st[:4], -8, *st[5:])),
              dict(strides=(ctypes.c_int64 * 8)(st[0], 1 << 23, *st[2:])), dict(pe=P + 8), dict(v=None), dict(q=None)):
        assert ex(**k) == INVALID, k
    assert ex(dr=32) == UNSUPPORTED and ex(dn=64, V=128) == UNSUPPORTED
    size = L.dsa_latent_mla_bwd_workspace_size
    assert size(1, 4, 4, 2, 1, 128, 64, 0) > 0 and size(1, 4, 4, 2, 1, 576, 512, 0) == 0 and size(1, 4, 4, 2, 3, 128, 64, 0) == 0
    n = size(1, 4, 4, 2, 1, 128, 64, 0)
    bwd = lambda **k: L.dsa_latent_mla_bwd(*({**dict(q=P, kv=P, o=P, lo=None, do=P, l=P, s=None, e=None, dq=P, dkv=P, ws=P, n=n, B=1, S=4, Sk=4, H=2,  # noqa: E731
                                                     G=1, D=128, V=64, scale=0.1, causal=1, st=None), **k}).values())
    assert bwd(ws=None) == WORKSPACE and bwd(n=n - 1) == WORKSPACE and bwd(ws=P + 16) == WORKSPACE
    for k in (dict(dq=None), dict(dkv=None), dict(do=P + 2), dict(lo=P + 8), dict(l=None), dict(scale=-1.0)):
        assert bwd(**k) == INVALID, k


def test_c_cache():
    L = _lib.load()
    assert L.dsa_latent_cache_row_bytes(576, 512, DTYPE_MXFP4) == 400 and L.dsa_latent_cache_row_bytes(192, 128, DTYPE_BF16) == 0
    add = lambda **k: L.dsa_latent_cache_append(*({**dict(c=P, x=P, xs=64, r=P, rs=64, s=P, T=1, nb=2, bs=16, D=128, V=64, dt=DTYPE_BF16,  # noqa: E731
                                                          st=None), **k}).values())
    for k in (dict(T=-1), dict(nb=0), dict(bs=0), dict(bs=65537), dict(dt=0 if DTYPE_BF16 else 1), dict(xs=60), dict(rs=-8), dict(x=P + 2),
              dict(c=None), dict(s=None)):
        assert add(**k) == INVALID, k
    assert add(D=192, V=128) == UNSUPPORTED and add(T=0, x=None) == OK
    get = lambda **k: L.dsa_latent_cache_gather(*({**dict(c=P, s=P, o=P, T=1, nb=2, bs=16, D=128, V=64, dt=DTYPE_MXFP4, st=None), **k}).values())  # noqa: E731
    assert get(o=P + 2) == INVALID and get(nb=1 << 31) == INVALID and get(T=0) == OK
    size = L.dsa_paged_latent_mla_workspace_size
    assert size(4, 2, 8, 16, 4, 128, 64) > 0 and size(4, 2, 8, 16, 4, 192, 128) == 0 and size(0, 2, 8, 16, 4, 128, 64) == 0
    n = size(4, 2, 8, 16, 4, 128, 64)
    f = lambda **k: L.dsa_paged_latent_mla_fwd(*({**dict(q=P, c=P, t=P, qs=P, kv=P, o=P, l=P, ws=P, n=n, T=4, R=2, W=8, H=4, D=128, V=64, nb=9,  # noqa: E731
                                                         bs=16, dt=DTYPE_BF16, scale=0.1, st=None), **k}).values())
    assert f(n=n - 1) == WORKSPACE and f(ws=None) == WORKSPACE and f(ws=P + 64) == WORKSPACE
    for k in (dict(T=-1), dict(W=0), dict(H=0), dict(H=8192), dict(R=1 << 20), dict(W=(1 << 31) // 16), dict(T=1 << 30), dict(scale=0.0),
              dict(q=None), dict(kv=None), dict(o=P + 8), dict(dt=3),
              dict(T=1 << 18, R=1 << 18, W=1 << 20)):                  # row groups times key blocks pass 32 bits
        assert f(**k) == INVALID, k
    assert f(T=0, q=None) == OK and f(R=0, kv=None) == OK


def test_c_cache_rows_past_a_grid():
    """A grid's axis has fewer than 2^32 threads."""
    L = _lib.load()
    for D, V, T in ((128, 64, (1 << 28) - 15), (576, 512, 59652321), (576, 512, (1 << 31) - 1)):
        for dt in (DTYPE_BF16, DTYPE_MXFP4):
            assert L.dsa_latent_cache_append(P, P, V, P, 64, P, T, 2, 16, D, V, dt, None) == INVALID
            assert L.dsa_latent_cache_gather(P, P, P, T, 2, 16, D, V, dt, None) == INVALID


def test_c_plan():
    L = _lib.load()
    names = "ctx new table free count t_out slots pos starts kv ctx_out granted f_out c_out".split()
    base = {n: P + 4096 * i for i, n in enumerate(names)} | dict(R=2, W=4, F=8, T=3, bs=16, st=None)
    f = lambda **k: L.dsa_latent_plan_step(*{**base, **k}.values())  # noqa: E731
    for k in (dict(R=-1), dict(W=0), dict(F=0), dict(bs=0), dict(bs=65537), dict(R=1 << 20), dict(W=1 << 30), dict(ctx=None), dict(c_out=None),
              dict(slots=None)):
        assert f(**k) == INVALID, k
    for i in names[:5]:
        for o in names[5:]:
            assert f(**{o: base[i]}) == INVALID, (i, o)


# ---------------------------------------------------------------- the oracle itself


def test_oracle_plan_keeps_pages_behind_a_context():
    """Context 15, four drafts, one kept: the page that the drafts took serves position 16, and a finished request gives it back."""
    one = oc.plan([15], [4], [[3, -1, -1]], [5, 6, 7, -1], 3, 4, 16)
    assert one["block_table"] == [[3, 7, -1]] and one["free_count"] == [2]
    two = oc.plan([16], [1], one["block_table"], one["free_blocks"], 2, 1, 16)
    assert two["block_table"] == [[3, 7, -1]] and two["slots"] == [7 * 16] and two["free_blocks"] == [5, 6, -1, -1]
    end = oc.plan([15], [-1], two["block_table"], two["free_blocks"], 2, 0, 16)
    assert end["free_blocks"] == [5, 6, 3, 7] and end["free_count"] == [4]



def test_oracle_gradients_are_differences():
    """The formulas of the oracle's gradients against central differences of its forward, in 64 bits."""
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, kv, do = r(1, 5, 4, 12), r(1, 7, 2, 12), r(1, 5, 4, 8)
    lo, hi = om.windows(1, 5, 7)
    g = om.absorbed(q, kv, 8, 0.3, lo, hi, do)
    f = lambda q, kv: (om.absorbed(q, kv, 8, 0.3, lo, hi)["out"] * do).sum()  # noqa: E731
    dq, dk = r(*q.shape), r(*kv.shape)
    h = 1e-5
    num = (f(q + h * dq, kv + h * dk) - f(q - h * dq, kv - h * dk)) / (2 * h)
    assert abs(num - (g["dq"] * dq).sum() - (g["dkv"] * dk).sum()) < 1e-7 * (1 + abs(num))
    q, kn, pe, v, do = r(1, 5, 2, 12), r(1, 6, 2, 8), r(1, 6, 4), r(1, 6, 2, 8), r(1, 5, 2, 8)
    starts, ends = torch.tensor([[0, 1, 3, 2, 0]]), torch.tensor([[2, 5, 3, 6, 6]])
    lo, hi = om.windows(1, 5, 6, starts=starts, ends=ends)
    g = om.expanded(q, kn, pe, v, 0.3, lo, hi, do)
    x, d = (q, kn, pe, v), [r(*t.shape) for t in (q, kn, pe, v)]
    f = lambda s: (om.expanded(*(a + s * b for a, b in zip(x, d)), 0.3, lo, hi)["out"] * do).sum()  # noqa: E731
    num = (f(h) - f(-h)) / (2 * h)
    assert abs(num - sum((g[n] * b).sum() for n, b in zip(("dq", "dk_nope", "dk_pe", "dv"), d))) < 1e-7 * (1 + abs(num))
