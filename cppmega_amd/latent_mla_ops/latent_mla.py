"""Dense latent attention, forward and backward (bf16, gfx950 HIP kernels).

The dense counterpart of ``sparse_mla_ops.SparseMLA``: every key of a row's window
instead of a top-k of them, as the DSA warm-up (which trains the indexer against dense
attention) and layers without an indexer need it.

  absorbed   ``LatentMLA``          q [B, S, H, d_qk], kv [B, S_kv, G, d_qk]; V is the first d_v channels of kv
             (d_qk, d_v) in {(128, 64), (128, 128), (192, 128)}
  expanded   ``LatentMLAExpanded``  q [B, S, H, d_nope + 64], k_nope [B, S_kv, H, d_nope], k_pe [B, S_kv, 64] of every
             head, v [B, S_kv, H, d_v]; (d_nope, d_v) in {(128, 128), (64, 64)}
  returns    (out [B, S, H, d_v] bf16, lse [B, S, H] f32, log2 units)

The default scale is (width of q)^-0.5: the two forms of one layer have different widths,
so the absorbed form of a layer trained expanded takes the expanded form's scale.

3-D q / kv without the batch are accepted as SparseMLA accepts them.  Masks: ``causal``
(query token t sees the keys up to position t + S_kv - S: the last S of S_kv tokens),
every key (``causal=False``), or per-row key windows ``starts`` / ``ends`` [B, S] int32
(keys [start, end), clipped to [0, S_kv): packed documents, padding, sliding windows),
which take causal's place.  A row without keys, or whose every score is -Inf, has out 0,
lse -inf and zero gradients; scores below -2^31 (log2 units) count as -Inf.
Keys that a row does not see may hold anything, Inf and NaN too.  The gradient of lse is
not taken, as SparseMLA does not take it.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ..sparse_mla_ops._common import normalize_sm_scale, unwrap_quantized
from ._common import dense, launch_on, same_device

_STRIDES = ctypes.c_int64 * 8


def _scale(sm_scale, d_qk):
    scale = normalize_sm_scale(sm_scale, d_qk)
    if not 2.0 ** -100 <= scale < float("inf"):
        raise ValueError(f"sm_scale must be finite and at least 2^-100, got {scale}")
    return scale


def _mask(causal, starts, ends, B, S):
    """-> causal flag; row windows checked."""
    assert (starts is None) == (ends is None), "starts and ends come together"
    if starts is None:
        return 1 if causal is None or causal else 0
    assert not causal, "starts / ends carry the mask: leave causal unset with them"
    for x in (starts, ends):
        assert x.dtype == torch.int32 and tuple(x.shape) == (B, S) and x.is_contiguous(), \
            f"starts / ends must be contiguous int32 [{B}, {S}], got {x.dtype} {tuple(x.shape)}"
    return 0


def _check_bf16(**ts):
    for name, t in ts.items():
        assert t.dtype == torch.bfloat16, f"{name} must be bfloat16, got {t.dtype}"


def _check_dense(**ts):
    for name, t in ts.items():
        assert t.is_contiguous(), f"{name} must be contiguous"
        assert t.data_ptr() % 16 == 0, f"{name} must be 16-byte aligned"


def _check_residual(residual, o):
    if residual is not None:
        assert residual.shape == o.shape, f"residual must be of out's shape {tuple(o.shape)}, got {tuple(residual.shape)}"
        _check_bf16(residual=residual)
        _check_dense(residual=residual)


def _batched(*ts):
    """3-D tensors as a batch of one."""
    return tuple(t.unsqueeze(0) for t in ts)


def _absorbed_dims(q, kv, d_v):
    assert q.ndim == 4 and kv.ndim == 4, f"q and kv must be 3-D or 4-D, got {tuple(q.shape)}, {tuple(kv.shape)}"
    B, S, H, D = q.shape
    _, S_kv, G, kv_dim = kv.shape
    assert kv.shape[0] == B, f"batch of q ({B}) and kv ({kv.shape[0]}) differ"
    assert kv_dim == D, "q and kv must have the same embedding dimension on the last axis"
    assert 0 < d_v <= D, f"d_v must be in (0, {D}], but got {d_v}"
    assert G > 0 and H % G == 0, f"heads={H} must be a multiple of kv_group={G}"
    return B, S, S_kv, H, G, D


def latent_mla_fwd_interface(q, kv, sm_scale=None, d_v=None, causal=None, starts=None, ends=None, residual=False):
    """Absorbed forward: (out, lse), with ``residual`` (out, lse, what rounding took from out, for the backward).
    Arguments as in the module's description; d_v: all channels where it is not given."""
    q, kv = unwrap_quantized(q), unwrap_quantized(kv)
    d_v = q.shape[-1] if d_v is None else d_v
    squeeze = q.ndim == 3
    if squeeze:
        q, kv = _batched(q, kv)
        starts, ends = (x if x is None or x.ndim == 2 else x.unsqueeze(0) for x in (starts, ends))
    B, S, S_kv, H, G, D = _absorbed_dims(q, kv, d_v)
    _check_bf16(q=q, kv=kv)
    _check_dense(q=q, kv=kv)
    same_device(q, kv, starts, ends)
    flag = _mask(causal, starts, ends, B, S)
    scale = _scale(sm_scale, D)
    stream, here = launch_on(q)
    with here:
        out = torch.empty((B, S, H, d_v), dtype=torch.bfloat16, device=q.device)
        lse = torch.empty((B, S, H), dtype=torch.float32, device=q.device)
        low = torch.empty_like(out) if residual else None
        rc = _lib.load().dsa_latent_mla_fwd(q.data_ptr(), kv.data_ptr(), _lib.ptr(starts), _lib.ptr(ends), out.data_ptr(),
                                            _lib.ptr(low), lse.data_ptr(), B, S, S_kv, H, G, D, d_v, scale, flag, stream)
    _lib.check(rc, "dsa_latent_mla_fwd")
    got = (out, lse, low) if residual else (out, lse)
    return tuple(t[0] for t in got) if squeeze else got


def latent_mla_bwd(q, kv, o, do, lse, sm_scale=None, causal=None, starts=None, ends=None, residual=None):
    """Absorbed backward: (dq, dkv) bf16, from the forward's out, lse and (for rows of few keys more exactly)
    residual.  Deterministic: repeated calls give the same bits."""
    q, kv, o, do = unwrap_quantized(q), unwrap_quantized(kv), unwrap_quantized(o), unwrap_quantized(do)
    squeeze = q.ndim == 3
    if squeeze:
        q, kv, o, do, lse = _batched(q, kv, o, do, lse)
        residual = None if residual is None else residual.unsqueeze(0)
        starts, ends = (x if x is None or x.ndim == 2 else x.unsqueeze(0) for x in (starts, ends))
    d_v = o.shape[-1]
    B, S, S_kv, H, G, D = _absorbed_dims(q, kv, d_v)
    assert tuple(o.shape) == (B, S, H, d_v) and tuple(do.shape) == (B, S, H, d_v) and tuple(lse.shape) == (B, S, H)
    _check_bf16(q=q, kv=kv, o=o, do=do)
    assert lse.dtype == torch.float32
    _check_dense(q=q, kv=kv, o=o, do=do, lse=lse)
    _check_residual(residual, o)
    same_device(q, kv, o, do, lse, starts, ends, residual)
    flag = _mask(causal, starts, ends, B, S)
    scale = _scale(sm_scale, D)
    stream, here = launch_on(q)
    L = _lib.load()
    with here:
        dq, dkv = torch.empty_like(q), torch.empty_like(kv)
        n = int(L.dsa_latent_mla_bwd_workspace_size(B, S, S_kv, H, G, D, d_v, 0))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        rc = L.dsa_latent_mla_bwd(q.data_ptr(), kv.data_ptr(), o.data_ptr(), _lib.ptr(residual), do.data_ptr(), lse.data_ptr(),
                                  _lib.ptr(starts), _lib.ptr(ends), dq.data_ptr(), dkv.data_ptr(), ws.data_ptr(), n, B, S, S_kv, H, G, D, d_v,
                                  scale, flag, stream)
    _lib.check(rc, "dsa_latent_mla_bwd")
    return (dq[0], dkv[0]) if squeeze else (dq, dkv)


def _rows(t):
    """``t`` as the kernels read keys and values: the last axis dense, strides of whole 16 bytes (views of one
    up-projection are taken as they are), else a contiguous copy."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(0 <= s < 1 << 23 and s % 8 == 0 for s in t.stride()[1:-1]) \
        and t.stride(0) % 8 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _expanded_args(q, k_nope, k_pe, v):
    assert q.ndim == 4 and k_nope.ndim == 4 and k_pe.ndim == 3 and v.ndim == 4, \
        "q, k_nope and v must be 4-D [batch, seq, heads, dim], k_pe 3-D [batch, seq, dim]"
    B, S, H, D = q.shape
    S_kv, dn, dr, dv = k_nope.shape[1], k_nope.shape[3], k_pe.shape[2], v.shape[3]
    assert tuple(k_nope.shape) == (B, S_kv, H, dn) and tuple(v.shape) == (B, S_kv, H, dv) and tuple(k_pe.shape) == (B, S_kv, dr), \
        f"k_nope {tuple(k_nope.shape)}, k_pe {tuple(k_pe.shape)} and v {tuple(v.shape)} do not belong to q {tuple(q.shape)}"
    assert dn + dr == D, f"q has {D} channels, k_nope and k_pe {dn} + {dr}"
    _check_bf16(q=q, k_nope=k_nope, k_pe=k_pe, v=v)
    _check_dense(q=q)
    strides = _STRIDES(*k_nope.stride()[:3], *k_pe.stride()[:2], *v.stride()[:3])
    return B, S, S_kv, H, dn, dr, dv, strides


def latent_mla_expanded_fwd(q, k_nope, k_pe, v, sm_scale=None, causal=None, starts=None, ends=None, residual=False):
    """Expanded forward: (out, lse), with ``residual`` a third as the absorbed form.  k_nope, k_pe and v may be strided views (last axis dense)."""
    k_nope, k_pe, v = _rows(k_nope), _rows(k_pe), _rows(v)
    B, S, S_kv, H, dn, dr, dv, strides = _expanded_args(q, k_nope, k_pe, v)
    same_device(q, k_nope, k_pe, v, starts, ends)
    flag = _mask(causal, starts, ends, B, S)
    scale = _scale(sm_scale, dn + dr)
    stream, here = launch_on(q)
    with here:
        out = torch.empty((B, S, H, dv), dtype=torch.bfloat16, device=q.device)
        lse = torch.empty((B, S, H), dtype=torch.float32, device=q.device)
        low = torch.empty_like(out) if residual else None
        rc = _lib.load().dsa_latent_mla_expanded_fwd(
            q.data_ptr(), k_nope.data_ptr(), k_pe.data_ptr(), v.data_ptr(), _lib.ptr(starts), _lib.ptr(ends), out.data_ptr(),
            _lib.ptr(low), lse.data_ptr(), B, S, S_kv, H, dn, dr, dv, strides, scale, flag, stream)
    _lib.check(rc, "dsa_latent_mla_expanded_fwd")
    return (out, lse, low) if residual else (out, lse)


def latent_mla_expanded_bwd(q, k_nope, k_pe, v, o, do, lse, sm_scale=None, causal=None, starts=None, ends=None, residual=None):
    """Expanded backward: (dq, dk_nope, dk_pe, dv) bf16, dk_pe summed over the heads.  Deterministic."""
    k_nope, k_pe, v = _rows(k_nope), _rows(k_pe), _rows(v)
    B, S, S_kv, H, dn, dr, dv, strides = _expanded_args(q, k_nope, k_pe, v)
    assert tuple(o.shape) == (B, S, H, dv) and tuple(do.shape) == (B, S, H, dv) and tuple(lse.shape) == (B, S, H)
    _check_bf16(o=o, do=do)
    assert lse.dtype == torch.float32
    _check_dense(o=o, do=do, lse=lse)
    _check_residual(residual, o)
    same_device(q, k_nope, k_pe, v, o, do, lse, starts, ends, residual)
    flag = _mask(causal, starts, ends, B, S)
    scale = _scale(sm_scale, dn + dr)
    stream, here = launch_on(q)
    L = _lib.load()
    with here:
        dq = torch.empty_like(q)
        dk_nope, dk_pe, dvv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (k_nope, k_pe, v))
        n = int(L.dsa_latent_mla_bwd_workspace_size(B, S, S_kv, H, H, dn + dr, dv, 1))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        rc = L.dsa_latent_mla_expanded_bwd(
            q.data_ptr(), k_nope.data_ptr(), k_pe.data_ptr(), v.data_ptr(), o.data_ptr(), _lib.ptr(residual), do.data_ptr(),
            lse.data_ptr(), _lib.ptr(starts), _lib.ptr(ends), dq.data_ptr(), dk_nope.data_ptr(), dk_pe.data_ptr(), dvv.data_ptr(),
            ws.data_ptr(), n, B, S, S_kv, H, dn, dr, dv, strides, scale, flag, stream)
    _lib.check(rc, "dsa_latent_mla_expanded_bwd")
    return dq, dk_nope, dk_pe, dvv


class LatentMLA(torch.autograd.Function):
    """Dense attention over packed latent KV (bf16): ``apply(q, kv, scaling, d_v, causal, starts, ends)``."""

    @staticmethod
    def forward(ctx, q, kv, scaling=None, d_v=None, causal=None, starts=None, ends=None):
        q, kv = dense(unwrap_quantized(q)), dense(unwrap_quantized(kv))
        ctx.args = dict(sm_scale=scaling, causal=causal)
        out, lse, *low = latent_mla_fwd_interface(q, kv, d_v=d_v, starts=starts, ends=ends, residual=any(ctx.needs_input_grad),
                                                  **ctx.args)
        ctx.save_for_backward(q, kv, out, lse, starts, ends, *low)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_lse):
        if grad_output is None:
            return (None,) * 7
        q, kv, out, lse, starts, ends, low = ctx.saved_tensors
        dq, dkv = latent_mla_bwd(q, kv, out, dense(grad_output), lse, starts=starts, ends=ends, residual=low, **ctx.args)
        return dq, dkv, None, None, None, None, None


class LatentMLAExpanded(torch.autograd.Function):
    """Dense attention with the keys and values of every head and one shared rope part (bf16):
    ``apply(q, k_nope, k_pe, v, scaling, causal, starts, ends)``."""

    @staticmethod
    def forward(ctx, q, k_nope, k_pe, v, scaling=None, causal=None, starts=None, ends=None):
        q = dense(q)
        ctx.args = dict(sm_scale=scaling, causal=causal)
        out, lse, *low = latent_mla_expanded_fwd(q, k_nope, k_pe, v, starts=starts, ends=ends, residual=any(ctx.needs_input_grad),
                                                 **ctx.args)
        ctx.save_for_backward(q, k_nope, k_pe, v, out, lse, starts, ends, *low)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_lse):
        if grad_output is None:
            return (None,) * 8
        q, k_nope, k_pe, v, out, lse, starts, ends, low = ctx.saved_tensors
        grads = latent_mla_expanded_bwd(q, k_nope, k_pe, v, out, dense(grad_output), lse, starts=starts, ends=ends, residual=low,
                                        **ctx.args)
        return (*grads, None, None, None, None)
