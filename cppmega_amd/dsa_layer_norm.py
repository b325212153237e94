"""Layer norm, forward and backward (gfx950 HIP kernels): the norm of the indexer's keys in
front of their rotary part, the scores (``IndexScores``) and the paged cache, and of any
other rows of up to 16384 elements.

    y = (x - mean) rstd weight + bias,    rstd = (mean((x - mean)^2) + eps)^-1/2

x [..., n] bf16 or f32; weight and bias [n], bf16 or f32, or None (ones, zeros); statistics
and sums in 32 bits, gradients bit-identical between runs.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .latent_mla_ops._common import launch_on, same_device

__all__ = ["LayerNorm", "layer_norm", "layer_norm_backward"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


def _rows(t, n, name):
    """t [..., n] as rows with a dense last axis and one row stride: a view where there is one."""
    assert t.dtype in _DTYPES, f"{name} must be bfloat16 or float32, got {t.dtype}"
    t = t.reshape(-1, n) if t.ndim != 2 else t
    return t if (t.stride(1) == 1 or n == 1) and t.stride(0) >= 0 else t.contiguous()


def _check_params(weight, bias, n):
    """-> dtype code of the parameters."""
    for name, t in (("weight", weight), ("bias", bias)):
        assert t is None or (t.dtype in _DTYPES and tuple(t.shape) == (n,)), \
            f"{name} must be bfloat16 or float32 [{n}], got {t.dtype} {tuple(t.shape)}"
    assert weight is None or bias is None or weight.dtype == bias.dtype, f"weight is {weight.dtype}, bias {bias.dtype}"
    t = bias if weight is None else weight
    return _lib.DTYPE_F32 if t is None else _DTYPES[t.dtype]


def layer_norm(x, weight=None, bias=None, eps=1e-5, return_stats=False):
    """y of x's shape and type; with ``return_stats`` (y, mean, rstd), f32 of x's leading shape, for the backward."""
    assert x.ndim >= 1 and x.shape[-1] > 0, f"x must be [..., n], got {tuple(x.shape)}"
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    n = x.shape[-1]
    rows = _rows(x, n, "x")
    w_code = _check_params(weight, bias, n)
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    same_device(x, weight, bias)
    stream, here = launch_on(x)
    with here:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean = rstd = None
        if return_stats:
            mean, rstd = torch.empty((2, *x.shape[:-1]), dtype=torch.float32, device=x.device)
        rc = _lib.load().dsa_layer_norm_fwd(rows.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(), _lib.ptr(mean),
                                            _lib.ptr(rstd), rows.shape[0], n, rows.stride(0), eps, _DTYPES[x.dtype], w_code, stream)
    _lib.check(rc, "dsa_layer_norm_fwd")
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, weight, mean, rstd, need=(True, True, True), param_dtype=None):
    """(dx, dweight, dbias) for the upstream gradient dy of x's shape and type, from the forward's statistics; ``need``
    says which are wanted (None for the others), param_dtype the type of dweight and dbias (default: weight's, else f32)."""
    n = x.shape[-1]
    assert dy.shape == x.shape and dy.dtype == x.dtype, f"dy is {dy.dtype} {tuple(dy.shape)}, x {x.dtype} {tuple(x.shape)}"
    for name, t in (("mean", mean), ("rstd", rstd)):
        assert t.dtype == torch.float32 and t.shape == x.shape[:-1] and t.is_contiguous(), \
            f"{name} must be contiguous float32 {tuple(x.shape[:-1])}, got {t.dtype} {tuple(t.shape)}"
    _check_params(weight, None, n)
    if param_dtype is None:
        param_dtype = torch.float32 if weight is None else weight.dtype
    assert weight is None or weight.dtype == param_dtype, f"weight is {weight.dtype}, param_dtype {param_dtype}"
    rows, grad = _rows(x, n, "x"), _rows(dy, n, "dy")
    weight = None if weight is None else weight.contiguous()
    same_device(x, dy, weight, mean, rstd)
    stream, here = launch_on(x)
    L = _lib.load()
    with here:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dw, db = (torch.empty(n, dtype=param_dtype, device=x.device) if k else None for k in need[1:])
        ws_bytes = int(L.dsa_layer_norm_bwd_workspace_size(rows.shape[0], n)) if need[1] or need[2] else 0
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
        rc = L.dsa_layer_norm_bwd(grad.data_ptr(), rows.data_ptr(), _lib.ptr(weight), mean.data_ptr(), rstd.data_ptr(), _lib.ptr(dx),
                                  _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), ws_bytes, rows.shape[0], n, grad.stride(0),
                                  rows.stride(0), _DTYPES[x.dtype], _DTYPES[param_dtype], stream)
    _lib.check(rc, "dsa_layer_norm_bwd")
    return dx, dw, db


class LayerNorm(torch.autograd.Function):
    """apply(x, weight=None, bias=None, eps=1e-5) -> y, with gradients to x, weight and bias."""

    @staticmethod
    def forward(ctx, x, weight=None, bias=None, eps=1e-5):
        y, mean, rstd = layer_norm(x, weight, bias, eps, return_stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.param_dtype = next((t.dtype for t in (weight, bias) if t is not None), None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        given = len(ctx.needs_input_grad)  # (arguments left to their defaults have no place in it)
        need = (*ctx.needs_input_grad[:3], False, False)[:3]
        return (*layer_norm_backward(dy, x, weight, mean, rstd, need, ctx.param_dtype), None)[:given]
