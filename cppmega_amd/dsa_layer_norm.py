"""Layer norm, forward and backward (gfx950 HIP kernels): the norm of the indexer's keys in
front of their rotary part, the scores (``IndexScores``) and the paged cache, and of any
other rows of up to 16384 elements.

    y = (x - mean) rstd weight + bias,    rstd = (mean((x - mean)^2) + eps)^-1/2

x [..., n] bf16 or f32; weight and bias [n], bf16 or f32, or None (ones, zeros); statistics
and sums in 32 bits, gradients bit-identical between runs.  A small step is bound by the host, half of it by the hand-off
between autograd's two threads: ``torch.autograd.set_multithreading_enabled(False)`` saves that, a captured graph both.
Capture a backward on leaves of its own (``x.detach().requires_grad_()``) while an eager graph of the same leaves is alive:
torch runs a leaf's accumulation on the stream of that graph, which a capture cannot join.
"""
from __future__ import annotations

import torch

from . import _lib
from .latent_mla_ops._common import launch_on, same_device

__all__ = ["LayerNorm", "layer_norm", "layer_norm_backward"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


def _rows(t, n, name):
    """t [..., n] as rows with a dense last axis and one row stride: a view where there is one."""
    assert t.dtype in _DTYPES, f"{name} must be bfloat16 or float32, got {t.dtype}"
    if t.ndim == 2 and t.is_contiguous():
        return t
    t = t.reshape(-1, n) if t.ndim != 2 else t
    return t if (t.stride(1) == 1 or n == 1) and t.stride(0) >= 0 else t.contiguous()


def _check_params(weight, bias, n):
    """-> dtype code of the parameters."""
    for name, t in (("weight", weight), ("bias", bias)):
        assert t is None or (t.dtype in _DTYPES and t.shape == (n,)), \
            f"{name} must be bfloat16 or float32 [{n}], got {t.dtype} {tuple(t.shape)}"
    assert weight is None or bias is None or weight.dtype == bias.dtype, f"weight is {weight.dtype}, bias {bias.dtype}"
    t = bias if weight is None else weight
    return _lib.DTYPE_F32 if t is None else _DTYPES[t.dtype]


def _like(x):
    """A new dense tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _forward(x, weight, bias, eps, keep):
    """-> y, and with ``keep`` the mean and rstd of every row, [2, rows] f32."""
    assert x.ndim >= 1 and x.shape[-1] > 0, f"x must be [..., n], got {tuple(x.shape)}"
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    n = x.shape[-1]
    rows = _rows(x, n, "x")
    w_code = _check_params(weight, bias, n)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    same_device(x, weight, bias)
    stream, here = launch_on(x)
    count, mean, stats = rows.shape[0], None, None
    with here:
        y = _like(x)
        if keep:
            stats = x.new_empty((2, count), dtype=torch.float32)
            mean = stats.data_ptr()
        rc = _lib.load().dsa_layer_norm_fwd(rows.data_ptr(), _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(), mean,
                                            mean + 4 * count if keep else None, count, n, rows.stride(0), eps, _DTYPES[x.dtype],
                                            w_code, stream)
    _lib.check(rc, "dsa_layer_norm_fwd")
    return y, stats


def _backward(dy, x, weight, mean, rstd, need, param_dtype):
    """-> (dx, dweight, dbias); mean and rstd are addresses, and what the callers checked holds."""
    n = x.shape[-1]
    rows, grad = _rows(x, n, "x"), _rows(dy, n, "dy")
    weight = None if weight is None else weight.contiguous()
    stream, here = launch_on(x)
    L = _lib.load()
    with here:
        dx = _like(x) if need[0] else None
        dw = x.new_empty((n,), dtype=param_dtype) if need[1] else None
        db = x.new_empty((n,), dtype=param_dtype) if need[2] else None
        ws_bytes = int(L.dsa_layer_norm_bwd_workspace_size(rows.shape[0], n)) if need[1] or need[2] else 0
        ws = x.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
        rc = L.dsa_layer_norm_bwd(grad.data_ptr(), rows.data_ptr(), _lib.ptr(weight), mean, rstd, _lib.ptr(dx),
                                  _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), ws_bytes, rows.shape[0], n, grad.stride(0),
                                  rows.stride(0), _DTYPES[x.dtype], _DTYPES[param_dtype], stream)
    _lib.check(rc, "dsa_layer_norm_bwd")
    return dx, dw, db


def layer_norm(x, weight=None, bias=None, eps=1e-5, return_stats=False):
    """y of x's shape and type, without a gradient (``LayerNorm.apply`` has one); with ``return_stats`` (y, mean, rstd), f32 of
    x's leading shape, for ``layer_norm_backward``."""
    y, stats = _forward(x, weight, bias, eps, return_stats)
    return (y, *stats.view(2, *x.shape[:-1])) if return_stats else y


def layer_norm_backward(dy, x, weight, mean, rstd, need=(True, True, True), param_dtype=None):
    """(dx, dweight, dbias) for the upstream gradient dy of x's shape and type, from the forward's statistics; ``need``
    says which are wanted (None for the others), param_dtype the type of dweight and dbias (default: weight's, else f32)."""
    assert dy.shape == x.shape and dy.dtype == x.dtype, f"dy is {dy.dtype} {tuple(dy.shape)}, x {x.dtype} {tuple(x.shape)}"
    for name, t in (("mean", mean), ("rstd", rstd)):
        assert t.dtype == torch.float32 and t.shape == x.shape[:-1] and t.is_contiguous(), \
            f"{name} must be contiguous float32 {tuple(x.shape[:-1])}, got {t.dtype} {tuple(t.shape)}"
    _check_params(weight, None, x.shape[-1])
    if param_dtype is None:
        param_dtype = torch.float32 if weight is None else weight.dtype
    assert weight is None or weight.dtype == param_dtype, f"weight is {weight.dtype}, param_dtype {param_dtype}"
    same_device(x, dy, weight, mean, rstd)
    return _backward(dy, x, weight, mean.data_ptr(), rstd.data_ptr(), need, param_dtype)


class LayerNorm(torch.autograd.Function):
    """apply(x, weight=None, bias=None, eps=1e-5) -> y, with gradients to x, weight and bias; second ones are refused."""

    @staticmethod
    def forward(ctx, x, weight=None, bias=None, eps=1e-5):
        y, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param_dtype = (bias.dtype if bias is not None else torch.float32) if weight is None else weight.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        given = ctx.needs_input_grad  # (arguments left to their defaults have no place in it)
        need = (*given, False, False)[:3]
        gradients = _Gradients.apply if torch.is_grad_enabled() else _gradients
        return (*gradients(dy, x, weight, stats, need, ctx.param_dtype), None)[:len(given)]


def _gradients(dy, x, weight, stats, need, param_dtype):
    mean = stats.data_ptr()
    return _backward(dy, x, weight, mean, mean + 4 * stats.shape[1], need, param_dtype)


class _Gradients(torch.autograd.Function):
    """The gradients under create_graph: they hang on dy, x and weight, so that whatever asks for theirs is refused."""

    @staticmethod
    def forward(ctx, *args):
        return _gradients(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("LayerNorm has no second gradients: detach what its first are used for")
