"""Shared host-side helpers of the dense latent attention entry points."""
from __future__ import annotations

import contextlib

import torch

from .. import _lib
from ..sparse_mla_ops._common import check_same_device

_HERE = contextlib.nullcontext()


def same_device(first, *rest):
    """``check_same_device`` at less time on the host where they are on one."""
    dev = first.device
    for t in rest:
        if t is not None and t.device != dev:
            check_same_device(first, *rest)


def dense(t: torch.Tensor) -> torch.Tensor:
    """``t`` if it is contiguous and 16-byte aligned, else a copy that is (``contiguous()`` leaves a misaligned tensor, and
    any strides of axes of one, as they are)."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def launch_on(t: torch.Tensor):
    """(stream pointer, context) for a launch on ``t``'s device: the context makes that device current
    where another one is, as a launch on a stream of its own needs."""
    dev = t.get_device()
    if dev not in _lib.checked_devices:  # (-1 for one that is on no GPU)
        dev = _lib.ensure_device(t)
    here = _HERE if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)
    return torch._C._cuda_getCurrentRawStream(dev), here  # (a Stream object of it would take a microsecond)
