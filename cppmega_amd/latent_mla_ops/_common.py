"""Shared host-side helpers of the dense latent attention entry points."""
from __future__ import annotations

import contextlib

import torch

from .. import _lib


def launch_on(t: torch.Tensor):
    """(stream pointer, context) for a launch on ``t``'s device: the context makes that device current
    where another one is, as a launch on a stream of its own needs."""
    dev = _lib.ensure_device(t)
    here = contextlib.nullcontext() if dev == torch.cuda.current_device() else torch.cuda.device(dev)
    return _lib.stream_ptr(dev), here
