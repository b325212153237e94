"""Shared host-side helpers of the dense latent attention entry points."""
from __future__ import annotations

import contextlib

import torch

from .. import _lib

_HERE = contextlib.nullcontext()


def launch_on(t: torch.Tensor):
    """(stream pointer, context) for a launch on ``t``'s device: the context makes that device current
    where another one is, as a launch on a stream of its own needs."""
    dev = _lib.ensure_device(t)
    here = _HERE if dev == torch.cuda.current_device() else torch.cuda.device(dev)
    return torch._C._cuda_getCurrentRawStream(dev), here  # (a Stream object of it would take a microsecond)
