"""Dense latent attention on gfx950: the attention of a latent-attention (MLA) layer
without an indexer's selection, in training and from a paged cache.

``LatentMLA`` (absorbed: one latent row per token) and ``LatentMLAExpanded`` (keys and
values of every head) stand beside ``sparse_mla_ops.SparseMLA``: the same layouts, the
same (out, lse) results, every admitted key instead of a top-k.  Every entry point
launches the HIP kernels of libdsa_hip.so; importing this package does not load the
library.
"""
from .latent_cache import (
    LatentCache,
    LatentStepPlan,
    latent_cache_append,
    latent_cache_gather,
    latent_cache_row_bytes,
    paged_latent_mla_fwd,
    plan_latent_step,
)
from .latent_mla import (
    LatentMLA,
    LatentMLAExpanded,
    latent_mla_bwd,
    latent_mla_expanded_bwd,
    latent_mla_expanded_fwd,
    latent_mla_fwd_interface,
)

__all__ = [
    "LatentCache",
    "LatentMLA",
    "LatentMLAExpanded",
    "LatentStepPlan",
    "latent_cache_append",
    "latent_cache_gather",
    "latent_cache_row_bytes",
    "latent_mla_bwd",
    "latent_mla_expanded_bwd",
    "latent_mla_expanded_fwd",
    "latent_mla_fwd_interface",
    "paged_latent_mla_fwd",
    "plan_latent_step",
]
