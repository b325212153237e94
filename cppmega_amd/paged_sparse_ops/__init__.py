"""Sparse attention from a paged cache on gfx950: what serves a DSA layer.

The index keys live in pages of their own (``IndexKeyCache``, bf16, MXFP8 or MXFP4) under
the page numbers and slots of the latent cache, so one ``plan_latent_step`` serves both;
``paged_indexer_topk`` picks each new token's top-k positions from them and
``paged_sparse_mla_fwd`` attends to the cached latent rows at those.  Every entry point
launches the HIP kernels of libdsa_hip.so; importing this package does not load the library.
"""
from .index_keys import (
    IndexKeyCache,
    index_key_append,
    index_key_gather,
    index_key_row_bytes,
    paged_index_scores,
    paged_indexer_topk,
)
from .paged_sparse_mla import paged_sparse_mla_fwd

__all__ = [
    "IndexKeyCache",
    "index_key_append",
    "index_key_gather",
    "index_key_row_bytes",
    "paged_index_scores",
    "paged_indexer_topk",
    "paged_sparse_mla_fwd",
]
