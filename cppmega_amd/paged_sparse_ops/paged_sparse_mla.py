"""SparseMLA over the paged latent cache (gfx950 HIP kernels)."""
from __future__ import annotations

import torch

from .. import _lib
from ..latent_mla_ops._common import launch_on, same_device
from ..latent_mla_ops.latent_mla import _check_bf16, _check_dense, _scale
from ..sparse_mla_ops._common import unwrap_quantized
from .index_keys import check_requests


def paged_sparse_mla_fwd(q, cache, indices, block_table, kv_lens, query_starts=None, sm_scale=None, out=None, lse=None):
    """Sparse attention of new tokens over a ``LatentCache`` (absorbed form): (out [T, H, d_v] bf16, lse [T, H] f32, log2
    units), as ``SparseMLA`` gives them for the same rows.

    indices [T, topk] int32: the positions in its request that token t attends to, in any order; a position outside the
    token's own ones (-1, or past itself) or on a page outside the cache is masked, a repeated one counts every time.
    ``paged_indexer_topk`` gives them.  Everything else as in ``paged_latent_mla_fwd``: q [T, H, d_qk] bf16, block_table
    [R, W], kv_lens [R] and query_starts [R + 1] int32 (None: one token a request); a token whose every pick is masked has
    out 0 and lse -inf, rows of tokens of no request are not written (pass ``out`` and ``lse`` to keep what they hold),
    and what is masked may hold anything.  sm_scale None is d_qk^-0.5: a layer passes its own head's.
    """
    q = unwrap_quantized(q)
    assert q.ndim == 3 and q.shape[2] == cache.d_qk, f"q must be [tokens, heads, {cache.d_qk}], got {tuple(q.shape)}"
    T, H, D = q.shape
    _check_bf16(q=q)
    _check_dense(q=q)
    assert indices.dtype == torch.int32 and indices.ndim == 2 and indices.shape[0] == T and indices.shape[1] > 0 \
        and indices.is_contiguous(), f"indices must be contiguous int32 [{T}, topk], got {indices.dtype} {tuple(indices.shape)}"
    R, W = check_requests(T, block_table, kv_lens, query_starts)
    topk = indices.shape[1]
    same_device(q, cache.data, indices, block_table, kv_lens, query_starts, out, lse)
    scale = _scale(sm_scale, D)
    stream, here = launch_on(q)
    L = _lib.load()
    with here:
        if out is None:
            out = q.new_empty((T, H, cache.d_v))
        if lse is None:
            lse = q.new_empty((T, H), dtype=torch.float32)
        assert out.shape == (T, H, cache.d_v) and lse.shape == (T, H) and lse.dtype == torch.float32
        _check_bf16(out=out)
        _check_dense(out=out, lse=lse)
        n = int(L.dsa_paged_sparse_mla_workspace_size(T, H, topk, D, cache.d_v))
        ws = q.new_empty((n,), dtype=torch.uint8) if n else None
        rc = L.dsa_paged_sparse_mla_fwd(q.data_ptr(), cache.data.data_ptr(), indices.data_ptr(), block_table.data_ptr(),
                                        _lib.ptr(query_starts), kv_lens.data_ptr(), out.data_ptr(), lse.data_ptr(), _lib.ptr(ws),
                                        n, T, R, W, H, topk, D, cache.d_v, cache.num_blocks, cache.block_size, cache.dtype_code,
                                        scale, stream)
    _lib.check(rc, "dsa_paged_sparse_mla_fwd")
    return out, lse
