"""A paged cache of index keys, and the indexer's scores and top-k over it (gfx950 HIP kernels).

A serving step of a DSA layer:

    plan = plan_latent_step(context_lens, query_lens, block_table, free_blocks, free_count, num_tokens, cache.block_size)
    latent_cache_append(cache, c_kv, k_pe, plan.slots)
    index_key_append(keys, k_index, plan.slots)                  # pages of the same numbers and size as the latent cache's
    picks = paged_indexer_topk(q_index, w_index, keys, plan.block_table, plan.kv_lens, topk, plan.query_starts)
    out, lse = paged_sparse_mla_fwd(q, cache, picks, plan.block_table, plan.kv_lens, plan.query_starts, sm_scale=scale)

Nothing synchronises with the host, so a step of fixed sizes can be captured in a HIP graph.
"""
from __future__ import annotations

import torch

from .. import _lib
from ..dsa_topk import topk_indices
from ..latent_mla_ops._common import launch_on, same_device
from ..latent_mla_ops.latent_cache import _check_slots, _strided
from ..latent_mla_ops.latent_mla import _check_bf16, _check_dense

_CODES = {"bf16": _lib.DTYPE_BF16, "mxfp8": _lib.DTYPE_MXFP8, "mxfp4": _lib.DTYPE_MXFP4}


def index_key_row_bytes(d, fmt):
    """Bytes of a page per key: bf16 2 d; MXFP8 d codes, MXFP4 d / 2, and four exponent bytes."""
    assert fmt in _CODES, f"fmt must be one of {tuple(_CODES)}, got {fmt!r}"
    return 2 * d if fmt == "bf16" else (d if fmt == "mxfp8" else d // 2) + 4


class IndexKeyCache:
    """Pages of index keys of d channels (64 or 128) over a tensor of the caller's: ``data`` [num_blocks, block_size, d]
    bfloat16, or [num_blocks, block_size, bytes per key] uint8 for MXFP8 (d + 4) and MXFP4 (d / 2 + 4): the format follows
    from the type and the width.  A page of an MX cache, whose block_size is a multiple of 4, holds the codes of its keys
    and behind them their exponents: ``data``'s rows are no keys."""

    __slots__ = ("data", "d", "fmt", "num_blocks", "block_size", "dtype_code")

    def __init__(self, data, d=128):
        assert d in (64, 128), f"index keys have 64 or 128 channels, got {d}"
        assert data.dtype in (torch.bfloat16, torch.uint8), f"a cache is bfloat16 or uint8 (MXFP8, MXFP4), got {data.dtype}"
        assert data.ndim == 3 and data.shape[0] > 0 and 0 < data.shape[1] <= 65536, \
            f"a cache is [num_blocks, block_size, width], got {tuple(data.shape)}"
        kinds = ("bf16",) if data.dtype == torch.bfloat16 else ("mxfp8", "mxfp4")
        widths = {(d if f == "bf16" else index_key_row_bytes(d, f)): f for f in kinds}
        assert data.shape[2] in widths, f"a {data.dtype} cache of {d} channels has a width of {tuple(widths)}, got {data.shape[2]}"
        self.fmt = widths[data.shape[2]]
        assert self.fmt == "bf16" or data.shape[1] % 4 == 0, f"pages of MX keys hold a multiple of 4, got {data.shape[1]}"
        _check_dense(data=data)
        self.data, self.d = data, d
        self.num_blocks, self.block_size = data.shape[0], data.shape[1]
        self.dtype_code = _CODES[self.fmt]

    @classmethod
    def empty(cls, num_blocks, block_size, d=128, fmt="mxfp8", device="cuda"):
        """A new cache; its pages hold nothing yet."""
        n = index_key_row_bytes(d, fmt)
        if fmt == "bf16":
            data = torch.empty((num_blocks, block_size, d), dtype=torch.bfloat16, device=device)
        else:
            data = torch.empty((num_blocks, block_size, n), dtype=torch.uint8, device=device)
        return cls(data, d)


def index_key_append(cache, k, slots):
    """Write tokens' index keys into the cache: k [T, d] bf16 (rows may be strided), token t into slot slots[t] (int64) =
    page * block_size + offset; a slot outside the cache is skipped.  A slot may be given once.  MXFP8: blocks of 32
    channels become e4m3 under the least power of two that keeps their largest magnitude at 448 or below; MXFP4: e2m1
    under 2^(floor(log2 amax) - 2), saturating at 6; both to nearest, ties to even.  A block that holds Inf or NaN reads
    back as NaN."""
    k = _strided(k, cache.d, "k")
    T = k.shape[0]
    _check_bf16(k=k)
    _check_slots(slots, T)
    same_device(cache.data, k, slots)
    stream, here = launch_on(cache.data)
    with here:
        rc = _lib.load().dsa_index_key_append(cache.data.data_ptr(), k.data_ptr(), k.stride(0), slots.data_ptr(), T,
                                              cache.num_blocks, cache.block_size, cache.d, cache.dtype_code, stream)
    _lib.check(rc, "dsa_index_key_append")


def index_key_gather(cache, slots):
    """The index keys at ``slots`` [T] int64 as bf16 [T, d] (MX: exactly the values that the codes stand for), zeros for
    a slot outside the cache."""
    T = slots.shape[0]
    _check_slots(slots, T)
    same_device(cache.data, slots)
    stream, here = launch_on(cache.data)
    with here:
        out = slots.new_empty((T, cache.d), dtype=torch.bfloat16)
        rc = _lib.load().dsa_index_key_gather(cache.data.data_ptr(), slots.data_ptr(), out.data_ptr(), T, cache.num_blocks,
                                              cache.block_size, cache.d, cache.dtype_code, stream)
    _lib.check(rc, "dsa_index_key_gather")
    return out


def check_requests(T, block_table, kv_lens, query_starts):
    """-> requests, pages of a request."""
    R = kv_lens.shape[0]
    assert kv_lens.ndim == 1 and block_table.ndim == 2 and block_table.shape[0] == R and block_table.shape[1] > 0, \
        f"kv_lens must be [requests] and block_table [requests, pages], got {tuple(kv_lens.shape)}, {tuple(block_table.shape)}"
    for name, t in (("block_table", block_table), ("kv_lens", kv_lens), ("query_starts", query_starts)):
        assert t is None or (t.dtype == torch.int32 and t.is_contiguous()), f"{name} must be contiguous int32"
    if query_starts is None:
        assert T == R, f"without query_starts every request has one token: {T} tokens, {R} requests"
    else:
        assert query_starts.shape == (R + 1,), f"query_starts must be [{R + 1}], got {tuple(query_starts.shape)}"
    return R, block_table.shape[1]


def _check_scores(q, weights, cache, block_table, kv_lens, query_starts, num_keys):
    assert q.ndim == 3 and q.shape[2] == cache.d, f"q must be [tokens, heads, {cache.d}], got {tuple(q.shape)}"
    T, H, _ = q.shape
    _check_bf16(q=q)
    _check_dense(q=q)
    assert weights.dtype in (torch.float32, torch.bfloat16) and weights.shape == (T, H) and weights.is_contiguous(), \
        f"weights must be contiguous float32 or bfloat16 [{T}, {H}], got {weights.dtype} {tuple(weights.shape)}"
    R, W = check_requests(T, block_table, kv_lens, query_starts)
    most = W * cache.block_size
    L = most if num_keys is None else num_keys
    assert 0 <= L <= most, f"num_keys must be in [0, {most}], got {num_keys}"
    return T, H, R, W, L


def paged_index_scores(q, weights, cache, block_table, kv_lens, query_starts=None, num_keys=None, use_relu=True, out=None):
    """The indexer's scores of new tokens over the cached index keys: [T, num_keys] f32,

        out[t, s] = sum_h weights[t, h] relu(q[t, h] . k[s])    for the positions s of t's request up to its own,

    -inf for the other positions and for keys whose page lies outside the cache.  q [T, H, d] bf16 (H 16, 32 or 64),
    weights [T, H] f32 or bf16; block_table, kv_lens and query_starts as ``paged_latent_mla_fwd`` takes them.  num_keys:
    columns of the result, by default all that block_table has room for; a caller that knows the longest request passes
    its length.  Rows of tokens that belong to no request are not written: pass ``out`` to keep what they hold.  What a
    key that a token does not see holds reaches nothing; Inf and NaN of one that it sees reach that key's score alone.
    """
    T, H, R, W, L = _check_scores(q, weights, cache, block_table, kv_lens, query_starts, num_keys)
    same_device(q, weights, cache.data, block_table, kv_lens, query_starts, out)
    stream, here = launch_on(q)
    with here:
        if out is None:
            out = q.new_empty((T, L), dtype=torch.float32)
        assert out.shape == (T, L) and out.dtype == torch.float32 and out.is_contiguous(), \
            f"out must be contiguous float32 [{T}, {L}], got {out.dtype} {tuple(out.shape)}"
        rc = _lib.load().dsa_paged_index_scores(
            q.data_ptr(), weights.data_ptr(), cache.data.data_ptr(), block_table.data_ptr(), _lib.ptr(query_starts),
            kv_lens.data_ptr(), out.data_ptr(), None, T, R, W, 0, T, L, H, cache.d, cache.num_blocks, cache.block_size,
            cache.dtype_code, _lib.DTYPE_F32 if weights.dtype == torch.float32 else _lib.DTYPE_BF16, 1 if use_relu else 0, stream)
    _lib.check(rc, "dsa_paged_index_scores")
    return out


def paged_indexer_topk(q, weights, cache, block_table, kv_lens, topk, query_starts=None, num_keys=None, use_relu=True,
                       max_scratch_bytes=1 << 30):
    """Positions of each new token's top-k scores, [T, topk] int32, ascending, -1 padded (``topk_indices`` over
    ``paged_index_scores``: equal scores prefer the lower position, NaN ranks as +inf): what ``paged_sparse_mla_fwd``
    takes.  The scores go through a scratch of at most ``max_scratch_bytes`` (one token's at least), tokens in chunks.
    A token with fewer than topk keys gets all of them (those on no page too, which the attention masks), a token of
    no request -1 alone.  num_keys, and topk with it, have ``topk_indices``' limits: a caller with room for more in
    its block_table passes the longest request's length.
    """
    T, H, R, W, L = _check_scores(q, weights, cache, block_table, kv_lens, query_starts, num_keys)
    assert topk > 0, f"topk must be positive, got {topk}"
    same_device(q, weights, cache.data, block_table, kv_lens, query_starts)
    stream, here = launch_on(q)
    lib = _lib.load()
    with here:
        if T == 0 or L == 0:
            return torch.full((T, topk), -1, dtype=torch.int32, device=q.device)
        step = max(1, min(T, max_scratch_bytes // (4 * L)))
        scores = q.new_empty((step, L), dtype=torch.float32)
        parts = []
        for first in range(0, T, step):
            n = min(step, T - first)
            windows = q.new_empty((2, n), dtype=torch.int32)
            rc = lib.dsa_paged_index_scores(
                q.data_ptr(), weights.data_ptr(), cache.data.data_ptr(), block_table.data_ptr(), _lib.ptr(query_starts),
                kv_lens.data_ptr(), scores.data_ptr(), windows.data_ptr(), T, R, W, first, n, L, H, cache.d, cache.num_blocks,
                cache.block_size, cache.dtype_code, _lib.DTYPE_F32 if weights.dtype == torch.float32 else _lib.DTYPE_BF16,
                1 if use_relu else 0, stream)
            _lib.check(rc, "dsa_paged_index_scores")
            parts.append(topk_indices(scores[:n], topk, causal=False, starts=windows[0], ends=windows[1]))
        return parts[0] if len(parts) == 1 else torch.cat(parts)
