"""A paged cache of latent rows, the plan of a serving step, and attention over the cache
(bf16 or MXFP4 rows, gfx950 HIP kernels).

A serving step of a latent-attention layer:

    plan = plan_latent_step(context_lens, query_lens, block_table, free_blocks, free_count, num_tokens, cache.block_size)
    latent_cache_append(cache, c_kv, k_pe, plan.slots)                     # every layer: the new tokens' rows
    out, lse = paged_latent_mla_fwd(q, cache, plan.block_table, plan.kv_lens, plan.query_starts, sm_scale=scale)
    # next step: plan.context_lens, plan.block_table, plan.free_blocks, plan.free_count

Nothing synchronises with the host, so a step of fixed sizes can be captured in a HIP
graph.  (d_qk, d_v) in {(576, 512), (128, 64)}: the latent's d_v channels, then the rope part.
``scale`` is the layer's: of the un-absorbed head, (d_nope + d_rope)^-0.5 (192^-0.5 where
LatentMLAExpanded trained it with its default), not of the cached row.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from ..sparse_mla_ops._common import unwrap_quantized
from ._common import launch_on, same_device
from .latent_mla import _check_bf16, _check_dense, _scale

_DIMS = ((576, 512), (128, 64))


def latent_cache_row_bytes(d_qk, d_v, fmt):
    """Bytes of a cache row: bf16 2 d_qk; MXFP4 d_v / 2 of e2m1 codes, 2 (d_qk - d_v) of bf16 rope and d_v / 32
    exponents, padded to 16 (576 / 512: 400 for bf16's 1152; 128 / 64: 176 for 256)."""
    if fmt == "bf16":
        return 2 * d_qk
    assert fmt == "mxfp4", f"fmt must be 'bf16' or 'mxfp4', got {fmt!r}"
    return (d_v // 2 + 2 * (d_qk - d_v) + d_v // 32 + 15) // 16 * 16


class LatentCache:
    """Pages of latent rows over a tensor of the caller's: ``data`` [num_blocks, block_size, d_qk] bfloat16, or
    [num_blocks, block_size, row bytes] uint8 for MXFP4 (the format follows from the type)."""

    __slots__ = ("data", "d_qk", "d_v", "fmt", "num_blocks", "block_size", "dtype_code")

    def __init__(self, data, d_qk=576, d_v=512):
        assert (d_qk, d_v) in _DIMS, f"(d_qk, d_v) must be one of {_DIMS}, got {(d_qk, d_v)}"
        assert data.dtype in (torch.bfloat16, torch.uint8), f"a cache is bfloat16 or uint8 (MXFP4), got {data.dtype}"
        self.fmt = "bf16" if data.dtype == torch.bfloat16 else "mxfp4"
        width = d_qk if self.fmt == "bf16" else latent_cache_row_bytes(d_qk, d_v, "mxfp4")
        assert data.ndim == 3 and data.shape[2] == width and data.shape[0] > 0 and 0 < data.shape[1] <= 65536, \
            f"a {self.fmt} cache of {d_qk} channels is [num_blocks, block_size, {width}], got {tuple(data.shape)}"
        _check_dense(data=data)
        self.data, self.d_qk, self.d_v = data, d_qk, d_v
        self.num_blocks, self.block_size = data.shape[0], data.shape[1]
        self.dtype_code = _lib.DTYPE_BF16 if self.fmt == "bf16" else _lib.DTYPE_MXFP4

    @classmethod
    def empty(cls, num_blocks, block_size, d_qk=576, d_v=512, fmt="bf16", device="cuda"):
        """A new cache; its rows hold nothing yet."""
        if fmt == "bf16":
            data = torch.empty((num_blocks, block_size, d_qk), dtype=torch.bfloat16, device=device)
        else:
            data = torch.empty((num_blocks, block_size, latent_cache_row_bytes(d_qk, d_v, fmt)), dtype=torch.uint8, device=device)
        return cls(data, d_qk, d_v)


def _check_slots(slots, T):
    assert slots.dtype == torch.int64 and slots.shape == (T,) and slots.is_contiguous(), \
        f"slots must be contiguous int64 [{T}], got {slots.dtype} {tuple(slots.shape)}"


def _strided(t, width, name):
    shape = t.shape
    assert len(shape) == 2 and shape[1] == width, f"{name} must be [tokens, {width}], got {tuple(shape)}"
    row, col = t.stride()
    return t if col == 1 and row % 8 == 0 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def latent_cache_append(cache, latent, rope, slots):
    """Write tokens' rows into the cache: latent [T, d_v] and rope [T, d_qk - d_v] bf16 (rows may be strided),
    token t into slot slots[t] = page * block_size + offset; a slot outside the cache is skipped.  A slot may be
    given once.  MXFP4: the latent is quantised in blocks of 32 channels to e2m1 with the scale
    2^(floor(log2 amax) - 2) (nearest even, saturating at 6), the rope part is kept in bf16; a block that holds
    Inf or NaN reads back as NaN."""
    latent, rope = _strided(latent, cache.d_v, "latent"), _strided(rope, cache.d_qk - cache.d_v, "rope")
    T = latent.shape[0]
    assert rope.shape[0] == T, f"latent has {T} tokens, rope {rope.shape[0]}"
    _check_bf16(latent=latent, rope=rope)
    _check_slots(slots, T)
    same_device(cache.data, latent, rope, slots)
    stream, here = launch_on(cache.data)
    with here:
        rc = _lib.load().dsa_latent_cache_append(cache.data.data_ptr(), latent.data_ptr(), latent.stride(0), rope.data_ptr(),
                                                 rope.stride(0), slots.data_ptr(), T, cache.num_blocks, cache.block_size,
                                                 cache.d_qk, cache.d_v, cache.dtype_code, stream)
    _lib.check(rc, "dsa_latent_cache_append")


def latent_cache_gather(cache, slots):
    """The rows at ``slots`` [T] int64 as bf16 [T, d_qk] (MXFP4: exactly the values that the codes stand for), zeros
    for a slot outside the cache: cached prefixes for the expanded form's up-projections."""
    T = slots.shape[0]
    _check_slots(slots, T)
    same_device(cache.data, slots)
    stream, here = launch_on(cache.data)
    with here:
        out = torch.empty((T, cache.d_qk), dtype=torch.bfloat16, device=slots.device)
        rc = _lib.load().dsa_latent_cache_gather(cache.data.data_ptr(), slots.data_ptr(), out.data_ptr(), T, cache.num_blocks,
                                                 cache.block_size, cache.d_qk, cache.d_v, cache.dtype_code, stream)
    _lib.check(rc, "dsa_latent_cache_gather")
    return out


class LatentStepPlan(NamedTuple):
    """What a step's calls take, and the state that the next step's plan takes (all on the device)."""

    block_table: torch.Tensor   # [R, W] int32: pages of every request after this step, -1 behind them
    slots: torch.Tensor         # [num_tokens] int64: cache slot of every new token, -1: none
    positions: torch.Tensor     # [num_tokens] int32: position in its request, -1: none
    query_starts: torch.Tensor  # [R + 1] int32: first token of every request; tokens from the last entry on are padding
    kv_lens: torch.Tensor       # [R] int32: keys of every request with its new tokens, 0 where it was not granted
    context_lens: torch.Tensor  # [R] int32: the next step's context lengths
    granted: torch.Tensor       # [R] int32: 1 where the request's new tokens (or none) have their pages
    free_blocks: torch.Tensor   # [F] int32: pages that are free after this step, -1 behind them
    free_count: torch.Tensor    # [1] int32


def plan_latent_step(context_lens, query_lens, block_table, free_blocks, free_count, num_tokens, block_size):
    """Pages, slots and lengths of a serving step, on the device, from the requests' lengths.

    context_lens [R] int32: cached tokens of every request; query_lens [R] int32: its new tokens, in the order in
    which they lie in the step's token batch (0: none, -1: the request is done and gives its pages back);
    block_table [R, W] int32: its pages, without gaps from the front, -1 behind them (a new request: -1 alone);
    free_blocks [F] int32, of which the first free_count [1] int32 are free (F at least the cache's pages, so that every
    page can come back); num_tokens: length of the token batch.

    A context may be shorter than the step before left it (speculative tokens that were not kept): the request keeps the
    pages behind it for its next tokens, and gives all back when it is done.
    New pages come from the end of the free list, request by request.  A request is granted its tokens where they
    lie within the batch and within W pages and the pages that it and the requests before it need are there (one
    that needs no page is granted all the same); otherwise its tokens get no slot, its kv length is 0 and its
    context stays as it was, for a later step.  Pages given back are free from the next step on, in request order
    behind those left.  The inputs are not written.  -> ``LatentStepPlan``
    """
    ins = dict(context_lens=context_lens, query_lens=query_lens, block_table=block_table, free_blocks=free_blocks,
               free_count=free_count)
    for name, t in ins.items():
        assert t.dtype == torch.int32 and t.is_contiguous(), f"{name} must be contiguous int32, got {t.dtype}"
    R, (F,) = context_lens.shape[0], free_blocks.shape
    assert context_lens.ndim == 1 and query_lens.shape == context_lens.shape, "context_lens and query_lens must be [requests]"
    assert block_table.ndim == 2 and block_table.shape[0] == R and block_table.shape[1] > 0, \
        f"block_table must be [{R}, pages], got {tuple(block_table.shape)}"
    assert free_count.numel() == 1 and F > 0, "free_blocks must hold a page at least, free_count one number"
    assert num_tokens >= 0 and block_size > 0, f"bad num_tokens={num_tokens} or block_size={block_size}"
    same_device(*ins.values())
    W, dev = block_table.shape[1], context_lens.device
    stream, here = launch_on(context_lens)
    with here:
        # one allocation for the int32 results: nine take half of the call's time on the host
        table, positions, starts, kv_lens, lens, granted, free, count = torch.empty(
            R * W + num_tokens + 4 * R + F + 2, dtype=torch.int32, device=dev).split((R * W, num_tokens, R + 1, R, R, R, F, 1))
        p = LatentStepPlan(block_table=table.view(R, W), slots=torch.empty(num_tokens, dtype=torch.int64, device=dev),
                           positions=positions, query_starts=starts, kv_lens=kv_lens, context_lens=lens, granted=granted,
                           free_blocks=free, free_count=count)
        rc = _lib.load().dsa_latent_plan_step(*(t.data_ptr() for t in ins.values()), *(t.data_ptr() for t in p), R, W, F,
                                              num_tokens, block_size, stream)
    _lib.check(rc, "dsa_latent_plan_step")
    return p


def paged_latent_mla_fwd(q, cache, block_table, kv_lens, query_starts=None, sm_scale=None, out=None, lse=None):
    """Attention of new tokens over the cache (absorbed form): (out [T, H, d_v] bf16, lse [T, H] f32, log2 units).

    q [T, H, d_qk] bf16; block_table [R, W] int32; kv_lens [R] int32: keys of every request, those of its new tokens
    among them; query_starts [R + 1] int32, ascending: request r has the tokens query_starts[r] .. query_starts[r + 1],
    the last of its kv_lens[r] positions, and each sees the positions up to its own; without query_starts token r is
    request r's one new token (decoding; T = R).  A page outside the cache hides its keys, and a token without keys
    (or with scores of -Inf alone, or below -2^31 in log2 units) has out 0 and lse -inf.  Rows of tokens that belong to no
    request are not written: pass ``out`` and ``lse`` to keep what they hold.  Keys that a token does not see may hold
    anything, Inf and NaN too.  sm_scale None is d_qk^-0.5, of the cached row's width: a layer whose scale is that of its
    un-absorbed heads (LatentMLAExpanded's default) passes its own.
    """
    q = unwrap_quantized(q)
    assert q.ndim == 3 and q.shape[2] == cache.d_qk, f"q must be [tokens, heads, {cache.d_qk}], got {tuple(q.shape)}"
    T, H, D = q.shape
    R = kv_lens.shape[0]
    _check_bf16(q=q)
    _check_dense(q=q)
    assert kv_lens.ndim == 1 and block_table.ndim == 2 and block_table.shape[0] == R and block_table.shape[1] > 0, \
        f"kv_lens must be [requests] and block_table [requests, pages], got {tuple(kv_lens.shape)}, {tuple(block_table.shape)}"
    for name, t in (("block_table", block_table), ("kv_lens", kv_lens), ("query_starts", query_starts)):
        assert t is None or (t.dtype == torch.int32 and t.is_contiguous()), f"{name} must be contiguous int32"
    if query_starts is None:
        assert T == R, f"without query_starts every request has one token: {T} tokens, {R} requests"
    else:
        assert tuple(query_starts.shape) == (R + 1,), f"query_starts must be [{R + 1}], got {tuple(query_starts.shape)}"
    same_device(q, cache.data, block_table, kv_lens, query_starts, out, lse)
    scale = _scale(sm_scale, D)
    stream, here = launch_on(q)
    L = _lib.load()
    W = block_table.shape[1]
    with here:
        if out is None:
            out = torch.empty((T, H, cache.d_v), dtype=torch.bfloat16, device=q.device)
        if lse is None:
            lse = torch.empty((T, H), dtype=torch.float32, device=q.device)
        assert tuple(out.shape) == (T, H, cache.d_v) and tuple(lse.shape) == (T, H) and lse.dtype == torch.float32
        _check_bf16(out=out)
        _check_dense(out=out, lse=lse)
        n = int(L.dsa_paged_latent_mla_workspace_size(T, R, W, cache.block_size, H, D, cache.d_v))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        rc = L.dsa_paged_latent_mla_fwd(q.data_ptr(), cache.data.data_ptr(), block_table.data_ptr(), _lib.ptr(query_starts),
                                        kv_lens.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), n, T, R, W, H, D,
                                        cache.d_v, cache.num_blocks, cache.block_size, cache.dtype_code, scale, stream)
    _lib.check(rc, "dsa_paged_latent_mla_fwd")
    return out, lse
