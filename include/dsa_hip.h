/*
 * dsa_hip.h — C-ABI of the MI355X (gfx950) DeepSeek Sparse Attention hot path.
 *
 * Every entry point is stateless, stream-ordered and returns an int status
 * (DSA_OK == 0, negative on error; dsa_last_error() holds a per-thread
 * message).  All device buffers are caller-owned.  `stream` is a hipStream_t
 * passed as void* so that this header needs no HIP include; NULL means the
 * null stream.  Tensors are dense, row-major and contiguous in the shapes
 * given below.  No entry point allocates device memory; scratch space comes
 * from a caller-provided workspace sized by the matching *_workspace_size().
 *
 * Index convention (all SparseMLA entry points): indices are int32 and any
 * value outside [0, S_kv) — in particular the -1 sentinel — marks a masked
 * slot.  Duplicate indices are legal and counted once per occurrence.
 * LSE is returned in log2 units: lse2 = log2(sum_j exp(sm_scale * q.k_j)).
 * A (token, head) whose slots are all masked yields out = 0, lse2 = -inf and
 * zero gradients.
 */
#ifndef DSA_HIP_H_
#define DSA_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum dsa_status {
  DSA_OK = 0,
  DSA_ERR_INVALID_ARG = -1,  /* shape / pointer / range violation           */
  DSA_ERR_UNSUPPORTED = -2,  /* valid request this build has no kernel for  */
  DSA_ERR_HIP = -3,          /* HIP runtime error (launch, device query)    */
  DSA_ERR_WORKSPACE = -4     /* workspace missing or smaller than required  */
};

enum dsa_dtype {
  DSA_DTYPE_BF16 = 0,        /* bfloat16                                     */
  DSA_DTYPE_E4M3 = 1,        /* OCP float8 e4m3fn (max 448), gfx950 native   */
  DSA_DTYPE_F32 = 2,         /* float32                                      */
  DSA_DTYPE_I32 = 3,         /* int32 (index tensors)                        */
  DSA_DTYPE_I64 = 4,         /* int64 (index tensors)                        */
  DSA_DTYPE_MXFP8 = 5,       /* e4m3 with one f32 scale per 32 channels      */
  DSA_DTYPE_MXFP4 = 6        /* latent cache rows: e2m1, one exponent byte per 32 channels */
};

/* Per-thread message for the last non-zero status returned on this thread. */
const char *dsa_last_error(void);

/* ABI version (major * 100 + minor). */
int dsa_abi_version(void);

/* Returns DSA_OK when `device` is a gfx950 (MI355X-class) GPU, otherwise
 * DSA_ERR_UNSUPPORTED with the architecture named in dsa_last_error(). */
int dsa_device_check(int device);

/*
 * SparseMLA forward (MQA, packed latent KV).
 * Replaces sparse_mla_fwd_interface / the TileLang `sparse_mla_fwd` kernel
 *   (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_fwd.py:128-290,293-391)
 * and, with dtype == DSA_DTYPE_E4M3, sparse_mla_fwd_fp8_interface
 *   (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_fwd_fp8.py:178-393,415-559).
 *
 *   q       [B, S, H, D_qk]      bf16 or e4m3 (dtype)
 *   kv      [B, S_kv, G, D_qk]   bf16 or e4m3 (dtype); V = kv[..., :D_v]
 *   indices [B, S, G, topk]      int32
 *   out     [B, S, H, D_v]       bf16
 *   lse2    [B, S, H]            f32 (log2 units)
 *   q_scale [B, S], kv_scale [B, S_kv]  f32 dequant factors (real = fp8 * scale),
 *                                 required for e4m3, ignored (may be NULL) for bf16.
 * dtype DSA_DTYPE_MXFP8 (block-scaled e4m3): q / kv e4m3 with
 *   q_scale [B, S, H, D_qk / 32], kv_scale [B, S_kv, G, D_qk / 32], one f32
 *   factor per 32 consecutive channels; each block's q.k over the codes is
 *   multiplied by q_scale[block] * kv_scale[block] before the blocks are
 *   summed, and V is dequantised per block to bf16.  Replaces the block-scaled
 *   forward sparse_mla_blockscaled_mxfp8_fwd_interface
 *   (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_blockscaled_fused.py:248-418,694-793).
 *   (d_qk, d_v) in {(128, 64), (128, 128), (192, 128)}.
 * Head h reads kv group h / (H / G).  sm_scale multiplies the raw q.k dot.
 */
int dsa_sparse_mla_fwd(const void *q, const void *kv, const int32_t *indices,
                       void *out, float *lse2, int64_t B, int64_t S,
                       int64_t S_kv, int64_t H, int64_t G, int64_t D_qk,
                       int64_t D_v, int64_t topk, float sm_scale, int dtype,
                       const float *q_scale, const float *kv_scale,
                       void *stream);

/*
 * The same forward with a workspace.  e4m3 input: the V rows (the first D_v
 * columns of kv) are dequantised to bf16 once per call into the workspace,
 * bit-identical to the per-gather dequantisation of dsa_sparse_mla_fwd, and
 * the kernel gathers those rows instead of converting every gathered row
 * again.  MXFP8 input (d_qk/d_v 128/64, 128/128, 192/128, 576/512): whole kv
 * rows are dequantised to bf16 (code times its block scale) and every q and kv
 * block scale is checked on the device; if each is zero or a power of two in
 * [2^-40, 2^40] (OCP MX scales are powers of two), every dequantised value is
 * exact and the bf16 kernel runs on those rows with q converted at load (the
 * block-scaled scores up to the order of the fp32 sums), otherwise the
 * block-scaled e4m3 kernel runs, with the same result as dsa_sparse_mla_fwd.
 * The choice is made on the device (no host synchronisation; graph capture
 * safe).  dsa_sparse_mla_fwd_workspace_size returns the bytes needed (e4m3:
 * B * S_kv * G * D_v bf16, 0 for the d_qk = 576 kernels, which keep converting
 * V in LDS; MXFP8: B * S_kv * G * D_qk bf16 plus 256; bf16 input: 0, and then
 * `workspace` may be NULL).  Replaces the same reference interfaces as
 * dsa_sparse_mla_fwd.  A bf16 call neither reads nor writes `workspace`.
 *
 * dsa_sparse_mla_fwd_call is the same call for a caller that gives bf16 input a
 * workspace too.  dsa_sparse_mla_fwd_call_workspace_size returns the bytes it can
 * use: those of dsa_sparse_mla_fwd_workspace_size for e4m3 and MXFP8; for bf16
 * input with too few tokens to fill the GPU, room for the results of several
 * workgroups per (token, head) that share its slots.  Given a smaller workspace
 * (or NULL), a bf16 call runs unsplit.  The contents belong to one call from its
 * launch to its end: two calls that may run at the same time (on two streams)
 * need a workspace each.  It is 16-byte aligned for bf16 input.
 */
size_t dsa_sparse_mla_fwd_workspace_size(int64_t B, int64_t S_kv, int64_t G,
                                         int64_t D_qk, int64_t D_v, int dtype);
size_t dsa_sparse_mla_fwd_call_workspace_size(int64_t B, int64_t S, int64_t S_kv,
                                              int64_t H, int64_t G, int64_t D_qk,
                                              int64_t D_v, int64_t topk, int dtype);
int dsa_sparse_mla_fwd_ws(const void *q, const void *kv, const int32_t *indices,
                          void *out, float *lse2, int64_t B, int64_t S,
                          int64_t S_kv, int64_t H, int64_t G, int64_t D_qk,
                          int64_t D_v, int64_t topk, float sm_scale, int dtype,
                          const float *q_scale, const float *kv_scale,
                          void *workspace, size_t workspace_bytes, void *stream);
int dsa_sparse_mla_fwd_call(const void *q, const void *kv, const int32_t *indices,
                            void *out, float *lse2, int64_t B, int64_t S,
                            int64_t S_kv, int64_t H, int64_t G, int64_t D_qk,
                            int64_t D_v, int64_t topk, float sm_scale, int dtype,
                            const float *q_scale, const float *kv_scale,
                            void *workspace, size_t workspace_bytes, void *stream);

/* dsa_sparse_mla_bwd flags */
enum dsa_bwd_flags {
  /* Keep the per-(token, slot) dKV rows in fp32 instead of bf16 before the
   * deterministic fp32 reduction (2x the workspace traffic, fp32-exact rows). */
  DSA_BWD_FP32_PARTIALS = 1
};

/*
 * pass_bytes (every backward entry point below): the per-pass cap on the
 * backward's partial dKV rows, in bytes; 0 means the default of 4 GiB, and
 * every cap is lowered to at most 4 GiB - 1 MiB (a pass's rows are addressed
 * with 32-bit offsets).  The backward runs in passes over contiguous token ranges sized to this cap, so
 * its workspace stays bounded at any sequence length; a batch split over
 * passes carries its kv rows' sums in fp32 between them.  The workspace /
 * index size queries and the call they size must be given the same value.
 * No counterpart in the reference (whose backward scatters into one fp32 dKV
 * buffer with atomics).
 */

/* Bytes of workspace dsa_sparse_mla_bwd needs for these dimensions, flags and cap. */
size_t dsa_sparse_mla_bwd_workspace_size(int64_t B, int64_t S, int64_t S_kv,
                                         int64_t H, int64_t G, int64_t D_qk,
                                         int64_t D_v, int64_t topk, int flags,
                                         uint64_t pass_bytes);

/*
 * SparseMLA backward.
 * Replaces sparse_mla_bwd = preprocess + bwd + postprocess
 *   (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_bwd.py:114-201,204-419,422-531)
 * and, with dtype == DSA_DTYPE_E4M3, sparse_mla_bwd_fp8
 *   (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_bwd_fp8.py:191-489,492-630).
 *
 *   q, kv, indices, q_scale, kv_scale as in dsa_sparse_mla_fwd
 *   o   [B, S, H, D_v] bf16 (forward output), dO [B, S, H, D_v] bf16
 *   lse2 [B, S, H] f32 (forward LSE, log2 units)
 *   delta [B, S, H] f32 = sum_d o * dO, or NULL to compute it from o and dO
 *   dq  [B, S, H, D_qk] bf16 (written), dkv [B, S_kv, G, D_qk] bf16 (written)
 * dKV is reduced deterministically: every kv row sums its per-(token, slot)
 * contribution rows (fp16 with a per-row power-of-two scale taken from a bound
 * on the row, max|Q| sum|dS| + max|dO| sum P; fp32 with DSA_BWD_FP32_PARTIALS) in
 * ascending (token, kv group, slot) order in fp32, so repeated calls are
 * bitwise identical.  Gradients are with respect to the dequantised values
 * for e4m3 inputs.  The work runs in passes over token ranges whose partial
 * rows fit the per-pass cap pass_bytes, so the workspace is bounded; results
 * are deterministic for a given cap.
 * Limits: B * S_kv * G < 2^31, B * S * G * topk < 2^31.
 */
int dsa_sparse_mla_bwd(const void *q, const void *kv, const void *o,
                       const void *dO, const int32_t *indices,
                       const float *lse2, const float *delta, void *dq,
                       void *dkv, void *workspace,
                       size_t workspace_bytes, int64_t B, int64_t S,
                       int64_t S_kv, int64_t H, int64_t G, int64_t D_qk,
                       int64_t D_v, int64_t topk, float sm_scale, int dtype,
                       const float *q_scale, const float *kv_scale,
                       int flags, uint64_t pass_bytes, void *stream);

/*
 * The backward's inverse index (kv row -> entries) depends on the indices
 * alone, so a caller may build it ahead of the backward, e.g. on a second
 * stream while the forward runs, and pass it to dsa_sparse_mla_bwd_indexed,
 * which then runs only the main kernel and the dKV reduction (same results,
 * bit for bit, as dsa_sparse_mla_bwd).  Available when the backward runs in one
 * pass: dsa_sparse_mla_bwd_index_size returns 0 otherwise (then use
 * dsa_sparse_mla_bwd).  The index buffer must stay untouched between the two
 * calls and the build must be ordered before the backward (same stream, or an
 * event).  dsa_sparse_mla_bwd_indexed_workspace_size is the partial-row
 * workspace it needs besides the index.  No counterpart in the reference
 * (its backward has no inverse index).
 */
size_t dsa_sparse_mla_bwd_index_size(int64_t B, int64_t S, int64_t S_kv,
                                     int64_t H, int64_t G, int64_t D_qk,
                                     int64_t D_v, int64_t topk, int flags,
                                     uint64_t pass_bytes);
size_t dsa_sparse_mla_bwd_indexed_workspace_size(int64_t B, int64_t S,
                                                 int64_t S_kv, int64_t H,
                                                 int64_t G, int64_t D_qk,
                                                 int64_t D_v, int64_t topk,
                                                 int flags, uint64_t pass_bytes);
int dsa_sparse_mla_bwd_build_index(const int32_t *indices, int64_t B, int64_t S,
                                   int64_t S_kv, int64_t H, int64_t G,
                                   int64_t D_qk, int64_t D_v, int64_t topk,
                                   int flags, uint64_t pass_bytes, void *index,
                                   size_t index_bytes, void *stream);
int dsa_sparse_mla_bwd_indexed(const void *q, const void *kv, const void *o,
                               const void *dO, const int32_t *indices,
                               const float *lse2, const float *delta, void *dq,
                               void *dkv, const void *index, size_t index_bytes,
                               void *workspace, size_t workspace_bytes,
                               int64_t B, int64_t S, int64_t S_kv, int64_t H,
                               int64_t G, int64_t D_qk, int64_t D_v,
                               int64_t topk, float sm_scale, int dtype,
                               const float *q_scale, const float *kv_scale,
                               int flags, uint64_t pass_bytes, void *stream);

/*
 * DSA indexer scores: score[b, t, s] = sum_h w[t, b, h] * act(q[t, b, h, :] . k[s, b, :])
 * with act = ReLU when use_relu != 0, identity otherwise; fp32 accumulate.
 * Replaces Megatron `_compute_index_scores` as patched by
 *   compute_index_scores_fused_bf16 (cppmega/megatron/dsa_indexer_fused_patch.py:71-133).
 *
 *   q [Sq, B, H, D] (dtype), w [Sq, B, H] (w_dtype: bf16 or f32),
 *   k [Sk, B, D] (dtype), scores [B, Sq, Sk] f32.
 *   dtype e4m3: q_scale / k_scale point to one f32 each (per-tensor dequant).
 * causal: 0 = every (t, s) computed;
 *         1 = s > t written as -inf;
 *         2 = only s <= t written (the rest of each row is left untouched).
 */
int dsa_indexer_scores(const void *q, const void *w, const void *k,
                       float *scores, int64_t B, int64_t Sq, int64_t Sk,
                       int64_t H, int64_t D, int dtype, int w_dtype,
                       const float *q_scale, const float *k_scale, int causal,
                       int use_relu, void *stream);

/*
 * DSA indexer scores restricted to per-row windows, with Megatron's additive
 * mask: the scores fused_qk_topk_naive ranks when it is given a mask or varlen
 * windows (call shapes cppmega/megatron/lemyx_dsa_warmup.py:169-176,
 * cppmega/megatron/index_cache_patch.py:148-153):
 *   scores[b, t, s] = sum_h w * act(q . k) + mask[b, t, s]   for starts[b, t] <= s < ends[b, t]
 *                   = -inf                                    elsewhere.
 *   q, w, k, scores, dtype, w_dtype, q_scale, k_scale, use_relu as in
 *   dsa_indexer_scores; starts, ends [B, Sq] int32 (device);
 *   mask [Mb, Sq, Sk] f32 with batch stride mask_bstride elements (0: one mask
 *   shared by every batch) or NULL (no additive term);
 *   row_plain [B, Sq] int32 (device) or NULL: rows flagged nonzero have a mask
 *   of +0.0 on their whole window (dsa_mask_windows' plain flags), which is
 *   then not read (score + 0.0f: the same bits as score + mask).
 * Key tiles outside every window of a group of query tokens are not computed,
 * so a causal window costs the lower-triangle work.  Every element is written.
 */
int dsa_indexer_scores_masked(const void *q, const void *w, const void *k,
                              float *scores, int64_t B, int64_t Sq, int64_t Sk,
                              int64_t H, int64_t D, int dtype, int w_dtype,
                              const float *q_scale, const float *k_scale,
                              const int32_t *starts, const int32_t *ends,
                              const float *mask, int64_t mask_bstride,
                              const int32_t *row_plain, int use_relu,
                              void *stream);

/*
 * Per-row candidate windows of Megatron's additive mask (fused_qk_topk_naive's
 * mask argument, call shapes cppmega/megatron/lemyx_dsa_warmup.py:169-176):
 * for every row t of mask [mask_batches, Sq, Sk] f32 (mask_batches 1 = one
 * mask for every batch, or B), starts / ends [B, Sq] int32 get the first
 * finite column and one past the last ((0, 0) for a row without one), and
 * plain [B, Sq] int32 gets 1 when every entry in between is +0.0 (no finite
 * bias, no -inf / NaN hole), else 0.  One read of the mask, no host
 * synchronisation.  No counterpart in the reference (Megatron adds the mask
 * to the dense scores).
 */
int dsa_mask_windows(const float *mask, int64_t mask_batches, int64_t B,
                     int64_t Sq, int64_t Sk, int32_t *starts, int32_t *ends,
                     int32_t *plain, void *stream);

/*
 * Last step of the masked top-k: idx [rows, topk] int32 (dsa_topk output,
 * ascending, -1 padded) -> out [rows, topk] int64.  On rows not flagged in
 * plain [rows] (NULL: no row is), picks whose score in scores (rows of
 * row_stride f32) is -inf -- mask holes inside a window that held fewer
 * finite columns than topk -- become -1 and the remaining picks stay
 * ascending, padded with -1 at the end.  Megatron returns such picks as
 * indices (torch.topk over index_scores + mask); this build's contract
 * returns only the finite-mask columns.
 */
int dsa_topk_finalize(const float *scores, int64_t row_stride,
                      const int32_t *idx, int64_t rows, int64_t topk,
                      const int32_t *plain, int64_t *out, void *stream);

/*
 * Backward of dsa_indexer_scores (bf16 q / k): given grad_scores G [B, Sq, Sk] f32,
 *   dw[t, b, h]    = sum_s G[b, t, s] * act(L)
 *   dq[t, b, h, :] = w[t, b, h] * sum_s G[b, t, s] * act'(L) * k[s, b, :]
 *   dk[s, b, :]    = sum_{t, h} G[b, t, s] * w[t, b, h] * act'(L) * q[t, b, h, :]
 * with L = q[t, b, h, :] . k[s, b, :] recomputed on MFMA (act = ReLU when
 * use_relu, act' its 0/1 derivative; identity otherwise).  G * act'(L)
 * (times w for dk) is rounded to bf16 for the MFMA; sums are fp32.
 * Replaces the autograd backward of compute_index_scores_fused_bf16's
 * per-head loop (cppmega/megatron/dsa_indexer_fused_patch.py:71-133), the
 * gradient Megatron's indexer loss sends to the indexer's q, weights and k.
 *   q [Sq, B, H, D] bf16, w [Sq, B, H] (w_dtype), k [Sk, B, D] bf16;
 *   dq [Sq, B, H, D] bf16, dw [Sq, B, H] (w_dtype), dk [Sk, B, D] bf16 (written).
 * causal: 0 = every (t, s); 1 = only s <= t (G above the diagonal ignored).
 * starts / ends [B, Sq] int32 (device; both or neither): row windows, the
 * backward of dsa_indexer_scores_masked -- G outside [start, end) is ignored
 * (the masked forward writes -inf there whatever the raw score) and key tiles
 * outside every window of a group of rows are not computed, so a causal
 * window costs the lower-triangle work.
 * Deterministic (fixed summation orders, no atomics).  workspace >=
 * dsa_indexer_scores_backward_workspace_size() bytes (fp32 dk partials per
 * token chunk, and the windows' chunk flags).  Limits: Sq * Sk < 2^30,
 * H in {16, 32, 64}, D in {64, 128}.
 */
size_t dsa_indexer_scores_backward_workspace_size(int64_t B, int64_t Sq,
                                                  int64_t Sk, int64_t H,
                                                  int64_t D);
int dsa_indexer_scores_backward(const float *grad_scores, const void *q,
                                const void *w, const void *k, void *dq,
                                void *dw, void *dk, int64_t B, int64_t Sq,
                                int64_t Sk, int64_t H, int64_t D, int dtype,
                                int w_dtype, int causal, int use_relu,
                                const int32_t *starts, const int32_t *ends,
                                void *workspace, size_t workspace_bytes,
                                void *stream);

/*
 * Per-row top-k selection over fp32 scores.
 * Replaces the top-k of Megatron `fused_qk_topk_naive`
 *   (restated in scripts/modal_dsa_indexer_bench.py:188-194) with a stricter,
 * deterministic contract: the candidates of row r are columns [start, end);
 * the min(topk, end - start) largest are selected, ties break to the lower
 * column, NaN ranks as +inf, -0.0 equals +0.0; selected columns are written
 * in ascending order and the row is padded with -1.
 *
 *   scores  rows of `row_len` f32, row r at scores + r * row_stride
 *   out_idx [rows, topk] int32
 *   starts/ends: per-row int32 window; when NULL the window is
 *     causal != 0 : [0, min(row_len, (r % seq_q) + 1 + causal_offset))
 *     causal == 0 : [0, row_len)
 */
int dsa_topk(const float *scores, int64_t rows, int64_t row_len,
             int64_t row_stride, int64_t seq_q, int causal,
             int64_t causal_offset, const int32_t *starts,
             const int32_t *ends, int64_t topk, int32_t *out_idx,
             void *stream);

/*
 * dsa_topk for rows of any length up to 64 x 32768 columns (with
 * ceil(row_len / 32768) * topk <= 32768), the reach of the reference's
 * tl_topk, which streams rows of any seq_len (topk_selector.py:30-186).
 * dsa_topk takes rows of up to 32768 columns in one pass; longer rows run as
 * segments of at most 32768 columns, each segment's top-k, then one top-k
 * over the segments' picks (which hold the row's top-k), so the result
 * follows the same contract bit for bit.  Those passes use a workspace of
 * dsa_topk_workspace_size(rows, row_len, topk) bytes (0 for rows that fit
 * one pass, where workspace may be NULL).
 */
size_t dsa_topk_workspace_size(int64_t rows, int64_t row_len, int64_t topk);
int dsa_topk_ws(const float *scores, int64_t rows, int64_t row_len,
                int64_t row_stride, int64_t seq_q, int causal,
                int64_t causal_offset, const int32_t *starts,
                const int32_t *ends, int64_t topk, int32_t *out_idx,
                void *workspace, size_t workspace_bytes, void *stream);

/*
 * Streaming indexer + top-k: the top-k of the indexer scores of every query
 * row without the [B, Sq, Sk] score matrix, the target the reference states
 * for its indexer ("emit only [b, sq, topk] indices and optional top-k
 * scores", docs/status/cppmega_architecture_status.md:340-362).  Query rows
 * go through the workspace in chunks of as many rows as it holds
 * (workspace_bytes / (B * Sk * 4); causal chunks hold only keys up to their
 * last query row): per chunk the indexer kernel writes the chunk's scores
 * (causal: only s <= t) and the top-k kernel selects from them, so the
 * indices equal dsa_topk's on the same fp32 scores, bit for bit.  Rows over
 * 32768 keys also keep the top-k's segment passes in the workspace
 * (dsa_topk_workspace_size of the chunk's B * rows rows).
 *   q, w, k, dtype, w_dtype, q_scale, k_scale, use_relu as in dsa_indexer_scores;
 *   out_idx [B, Sq, topk] int32 (ascending, -1 padded; candidates s <= t when
 *   causal, every key otherwise); out_scores [B, Sq, topk] f32 (the selected
 *   scores, -inf for padding) or NULL.
 * workspace: >= dsa_indexer_topk_streaming_workspace_size(B, Sq, Sk, rows)
 * bytes for chunks of `rows` query rows (at least one row); for Sk > 32768
 * add 256 + dsa_topk_workspace_size(B * rows, Sk, topk).
 */
size_t dsa_indexer_topk_streaming_workspace_size(int64_t B, int64_t Sq, int64_t Sk,
                                                 int64_t chunk_rows);
int dsa_indexer_topk_streaming(const void *q, const void *w, const void *k,
                               int32_t *out_idx, float *out_scores, int64_t B,
                               int64_t Sq, int64_t Sk, int64_t H, int64_t D,
                               int dtype, int w_dtype, const float *q_scale,
                               const float *k_scale, int64_t topk, int causal,
                               int use_relu, void *workspace,
                               size_t workspace_bytes, void *stream);

/*
 * Fused indexer + top-k: the same indices (and selected scores) as
 * dsa_indexer_topk_streaming and as dsa_topk over dsa_indexer_scores, bit for
 * bit, with no score matrix and no workspace at all: each query row keeps a
 * bounded candidate list in on-chip memory while its keys are scored, and an
 * exact selection under the top-k contract (value descending, NaN as +inf,
 * -0 equal to +0, ties to the lower column) keeps its running top-k.  This is
 * the reference's stated target for its indexer ("fold top-k selection into
 * the per-head/tiled accumulation so the runtime emits only [b,sq,topk]",
 * docs/status/cppmega_architecture_status.md:358-359); the reference itself
 * materialises the scores (dsa_indexer_fused_patch.py:71-133 + topk).
 * Arguments as in dsa_indexer_topk_streaming (no workspace).  topk is at most
 * dsa_indexer_topk_fused_max_topk(H, D) (0: no kernel for that shape);
 * larger requests return DSA_ERR_UNSUPPORTED.
 */
int64_t dsa_indexer_topk_fused_max_topk(int64_t H, int64_t D);
int dsa_indexer_topk_fused(const void *q, const void *w, const void *k,
                           int32_t *out_idx, float *out_scores, int64_t B,
                           int64_t Sq, int64_t Sk, int64_t H, int64_t D,
                           int dtype, int w_dtype, const float *q_scale,
                           const float *k_scale, int64_t topk, int causal,
                           int use_relu, void *stream);

/*
 * Tensorwise (current-scaling) quantisation to OCP e4m3:
 *   amax = max|x|, scale = 448 / amax (1 when amax == 0),
 *   out = e4m3(RNE(x * scale)) saturated to +-448, scale_inv = 1 / scale.
 * Replaces the TE Float8CurrentScalingQuantizer call in per_token_cast_to_fp8
 *   (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_fwd_fp8.py:74-99,396-412).
 *   x [n] (in_dtype bf16 or f32), out_fp8 [n] e4m3, scale_inv [1] f32,
 *   workspace >= dsa_fp8_quantize_workspace_size() bytes.
 */
size_t dsa_fp8_quantize_workspace_size(void);
int dsa_fp8_tensorwise_quantize(const void *x, int64_t n, int in_dtype,
                                uint8_t *out_fp8, float *scale_inv,
                                void *workspace, size_t workspace_bytes,
                                void *stream);

/*
 * dsa_fp8_tensorwise_quantize without a workspace argument, for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  No counterpart in the reference.
 * Same arguments, result and error behaviour as dsa_fp8_tensorwise_quantize;
 * the scratch comes from a static device array of
 * dsa_fp8_quantize_workspace_size() bytes (4352) that each GPU holds until
 * the process ends, so every n is accepted.  The call allocates nothing.
 * Calls that overlap on one GPU (different streams) share that scratch and
 * race; serialise them on one stream.
 */
int dsa_fp8_tensorwise_quantize_noalloc(const void *x, int64_t n, int in_dtype,
                                        uint8_t *out_fp8, float *scale_inv,
                                        void *stream);

/*
 * e4m3 dequantisation: out[i] = value(x_fp8[i]) * scale_inv[0] (bf16 RNE or f32).
 * Replaces Float8Tensor.dequantize() (the TE tensors whose _data / _scale_inv
 *   cppmega's SparseMLA_FP8 unpacks, cppmega/megatron/sparse_mla_ops/sparse_mla.py:310-353);
 *   decodes with the same hardware conversion the e4m3 SparseMLA kernels use.
 *   x_fp8 [n] OCP e4m3fn, scale_inv [1] f32 (device), out [n] (out_dtype bf16 or f32).
 */
int dsa_fp8_dequantize(const uint8_t *x_fp8, int64_t n, const float *scale_inv,
                       void *out, int out_dtype, void *stream);

/*
 * Block-scaled e4m3 dequantisation: out[i] = value(x_fp8[i]) * scales[i / block]
 * (block a positive multiple of 4; 32 for MXFP8 rows).  Replaces
 *   _dequantize_mxfp8_tensor (cppmega/megatron/sparse_mla_ops/tilelang_sparse_mla_blockscaled_fused.py:961-969),
 *   which the reference's block-scaled backward runs before a bf16 backward.
 *   x_fp8 [n] e4m3, scales [n / block] f32, out [n] bf16 (RNE) or f32.
 */
int dsa_fp8_dequantize_blockwise(const uint8_t *x_fp8, int64_t n, int64_t block,
                                 const float *scales, void *out, int out_dtype,
                                 void *stream);

/*
 * DSA indexer KL loss (the indexer's training signal):
 *   a_h[t, s] = softmax_scale * query[t, b, h] . key[s, b, h / (H / G)]
 *   P[t, s]   = mean_h softmax over s <= t of a_h[t, :]      (sparse: and s in
 *               the row's top-k set)
 *   Q[t, s]   = softmax over all s in [0, Sk) of index_scores[b, t, :] (sparse:
 *               over the top-k set)
 *   row_loss[b, t] = sum_s P (ln(P + 1e-10) - ln(Q + 1e-10)),
 *   loss = loss_coeff * mean over (b, t) of row_loss.
 * Replaces compute_dsa_indexer_loss_splitk
 *   (cppmega/megatron/dsa_splitk_indexer_loss.py:328-468), the Triton split-K
 *   form of Megatron's compute_dsa_indexer_loss
 *   (clone at tests/test_dsa_splitk_indexer_loss.py:29-83).
 *
 *   index_scores [B, Sq, Sk] f32
 *   topk_indices [B, Sq, topk] int32 / int64 (topk_dtype), used when sparse != 0;
 *                values outside [0, Sk) are ignored, duplicates count once
 *   query [Sq, B, H, D] bf16, key [Sk, B, G, D] bf16 (G divides H; G = H is
 *                the reference's per-head key), D in {64, 128, 192, 256}
 *   loss [1] f32 (written), row_loss [B, Sq] f32 (written; may be NULL)
 * A row with no admissible attention column (sparse: no top-k column <= t) or
 * whose index softmax is undefined (all -inf, any NaN or +inf) gets a NaN row
 * loss, as the reference's softmax does, and the mean is then NaN.
 * Deterministic: fixed summation orders, no global atomics.
 * Limits: softmax_scale > 0, B * Sq * Sk < 2^29; sparse mode Sk <= 32768.
 */
size_t dsa_indexer_kl_loss_workspace_size(int64_t B, int64_t Sq, int64_t Sk,
                                          int64_t H, int64_t D, int sparse);
int dsa_indexer_kl_loss(const float *index_scores, const void *topk_indices,
                        int topk_dtype, int64_t topk, const void *query,
                        const void *key, float *loss, float *row_loss,
                        int64_t B, int64_t Sq, int64_t Sk, int64_t H,
                        int64_t G, int64_t D, float softmax_scale,
                        float loss_coeff, int sparse, void *workspace,
                        size_t workspace_bytes, void *stream);

/*
 * Gradient of dsa_indexer_kl_loss's scalar with respect to index_scores:
 *   grad_index_scores[b, t, s] = grad_loss[0] * loss_coeff / (B * Sq)
 *                                * (Q_s * R - P_s * Q_s / (Q_s + 1e-10)),
 *   R = sum_j P_j * Q_j / (Q_j + 1e-10)
 * (P the detached head-mean attention target, Q the index softmax; 0 where
 * Q_s = 0, NaN over a row whose loss is NaN).  Replaces the autograd path
 * through Megatron's compute_dsa_indexer_loss that the reference's split-K
 * loss (cppmega/megatron/dsa_splitk_indexer_loss.py:328-468) does not provide,
 * and the gradient the lemyx fused indexer loss returns to the index scores
 * (cppmega/megatron/lemyx_dsa_warmup.py:78-178).  grad_loss is a device
 * pointer (no host synchronisation).  Same arguments, limits and workspace
 * size as dsa_indexer_kl_loss; grad_index_scores [B, Sq, Sk] f32 must not
 * alias index_scores.
 */
int dsa_indexer_kl_loss_backward(const float *index_scores,
                                 const void *topk_indices, int topk_dtype,
                                 int64_t topk, const void *query,
                                 const void *key, const float *grad_loss,
                                 float *grad_index_scores, int64_t B,
                                 int64_t Sq, int64_t Sk, int64_t H, int64_t G,
                                 int64_t D, float softmax_scale,
                                 float loss_coeff, int sparse, void *workspace,
                                 size_t workspace_bytes, void *stream);

/*
 * The loss and the gradient together, for a caller that will ask for both: one
 * run leaves the loss (and row_loss, or NULL, as dsa_indexer_kl_loss; sparse: the
 * row sums in another order) and a state of
 * dsa_indexer_kl_loss_state_size bytes, from which
 * dsa_indexer_kl_loss_grad_apply forms grad_index_scores (as
 * dsa_indexer_kl_loss_backward up to that order) for any upstream gradient, any
 * number of times, without the scores, query or key.  The state is the size of
 * the scores, or (sparse) 4 bytes per top-k entry and about Sk / 8 + Sk / 32
 * bytes per row.  loss_coeff is read by the second call.  The workspace
 * (dsa_indexer_kl_loss_with_grad_workspace_size) is needed by the first only.
 * dsa_indexer_kl_loss_grad_state leaves the same state and no loss.
 */
size_t dsa_indexer_kl_loss_state_size(int64_t B, int64_t Sq, int64_t Sk, int64_t D,
                                      int64_t topk, int sparse);
size_t dsa_indexer_kl_loss_with_grad_workspace_size(int64_t B, int64_t Sq, int64_t Sk,
                                                    int64_t H, int64_t D, int64_t topk,
                                                    int sparse);
int dsa_indexer_kl_loss_with_grad(const float *index_scores, const void *topk_indices,
                                  int topk_dtype, int64_t topk, const void *query,
                                  const void *key, float *loss, float *row_loss,
                                  void *state, size_t state_bytes, int64_t B,
                                  int64_t Sq, int64_t Sk, int64_t H, int64_t G, int64_t D,
                                  float softmax_scale, float loss_coeff, int sparse,
                                  void *workspace, size_t workspace_bytes,
                                  void *stream);
int dsa_indexer_kl_loss_grad_state(const float *index_scores, const void *topk_indices,
                                   int topk_dtype, int64_t topk, const void *query,
                                   const void *key, void *state, size_t state_bytes,
                                   int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t G,
                                   int64_t D, float softmax_scale, float loss_coeff,
                                   int sparse, void *workspace, size_t workspace_bytes,
                                   void *stream);
int dsa_indexer_kl_loss_grad_apply(const void *state, size_t state_bytes,
                                   const float *grad_loss, float *grad_index_scores,
                                   int64_t B, int64_t Sq, int64_t Sk, int64_t D,
                                   int64_t topk, float loss_coeff, int sparse,
                                   void *stream);

/*
 * Top-k index mask of the sparse indexer loss.
 * Replaces Megatron's _scatter_topk_into_index_mask in the CUDA-graph-safe form
 *   cppmega patches in (cppmega/megatron/upstream_patches/apply_dsa_cg_patches.py:267-291;
 *   eager oracle upstream_prs/examples/01_dsa_cuda_graph_safety/reproducer.py:124-138).
 *
 *   topk_indices [B, rows, topk] int32 / int64 (topk_dtype): the top-k columns
 *                of mask rows [row0, row0 + rows); values outside [0, Sk) (the
 *                -1 sentinel) are skipped, duplicates are harmless
 *   mask [B, Sq, Sk] f32
 * fill_rows == 0: mask[b, row0 + r, s] = value for every listed s; nothing
 *                 else is written (the reference's in-place scatter).
 * fill_rows != 0: every element of rows [row0, row0 + rows) is written:
 *                 value on listed columns, fill elsewhere (Sk <= 262144).
 * One launch, no host synchronisation, idempotent: safe under graph capture.
 */
int dsa_topk_index_mask(const void *topk_indices, int topk_dtype, int64_t topk,
                        float *mask, int64_t B, int64_t Sq, int64_t Sk,
                        int64_t row0, int64_t rows, float value, float fill,
                        int fill_rows, void *stream);

/*
 * Dense latent attention: every key of a row's window instead of a top-k of them
 * (the attention of the DSA warm-up, and of layers without an indexer; bf16).
 *
 * Absorbed: q [B, S, H, D_qk], kv [B, S_kv, G, D_qk], V = kv[..., :D_v]; head h
 *   reads kv group h / (H / G).  (D_qk, D_v) in {(128, 64), (128, 128), (192, 128)}.
 * Expanded: q [B, S, H, D_nope + D_pe], k_nope [B, S_kv, H, D_nope], k_pe
 *   [B, S_kv, D_pe] shared by the heads, v [B, S_kv, H, D_v]; D_pe = 64 and
 *   (D_nope, D_v) in {(128, 128), (64, 64)}.  strides: in elements, of
 *   (k_nope: batch, token, head; k_pe: batch, token; v: batch, token, head), multiples
 *   of 8 (0 broadcasts), token strides below 2^23; the last axes are dense.
 * Row t sees the keys [starts[b, t], ends[b, t]) clipped to [0, S_kv) where the int32
 *   [B, S] windows are given (both or neither, causal 0); else, with causal, the keys up
 *   to position t + S_kv - S; else all.  A row without keys, or with scores of -Inf alone:
 *   out 0, lse2 -inf, no gradient.
 *   Keys outside a row's window reach neither its results nor its gradients, whatever
 *   they hold.
 *   Scores below -2^31 in log2 units (sm_scale log2(e) q . k) count as -Inf; a row whose
 *   largest score passes 2^24 in magnitude has an lse2 that does not tell its weights apart.
 *   out [B, S, H, D_v] bf16, lse2 [B, S, H] f32 (log2 units); sm_scale >= 2^-100.
 *   out_lo (may be NULL) [B, S, H, D_v] bf16: what rounding took from out.
 *
 * Backward, from the forward's out (o), out_lo (o_lo, may be NULL: the rows' o . dO is then
 * that of the rounded out, which costs up to a half more error in dq and dk where rows
 * have few keys), lse2 and the upstream gradient dO:
 *   dq, and dkv (absorbed) or dk_nope, dk_pe (summed over the heads), dv (expanded),
 *   all dense bf16.  No float atomics: repeated calls give the same bits.  workspace:
 *   dsa_latent_mla_bwd_workspace_size() bytes, 256-byte aligned (expanded: G = H,
 *   D_qk = D_nope + D_pe, expanded = 1; 0 where the sizes are refused).
 * Device pointers are 16-byte aligned.  Outputs and workspace overlap no input.
 */
int dsa_latent_mla_fwd(const void *q, const void *kv, const int32_t *starts, const int32_t *ends,
                       void *out, void *out_lo, float *lse2, int64_t B, int64_t S, int64_t S_kv,
                       int64_t H, int64_t G, int64_t D_qk, int64_t D_v, float sm_scale, int causal,
                       void *stream);
int dsa_latent_mla_expanded_fwd(const void *q, const void *k_nope, const void *k_pe, const void *v,
                                const int32_t *starts, const int32_t *ends, void *out, void *out_lo,
                                float *lse2, int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t D_nope,
                                int64_t D_pe, int64_t D_v, const int64_t *strides, float sm_scale,
                                int causal, void *stream);
size_t dsa_latent_mla_bwd_workspace_size(int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t G,
                                         int64_t D_qk, int64_t D_v, int expanded);
int dsa_latent_mla_bwd(const void *q, const void *kv, const void *o, const void *o_lo,
                       const void *dO, const float *lse2, const int32_t *starts, const int32_t *ends, void *dq, void *dkv, void *workspace,
                       size_t workspace_bytes, int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t G,
                       int64_t D_qk, int64_t D_v, float sm_scale, int causal, void *stream);
int dsa_latent_mla_expanded_bwd(const void *q, const void *k_nope, const void *k_pe, const void *v,
                                const void *o, const void *o_lo, const void *dO, const float *lse2,
                                const int32_t *starts, const int32_t *ends, void *dq, void *dk_nope, void *dk_pe, void *dv,
                                void *workspace, size_t workspace_bytes, int64_t B, int64_t S,
                                int64_t S_kv, int64_t H, int64_t D_nope, int64_t D_pe, int64_t D_v,
                                const int64_t *strides, float sm_scale, int causal, void *stream);

/*
 * Paged cache of latent rows: [num_blocks][block_size] rows of D_qk channels, the
 * latent's D_v and then the rope part; (D_qk, D_v) in {(576, 512), (128, 64)}.
 *   DSA_DTYPE_BF16   D_qk bf16
 *   DSA_DTYPE_MXFP4  D_v / 2 bytes of e2m1 codes (channel 2 i in the low half of byte
 *                    i), the rope part in bf16, D_v / 32 exponent bytes e (scale
 *                    2^(e - 127), 255: NaN), zero or more bytes up to a multiple of 16
 * A slot is page * block_size + offset.  dsa_latent_cache_row_bytes: bytes of a row (0
 * where the sizes are refused).
 * append: token t's latent (row stride latent_stride elements) and rope to slots[t];
 *   slots outside the cache are skipped; a slot may be given once.  MXFP4: scale
 *   2^(floor(log2 amax) - 2) of each 32 channels, its exponent held to +-125 (all zeros:
 *   2^0), codes to nearest even, saturating at 6; a block with Inf or NaN gets 255.
 * gather: out [T, D_qk] bf16 of slots (zeros outside the cache), exact.
 * Pointers of rows are 16-byte aligned, row strides multiples of 8 elements; T * D_qk / 8 at
 * most 2^32 - 256.
 */
int64_t dsa_latent_cache_row_bytes(int64_t D_qk, int64_t D_v, int dtype);
int dsa_latent_cache_append(void *cache, const void *latent, int64_t latent_stride, const void *rope,
                            int64_t rope_stride, const int64_t *slots, int64_t T, int64_t num_blocks,
                            int64_t block_size, int64_t D_qk, int64_t D_v, int dtype, void *stream);
int dsa_latent_cache_gather(const void *cache, const int64_t *slots, void *out, int64_t T,
                            int64_t num_blocks, int64_t block_size, int64_t D_qk, int64_t D_v, int dtype,
                            void *stream);

/*
 * Plan of a serving step, one launch: from context_lens [R] (cached tokens), query_lens
 * [R] (new tokens; negative: the request is done), block_table [R, W], free_blocks [F]
 * and free_count [1] (how many of its first entries are free), all int32 on the device,
 *   block_table_out [R, W]; slots int64 [T], positions [T] of the token batch (-1: none);
 *   query_starts [R + 1]; kv_lens [R] (context + new tokens, 0 where not granted);
 *   context_lens_out [R]; granted [R]; free_blocks_out [F], free_count_out [1].
 * A request's pages lie at the front of its row of block_table without gaps, a negative
 * entry ends them: its context's, and those of earlier tokens that were not kept (its
 * context may have shrunk since), which its next tokens take first.
 * New pages are taken from the end of the free list in request order; a request is
 * granted its tokens where they lie within T and W pages and the pages needed up to and
 * with it are free (or it needs none).  All pages of done requests are appended to what
 * is left.  Lengths and counts are clipped to their ranges.  No output may be an input.
 */
int dsa_latent_plan_step(const int32_t *context_lens, const int32_t *query_lens, const int32_t *block_table,
                         const int32_t *free_blocks, const int32_t *free_count, int32_t *block_table_out,
                         int64_t *slots, int32_t *positions, int32_t *query_starts, int32_t *kv_lens,
                         int32_t *context_lens_out, int32_t *granted, int32_t *free_blocks_out,
                         int32_t *free_count_out, int64_t R, int64_t W, int64_t F, int64_t T,
                         int64_t block_size, void *stream);

/*
 * Latent attention over the paged cache (absorbed form): q [T, H, D_qk] bf16, request
 * r's tokens query_starts[r] .. query_starts[r + 1] (ascending; NULL: token r alone) are
 * the last of its kv_lens[r] positions; a token sees the positions up to its own.
 * block_table [R, W] int32: an entry outside [0, num_blocks) hides its keys; lengths
 * past W * block_size are cut.  out [T, H, D_v] bf16, lse2 [T, H] f32; a token without
 * keys, or with scores of -Inf (below -2^31) alone: 0 and -inf; tokens of no request are
 * not written.  Keys that a token does not see do not reach it, whatever they hold.
 * workspace:
 * dsa_paged_latent_mla_workspace_size() bytes, 256-byte aligned.
 */
size_t dsa_paged_latent_mla_workspace_size(int64_t T, int64_t R, int64_t W, int64_t block_size, int64_t H,
                                           int64_t D_qk, int64_t D_v);
int dsa_paged_latent_mla_fwd(const void *q, const void *cache, const int32_t *block_table,
                             const int32_t *query_starts, const int32_t *kv_lens, void *out, float *lse2,
                             void *workspace, size_t workspace_bytes, int64_t T, int64_t R, int64_t W,
                             int64_t H, int64_t D_qk, int64_t D_v, int64_t num_blocks, int64_t block_size,
                             int dtype, float sm_scale, void *stream);

/*
 * Paged cache of index keys (the indexer's k), pages of the same numbers as the latent
 * cache's: [num_blocks] pages of block_size keys of D channels, D in {64, 128}.
 *   DSA_DTYPE_BF16   D bf16 a key
 *   DSA_DTYPE_MXFP8  the page's keys of D e4m3 codes, then four exponent bytes a key: byte b
 *                    is that of channels 32 b .. 32 b + 31 (scale 2^(e - 127), 255: NaN),
 *                    bytes past the last channel 0
 *   DSA_DTYPE_MXFP4  the same with D / 2 bytes of e2m1 codes a key (channel 2 i in the low
 *                    half of byte i)
 * block_size is a multiple of 4 for the MX formats.  dsa_index_key_row_bytes: a page's bytes
 * per key (0 where the sizes are refused).  A slot is page * block_size + offset.
 * append: k [T, D] bf16 (row stride k_stride elements) to slots[t]; slots outside the cache
 *   are skipped; a slot may be given once.  MXFP8: the scale of 32 channels is the least power
 *   of two under which their largest magnitude is at most 448, its exponent held to -117 ..
 *   119 (all zeros: 2^0); MXFP4: 2^(floor(log2 amax) - 2), held to +-125; codes to nearest
 *   even, saturating; a block with Inf or NaN gets 255.
 * gather: out [T, D] bf16 of slots (zeros outside the cache), exact.
 * Pointers of rows are 16-byte aligned, k_stride a multiple of 8; T < 2^28 (128 channels: T <= 2^28 - 16).
 */
int64_t dsa_index_key_row_bytes(int64_t D, int dtype);
int dsa_index_key_append(void *cache, const void *k, int64_t k_stride, const int64_t *slots, int64_t T,
                         int64_t num_blocks, int64_t block_size, int64_t D, int dtype, void *stream);
int dsa_index_key_gather(const void *cache, const int64_t *slots, void *out, int64_t T, int64_t num_blocks,
                         int64_t block_size, int64_t D, int dtype, void *stream);

/*
 * Indexer scores over the paged index keys: for tokens first .. first + tokens - 1 of a batch
 * of T,
 *   scores[t - first, s] = sum_h w[t, h] act(q[t, h] . k[s])   0 <= s < L (L <= W * block_size)
 * with act = ReLU when use_relu != 0, for the positions s of token t's request up to its own,
 * -inf for the others and for keys whose page lies outside the cache.  q [T, H, D] bf16, w
 * [T, H] bf16 or f32 (w_dtype), H in {16, 32, 64}; requests, block_table [R, W], query_starts
 * and kv_lens as in dsa_paged_latent_mla_fwd.  A NaN or Inf of a key, a query or a weight
 * reaches the scores of that key, token and no other.  Rows of tokens of no request are not
 * written.  windows [2, tokens] int32 (or NULL): the starts and ends of a top-k over the scores,
 * 0 and the columns that each token sees (0 for a token of no request).  With windows, columns
 * past a token's own may be left as they were.
 */
int dsa_paged_index_scores(const void *q, const void *w, const void *cache, const int32_t *block_table,
                           const int32_t *query_starts, const int32_t *kv_lens, float *scores, int32_t *windows,
                           int64_t T, int64_t R, int64_t W, int64_t first, int64_t tokens, int64_t L, int64_t H,
                           int64_t D, int64_t num_blocks, int64_t block_size, int dtype, int w_dtype, int use_relu,
                           void *stream);

/*
 * SparseMLA over the paged latent cache: token t attends to the cached rows at indices[t]
 * (int32 [T, topk], positions in its request, any order; a position outside the token's own
 * ones, in particular -1, is masked; a repeated one counts every time).  Everything else as
 * in dsa_paged_latent_mla_fwd, whose results for the same rows it gives; num_blocks *
 * block_size < 2^31, topk <= 2^27, T * ceil(H / 32) < 2^26 (128 channels: at most 2^26 - 4).  workspace:
 * dsa_paged_sparse_mla_workspace_size() bytes, 256-byte aligned (0: none, may be NULL).
 */
size_t dsa_paged_sparse_mla_workspace_size(int64_t T, int64_t H, int64_t topk, int64_t D_qk, int64_t D_v);
int dsa_paged_sparse_mla_fwd(const void *q, const void *cache, const int32_t *indices, const int32_t *block_table,
                             const int32_t *query_starts, const int32_t *kv_lens, void *out, float *lse2,
                             void *workspace, size_t workspace_bytes, int64_t T, int64_t R, int64_t W, int64_t H,
                             int64_t topk, int64_t D_qk, int64_t D_v, int64_t num_blocks, int64_t block_size,
                             int dtype, float sm_scale, void *stream);

/*
 * Layer norm over rows of n <= 16384 elements (the index keys', or any other):
 *   y = (x - mean) rstd weight + bias,  rstd = (mean((x - mean)^2) + eps)^-1/2
 * x [rows, n] bf16 or f32 (dtype; row stride x_stride elements, 0 repeats a row), weight and
 * bias [n] bf16 or f32 (w_dtype; NULL: ones, zeros), y [rows, n] of x's type; mean, rstd
 * [rows] f32 for the backward (or both NULL).
 * Backward, from dy [rows, n] of x's type (row stride dy_stride): dx [rows, n], dweight and
 * dbias [n] of the weights' type; each may be NULL.  No atomics: repeated calls give the same
 * bits.  workspace: dsa_layer_norm_bwd_workspace_size() bytes, 4-byte aligned (needed for
 * dweight and dbias).  Pointers are aligned to their elements.  Outputs overlap no input.
 */
int dsa_layer_norm_fwd(const void *x, const void *weight, const void *bias, void *y, float *mean, float *rstd,
                       int64_t rows, int64_t n, int64_t x_stride, float eps, int dtype, int w_dtype,
                       void *stream);
size_t dsa_layer_norm_bwd_workspace_size(int64_t rows, int64_t n);
int dsa_layer_norm_bwd(const void *dy, const void *x, const void *weight, const float *mean, const float *rstd,
                       void *dx, void *dweight, void *dbias, void *workspace, size_t workspace_bytes,
                       int64_t rows, int64_t n, int64_t dy_stride, int64_t x_stride, int dtype, int w_dtype,
                       void *stream);

/*
 * Stage timing (measurement aid; no counterpart in the reference, which
 * times whole calls with CUDA events in its benchmark scripts).  With
 * dsa_stage_timing(1) on a thread, every later dsa_sparse_mla_bwd call on
 * that thread records HIP events on its stream at its stage boundaries:
 * stage 0 = inverse index (CSR), 1 = main kernel (dQ + dKV partial rows),
 * 2 = dKV reduction.  Nothing synchronises until dsa_stage_times(back, ...)
 * reads the record of the call `back` calls ago (0 = most recent, up to 255)
 * and writes the elapsed milliseconds of its stages; it returns the number
 * of stages written (or a negative status).
 */
int dsa_stage_timing(int enable);
int dsa_stage_times(int back, float *ms, int max_stages);

#ifdef __cplusplus
}
#endif

#endif /* DSA_HIP_H_ */
