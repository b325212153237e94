// C entry points of the paged latent cache: argument checks.
#include <math.h>

#include "latent_cache.hpp"
#include "latent_paged.hpp"

using namespace dsa;

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int check_cache(const char *who, int64_t num_blocks, int64_t block, int64_t d_qk, int64_t d_v, int dtype) {
  DSA_REQUIRE(num_blocks > 0 && num_blocks < (1ll << 31) && block > 0 && block <= 65536,
              "%s: num_blocks=%lld must be in [1, 2^31), block_size=%lld in [1, 65536]", who, (long long)num_blocks, (long long)block);
  DSA_REQUIRE(dtype == DSA_DTYPE_BF16 || dtype == DSA_DTYPE_MXFP4, "%s: the cache is bf16 or MXFP4, got dtype %d", who, dtype);
  if (!((d_qk == 576 && d_v == 512) || (d_qk == 128 && d_v == 64)))
    return set_error(DSA_ERR_UNSUPPORTED, "%s: no kernel for rows of %lld channels, %lld of them latent (576 / 512, 128 / 64)", who,
                     (long long)d_qk, (long long)d_v);
  return DSA_OK;
}

extern "C" int64_t dsa_latent_cache_row_bytes(int64_t D_qk, int64_t D_v, int dtype) {
  if (check_cache("dsa_latent_cache_row_bytes", 1, 1, D_qk, D_v, dtype)) return 0;
  return cache_row_bytes(D_qk, D_v, dtype == DSA_DTYPE_MXFP4);
}

extern "C" int dsa_latent_cache_append(void *cache, const void *latent, int64_t latent_stride, const void *rope,
                                       int64_t rope_stride, const int64_t *slots, int64_t T, int64_t num_blocks,
                                       int64_t block_size, int64_t D_qk, int64_t D_v, int dtype, void *stream) {
  const char *who = "dsa_latent_cache_append";
  const int rc = check_cache(who, num_blocks, block_size, D_qk, D_v, dtype);
  if (rc) return rc;
  DSA_REQUIRE(T >= 0 && T < (1ll << 31), "%s: T=%lld out of range", who, (long long)T);
  if (T == 0) return DSA_OK;
  DSA_REQUIRE(cache && latent && rope && slots && aligned16(cache) && aligned16(latent) && aligned16(rope),
              "%s: null or misaligned pointer", who);
  DSA_REQUIRE(latent_stride >= 0 && rope_stride >= 0 && latent_stride % 8 == 0 && rope_stride % 8 == 0,
              "%s: row strides must be non-negative multiples of 8 elements", who);
  return launch_cache_append(cache, latent, latent_stride * 2, rope, rope_stride * 2, slots, T, num_blocks * block_size, D_qk,
                             dtype == DSA_DTYPE_MXFP4, (hipStream_t)stream);
}

extern "C" int dsa_latent_cache_gather(const void *cache, const int64_t *slots, void *out, int64_t T, int64_t num_blocks,
                                       int64_t block_size, int64_t D_qk, int64_t D_v, int dtype, void *stream) {
  const char *who = "dsa_latent_cache_gather";
  const int rc = check_cache(who, num_blocks, block_size, D_qk, D_v, dtype);
  if (rc) return rc;
  DSA_REQUIRE(T >= 0 && T < (1ll << 31), "%s: T=%lld out of range", who, (long long)T);
  if (T == 0) return DSA_OK;
  DSA_REQUIRE(cache && slots && out && aligned16(cache) && aligned16(out), "%s: null or misaligned pointer", who);
  return launch_cache_gather(cache, slots, out, T, num_blocks * block_size, D_qk, dtype == DSA_DTYPE_MXFP4, (hipStream_t)stream);
}

extern "C" int dsa_latent_plan_step(const int32_t *context_lens, const int32_t *query_lens, const int32_t *block_table,
                                    const int32_t *free_blocks, const int32_t *free_count, int32_t *block_table_out,
                                    int64_t *slots, int32_t *positions, int32_t *query_starts, int32_t *kv_lens,
                                    int32_t *context_lens_out, int32_t *granted, int32_t *free_blocks_out,
                                    int32_t *free_count_out, int64_t R, int64_t W, int64_t F, int64_t T, int64_t block_size,
                                    void *stream) {
  const char *who = "dsa_latent_plan_step";
  DSA_REQUIRE(R >= 0 && W > 0 && F > 0 && T >= 0 && block_size > 0 && block_size <= 65536, "%s: bad sizes", who);
  DSA_REQUIRE(R < (1 << 20) && W < (1ll << 30) && F < (1ll << 31) && T < (1ll << 31) && R * W < (1ll << 31) &&
                  W * block_size < (1ll << 31),
              "%s: sizes out of range (R < 2^20, R * W and W * block_size below 2^31)", who);
  DSA_REQUIRE(free_blocks && free_count && query_starts && free_blocks_out && free_count_out &&
                  (T == 0 || (slots && positions)) &&
                  (R == 0 || (context_lens && query_lens && block_table && block_table_out && kv_lens && context_lens_out && granted)),
              "%s: null pointer", who);
  const void *ins[] = {context_lens, query_lens, block_table, free_blocks, free_count};
  const void *outs[] = {block_table_out, slots, positions, query_starts, kv_lens, context_lens_out, granted, free_blocks_out,
                        free_count_out};
  for (const void *in : ins)
    for (const void *out : outs)
      DSA_REQUIRE(in == nullptr || in != out, "%s: an output is an input (the workgroups read the inputs while others write)", who);
  PlanParams p{context_lens, query_lens, block_table, free_blocks, free_count, slots, positions, query_starts, kv_lens,
               context_lens_out, granted, block_table_out, free_blocks_out, free_count_out, T, (int)R, (int)W, (int)F,
               (int)block_size, 0};
  return launch_latent_plan(p, (hipStream_t)stream);
}

static int check_paged(const char *who, int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk) {
  DSA_REQUIRE(T >= 0 && R >= 0 && W > 0 && H > 0, "%s: bad sizes T=%lld R=%lld W=%lld H=%lld", who, (long long)T, (long long)R,
              (long long)W, (long long)H);
  DSA_REQUIRE(H <= 4096 && R < (1 << 20) && T < (1ll << 30) && T * H < (1ll << 31) - 1024 && W < (1ll << 31) &&
                  W * block < (1ll << 31) - 1024,
              "%s: sizes out of range (H <= 4096, R < 2^20, T * H and W * block_size below 2^31 - 1024)", who);
  DSA_REQUIRE(T == 0 || R == 0 || paged_countable(T, R, W, block, H, d_qk),
              "%s: sizes out of range (row groups times key blocks must stay below 2^31)", who);
  return DSA_OK;
}

extern "C" size_t dsa_paged_latent_mla_workspace_size(int64_t T, int64_t R, int64_t W, int64_t block_size, int64_t H, int64_t D_qk,
                                                      int64_t D_v) {
  const char *who = "dsa_paged_latent_mla_workspace_size";
  if (check_cache(who, 1, block_size, D_qk, D_v, DSA_DTYPE_BF16) || check_paged(who, T, R, W, block_size, H, D_qk)) return 0;
  return T == 0 || R == 0 ? 0 : paged_workspace(T, R, W, block_size, H, D_qk, D_v);
}

extern "C" int dsa_paged_latent_mla_fwd(const void *q, const void *cache, const int32_t *block_table, const int32_t *query_starts,
                                        const int32_t *kv_lens, void *out, float *lse2, void *workspace, size_t workspace_bytes,
                                        int64_t T, int64_t R, int64_t W, int64_t H, int64_t D_qk, int64_t D_v, int64_t num_blocks,
                                        int64_t block_size, int dtype, float sm_scale, void *stream) {
  const char *who = "dsa_paged_latent_mla_fwd";
  int rc = check_cache(who, num_blocks, block_size, D_qk, D_v, dtype);
  if (!rc) rc = check_paged(who, T, R, W, block_size, H, D_qk);
  if (rc) return rc;
  DSA_REQUIRE(isfinite(sm_scale) && sm_scale >= 0x1p-100f, "%s: sm_scale must be finite and at least 2^-100, got %g", who, (double)sm_scale);
  if (T == 0 || R == 0) return DSA_OK;
  DSA_REQUIRE(q && cache && block_table && kv_lens && out && lse2 && aligned16(q) && aligned16(cache) && aligned16(out),
              "%s: null or misaligned pointer", who);
  const size_t need = paged_workspace(T, R, W, block_size, H, D_qk, D_v);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return set_error(DSA_ERR_WORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, got %zu", who, need, workspace_bytes);
  PagedParams p{};
  p.q = (const unsigned char *)q;
  p.cache = (const unsigned char *)cache;
  p.table = block_table;
  p.query_starts = query_starts;
  p.kv_lens = kv_lens;
  p.out = (uint16_t *)out;
  p.lse = lse2;
  p.T = T;
  p.R = (int)R;
  p.W = (int)W;
  p.H = (int)H;
  p.block = (int)block_size;
  p.block_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)block_size) : -1;
  p.num_blocks = (int)num_blocks;
  p.sl2 = sm_scale * kLog2e;
  return launch_paged_fwd(p, D_qk, D_v, dtype == DSA_DTYPE_MXFP4, (unsigned char *)workspace, (hipStream_t)stream);
}
