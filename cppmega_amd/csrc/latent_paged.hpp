// Parameter block of latent attention over a paged cache.
#pragma once

#include "dsa_common.hpp"
#include "latent_cache.hpp"

namespace dsa {

struct PagedParams {
  const unsigned char *q;        // [T, H, d_qk] bf16
  const unsigned char *cache;    // [num_blocks][block] rows
  const int32_t *table;          // [R, W] pages, others mask their keys
  const int32_t *query_starts;   // [R + 1] first token of every request, or null: one token each
  const int32_t *kv_lens;        // [R] keys of a request, its new tokens' among them
  uint16_t *out;                 // [T, H, d_v]
  float *lse;                    // [T, H]
  int64_t T;
  int R, W, H, block, num_blocks;
  float sl2;
  // plan and partial results
  int unit_rows, max_units, nwg;
  int32_t *unit0, *unit_req, *unit_first;
  int64_t *unit_at;
  float *part_ml, *part_o;       // [2 nwg][unit_rows]: (m, l), [d_v]
};

size_t paged_workspace(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v);
int launch_paged_fwd(PagedParams p, int64_t d_qk, int64_t d_v, bool fp4, unsigned char *ws, hipStream_t st);

}  // namespace dsa
