// Parameter block of sparse attention over the paged latent cache.
#pragma once

#include "index_keys.hpp"

namespace dsa {

struct SparseParams {
  const unsigned char *q;          // [T, H, d_qk] bf16
  const unsigned char *cache;      // [num_blocks][block] rows
  const int32_t *indices, *table;  // [T, topk] positions, [R, W] pages
  Requests req;
  uint16_t *out;                   // [T, H, d_v]
  float *lse;                      // [T, H]
  int W, H, topk, block, block_shift, num_blocks;
  float sl2;
  int htiles, nsplit;              // head tiles of a token; workgroups that share a unit's picks
  float *part_o, *part_ml;         // their sums
  __device__ __forceinline__ int page_of(int pos) const {
    return block_shift >= 0 ? pos >> block_shift : (int)((uint32_t)pos / (uint32_t)block);
  }
};

size_t sparse_narrow_workspace(int64_t T, int64_t topk, int64_t H);
int launch_sparse_narrow(SparseParams p, bool fp4, unsigned char *ws, hipStream_t st);

}  // namespace dsa
