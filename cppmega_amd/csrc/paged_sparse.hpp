// Parameter block of sparse attention over the paged latent cache, rows of 128 channels.
#pragma once

#include "requests.hpp"

namespace dsa {

struct SparseParams {
  const unsigned char *q;      // [T, H, d_qk] bf16
  const unsigned char *cache;  // [num_blocks][block] rows
  Picks picks;
  uint16_t *out;               // [T, H, d_v]
  float *lse;                  // [T, H]
  int H;
  float sl2;
  int htiles, nsplit;          // head tiles of a token; workgroups that share a unit's picks
  float *part_o, *part_ml;     // their sums
};

size_t sparse_narrow_workspace(int64_t T, int64_t topk, int64_t H);
int launch_sparse_narrow(SparseParams p, bool fp4, unsigned char *ws, hipStream_t st);

}  // namespace dsa
