// SparseMLA of new tokens over the paged latent cache, on gfx950: each token attends to the cached rows that its top-k
// names by their positions in its request.
//
// Positions become cache slots once a call (sparse_slots_kernel); a token is then a request of one token whose pages are
// single rows, and the kernels of paged latent attention take it: their workgroups share all tokens' picks evenly, 32 or 64
// at a time, whatever the number of tokens, and add the pieces of a token that was cut.
#include <math.h>

#include "index_keys.hpp"
#include "latent_paged.hpp"
#include "paged_sparse.hpp"

namespace dsa {

struct SparseSlotParams {
  const int32_t *indices, *table;  // [T, topk] positions, [R, W]
  Requests req;
  int32_t *slots, *picks;          // [T, topk]; [T] one past the last valid pick
  int32_t *unit0, *unit_req, *unit_first, *unit_at;
  int W, topk, block, block_shift, num_blocks;
  int H, units, unit_rows, unit_blocks;  // units of a token, their rows and blocks of keys
};

// A workgroup a token: its slots (-1: a position that it does not see, or on no page), and its units for the attention.
__global__ void __launch_bounds__(256) sparse_slots_kernel(const SparseSlotParams p) {
  __shared__ int last[4];
  const int t = (int)blockIdx.x, tid = (int)threadIdx.x, lane = lane_id(), w = wave_id();
  int r = 0, lim = -1;
  if (p.req.R > 0) {
    r = __builtin_amdgcn_readfirstlane(p.req.of(t));
    const int at = p.req.start(r), n = p.req.tokens(r);
    if (t >= at && t < at + n) lim = max(p.req.kv(r) - n + (t - at) + 1, 0);
  }
  const int32_t *idx = p.indices + (int64_t)t * p.topk, *table = p.table + (int64_t)r * p.W;
  int32_t *slots = p.slots + (int64_t)t * p.topk;
  int end = 0;
#pragma unroll 8
  for (int i = tid; i < p.topk; i += 256) {
    const int pos = idx[i];
    int slot = -1;
    if (pos >= 0 && pos < lim) {
      const int pg = p.block_shift >= 0 ? pos >> p.block_shift : (int)((uint32_t)pos / (uint32_t)p.block);
      const int e = table[pg];
      if (e >= 0 && e < p.num_blocks) {
        slot = e * p.block + (pos - pg * p.block);
        end = i + 1;
      }
    }
    slots[i] = slot;
  }
  for (int x = 32; x >= 1; x >>= 1) end = max(end, __shfl_xor(end, x, 64));
  if (lane == 0) last[w] = end;
  __syncthreads();
  end = max(max(last[0], last[1]), max(last[2], last[3]));
  if (tid == 0) {
    p.picks[t] = end;
    if (t == 0) p.unit0[p.req.T] = p.req.T * p.units;
    if (t + 1 == p.req.T) p.unit_at[p.req.T * p.units] = p.req.T * p.units * p.unit_blocks;
  }
  for (int i = tid; i < p.units; i += 256) {
    const int u = t * p.units + i;
    p.unit_req[u] = t;
    // (a token of no request: rows past its last, which are nobody's)
    p.unit_first[u] = lim < 0 ? p.H : i * p.unit_rows;
    p.unit_at[u] = u * p.unit_blocks;
  }
}

static size_t slots_at(int64_t T, int64_t topk, int64_t H, int64_t d_qk, int64_t d_v) {  // (256-byte aligned)
  return (paged_workspace(T, T, topk, 1, H, d_qk, d_v) + 255) & ~(size_t)255;
}
size_t paged_sparse_workspace(int64_t T, int64_t topk, int64_t H, int64_t d_qk, int64_t d_v) {
  if (d_qk == 128) return sparse_narrow_workspace(T, topk, H);
  return slots_at(T, topk, H, d_qk, d_v) + (size_t)T * ((size_t)topk + 1) * 4;
}

int launch_paged_sparse(const PagedParams &p, const int32_t *indices, int64_t topk, int64_t d_qk, int64_t d_v, bool fp4,
                        unsigned char *ws, hipStream_t st) {
  const Requests req{p.query_starts, p.kv_lens, (int64_t)p.W * p.block, (int)p.T, p.R};
  if (d_qk == 128) {
    SparseParams n{};
    n.q = p.q;
    n.cache = p.cache;
    n.indices = indices;
    n.table = p.table;
    n.req = req;
    n.out = p.out;
    n.lse = p.lse;
    n.W = p.W;
    n.H = p.H;
    n.topk = (int)topk;
    n.block = p.block;
    n.block_shift = p.block_shift;
    n.num_blocks = p.num_blocks;
    n.sl2 = p.sl2;
    return launch_sparse_narrow(n, fp4, ws, st);
  }
  int32_t *slots = (int32_t *)(ws + slots_at(p.T, topk, p.H, d_qk, d_v)), *picks = slots + p.T * topk;
  // every token a request of one token, its keys on pages of one row
  PagedParams a = p;
  a.table = slots;
  a.query_starts = nullptr;
  a.kv_lens = picks;
  a.R = (int)p.T;
  a.W = (int)topk;
  a.block = 1;
  a.block_shift = 0;
  a.num_blocks = p.num_blocks * p.block;
  paged_setup(a, d_qk, d_v, fp4, ws);
  SparseSlotParams s{};
  s.indices = indices;
  s.table = p.table;
  s.req = req;
  s.slots = slots;
  s.picks = picks;
  s.unit0 = a.unit0;
  s.unit_req = a.unit_req;
  s.unit_first = a.unit_first;
  s.unit_at = a.unit_at;
  s.W = p.W;
  s.topk = (int)topk;
  s.block = p.block;
  s.block_shift = p.block_shift;
  s.num_blocks = p.num_blocks;
  s.H = p.H;
  s.unit_rows = a.unit_rows;
  s.units = (p.H + a.unit_rows - 1) / a.unit_rows;
  s.unit_blocks = ((int)topk + a.step_keys - 1) / a.step_keys;
  hipLaunchKernelGGL(sparse_slots_kernel, dim3((unsigned)p.T), dim3(256), 0, st, s);
  const int rc = check_launch("dsa_paged_sparse_mla_fwd (slots)");
  return rc ? rc : launch_paged_units(a, d_qk, d_v, fp4, st);
}

}  // namespace dsa
