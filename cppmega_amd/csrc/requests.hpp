// The requests of a paged call and the picks of their tokens.
#pragma once

#include "dsa_common.hpp"
#include "wave_ops.hpp"

namespace dsa {

// Sums that stop at 2^32 - 1: starts that do not ascend may count a token many times over.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ uint32_t wave_scan_sat(uint32_t x) {  // wv::wave_incl_scan's steps
  x = add_sat(x, wv::dpp<0x111, 0xf, true>(x));
  x = add_sat(x, wv::dpp<0x112, 0xf, true>(x));
  x = add_sat(x, wv::dpp<0x114, 0xf, true>(x));
  x = add_sat(x, wv::dpp<0x118, 0xf, true>(x));
  x = add_sat(x, wv::dpp<0x142, 0xa>(x));
  x = add_sat(x, wv::dpp<0x143, 0xc>(x));
  return x;
}
// Exclusive prefix over the workgroup of one value below 2^31 per thread; total in every thread.  Exact below 2^32 - 1,
// at least 2^31 (the stop, less the thread's value) past it.
template <int NTHR>
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *tmp, uint32_t &total) {
  const int lane = lane_id(), w = (int)(threadIdx.x >> 6);
  const uint32_t v = wave_scan_sat(x);
  __syncthreads();
  if (lane == 63) tmp[w] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NTHR / 64; ++i) {
    const uint32_t t = tmp[i];
    if (i < w) before = add_sat(before, t);
    total = add_sat(total, t);
  }
  return add_sat(before, v) - x;
}

// Keys that token t of n new ones sees.
__device__ __forceinline__ int token_keys(int kv, int n, int t) { return max(kv - n + t + 1, 0); }

// The requests of a call: tokens query_starts[r] .. query_starts[r + 1] of the batch (null: token r alone) are the last of
// request r's kv_lens[r] positions.
struct Requests {
  const int32_t *query_starts, *kv_lens;
  int64_t cap;  // W * block: lengths past it are cut
  int T, R;
  __device__ __forceinline__ int start(int r) const { return query_starts == nullptr ? r : min(max(query_starts[r], 0), T); }
  __device__ __forceinline__ int tokens(int r) const {
    if (query_starts == nullptr) return r < T ? 1 : 0;
    const int n = start(r + 1) - start(r);
    return n > 0 ? n : 0;
  }
  __device__ __forceinline__ int kv(int r) const {
    const int k = kv_lens[r];
    return k < 0 ? 0 : (k < cap ? k : (int)cap);
  }
  // The last request that begins at or before token t (the whole wave: 64 of them are looked at in a step).
  __device__ __forceinline__ int of(int t) const {
    if (query_starts == nullptr) return t < R ? t : R - 1;
    const int lane = lane_id();
    int lo = 0, n = R;
    while (n > 1) {
      const int step = (n + 63) / 64, at = lo + lane * step;
      const uint64_t before = __builtin_amdgcn_ballot_w64(lane * step < n && start(at < R ? at : 0) <= t);
      const int k = before == 0 ? 0 : 63 - (int)__builtin_clzll(before);
      n = n - k * step < step ? n - k * step : step;
      lo += k * step;
    }
    return lo;
  }
  // The same, lane by lane.
  __device__ __forceinline__ int of_lane(int t) const {
    if (query_starts == nullptr) return t < R ? t : R - 1;
    int lo = 0, hi = R - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (start(mid) <= t) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
  // Positions that token t of request r sees, -1 where it is not one of the request's.
  __device__ __forceinline__ int keys_of(int t, int r) const {
    const int at = start(r), n = tokens(r);
    return t >= at && t < at + n ? token_keys(kv(r), n, t - at) : -1;
  }
};

// Positions [T, topk] that tokens attend to, and the pages that they lie on.
struct Picks {
  const int32_t *indices, *table;  // [T, topk], [R, W]
  Requests req;
  int W, topk, block, block_shift, num_blocks;
  __device__ __forceinline__ int page_of(int pos) const {
    return block_shift >= 0 ? pos >> block_shift : (int)((uint32_t)pos / (uint32_t)block);
  }
  // Pick i of token t, of `lim` positions (-1: none, or not among them).
  __device__ __forceinline__ int position(int64_t t, int i, int lim) const {
    const int pos = indices[t * topk + (i < topk ? i : topk - 1)];
    return i < topk && pos >= 0 && pos < lim ? pos : -1;
  }
  // Its entry of request r's table, and the cache slot that it makes (-1: none).
  __device__ __forceinline__ int entry(int r, int pos) const { return table[(int64_t)r * W + (pos > 0 ? page_of(pos) : 0)]; }
  __device__ __forceinline__ int slot(int pos, int e) const {
    return pos < 0 || e < 0 || e >= num_blocks ? -1 : e * block + (pos - page_of(pos) * block);
  }
};

}  // namespace dsa
