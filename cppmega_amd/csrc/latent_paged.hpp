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
  int block_shift;               // log2 of a page's rows, -1: no power of two
  float sl2;
  // plan and partial results
  int unit_rows, step_keys, max_units, nwg, min_blocks;  // rows of a unit, keys of a block of it
  int32_t *unit0, *unit_req, *unit_first;
  int32_t *unit_at;
  float *part_ml, *part_o;       // [2 nwg][unit_rows]: (m, l), [d_v]
};

static __device__ const i32x4 kZeroRow[80] = {};  // a masked key's row
// A load from p.cache, p.q or kZeroRow, chosen by a select: said to be global, since the compiler takes the choice for a flat
// address, whose loads are also counted as LDS operations, so that the next barrier waits for them.
__device__ __forceinline__ i32x4 ld_row_16(const unsigned char *x) {
  return *reinterpret_cast<const __attribute__((address_space(1))) i32x4 *>(reinterpret_cast<uint64_t>(x));
}
__device__ __forceinline__ uint32_t ld_row_1(const unsigned char *x) {
  return *reinterpret_cast<const __attribute__((address_space(1))) unsigned char *>(reinterpret_cast<uint64_t>(x));
}

__device__ __forceinline__ int request_start(const PagedParams &p, int r) {
  return p.query_starts == nullptr ? r : min(max(p.query_starts[r], 0), (int)p.T);
}
// new tokens of request r (within q's rows)
__device__ __forceinline__ int request_tokens(const PagedParams &p, int r) {
  if (p.query_starts == nullptr) return r < p.T ? 1 : 0;
  const int n = request_start(p, r + 1) - request_start(p, r);
  return n > 0 ? n : 0;
}
__device__ __forceinline__ int request_kv(const PagedParams &p, int r) {
  const int kv = p.kv_lens[r];
  const int64_t cap = (int64_t)p.W * p.block;
  return kv < 0 ? 0 : (kv < cap ? kv : (int)cap);
}
// keys that token t of n new ones sees
__device__ __forceinline__ int token_keys(int kv, int n, int t) { return max(kv - n + t + 1, 0); }

// Blocks of a workgroup's range: at least min_blocks, so that a piece is worth its prologue.
__device__ __forceinline__ int range_blocks(const PagedParams &p, int total) {
  const int per = (int)(((uint32_t)total + (uint32_t)p.nwg - 1u) / (uint32_t)p.nwg);
  return per > p.min_blocks ? per : p.min_blocks;
}
// A wave-uniform value as a scalar.
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A piece of a unit: blocks [b0, b1) of it, from a workgroup's range of all blocks.
struct PagedPiece {
  int b0, b1, first, n, kv, nrows, slot;  // first row within the request; partial result's place
  bool whole;                             // the unit entire
  int64_t row0;                           // first row in q, out and lse
  const int32_t *table;
};
// Piece at block `at` of unit u, for a range that ends at `end`; at moves past it.
__device__ __forceinline__ PagedPiece next_piece(const PagedParams &p, int u, int &at, int end) {
  const int ub = uni(p.unit_at[u]), ue = uni(p.unit_at[u + 1]), req = uni(p.unit_req[u]);
  PagedPiece x;
  x.b0 = at - ub;
  x.b1 = (ue < end ? ue : end) - ub;
  x.whole = x.b0 == 0 && ub + x.b1 == ue;
  x.slot = (int)blockIdx.x * 2 + (x.b0 == 0 ? 1 : 0);
  at = ub + x.b1;
  x.first = uni(p.unit_first[u]);
  x.n = uni(request_tokens(p, req));
  x.kv = uni(request_kv(p, req));
  x.nrows = min(x.n * p.H - x.first, p.unit_rows);
  x.row0 = (int64_t)uni(request_start(p, req)) * p.H + x.first;
  x.table = p.table + (int64_t)req * p.W;
  return x;
}

// The last unit that begins at or before block `at` (the whole wave: 64 units are looked at in a step).
__device__ __forceinline__ int unit_of(const PagedParams &p, int units, int at) {
  const int lane = lane_id();
  int lo = 0, n = units;  // it is one of lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 63) / 64, at_lane = lo + lane * step;
    const uint64_t before = __builtin_amdgcn_ballot_w64(lane * step < n && p.unit_at[at_lane < units ? at_lane : 0] <= at);
    const int k = (int)__builtin_popcountll(before) - 1;
    n = n - k * step < step ? n - k * step : step;
    lo += k * step;
  }
  return lo;
}

__device__ __forceinline__ void dma_16_at(uint32_t lds, const unsigned char *src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ const unsigned char *shfl_ptr(const unsigned char *x, int src) {
  const uint64_t v = reinterpret_cast<uint64_t>(x);
  const uint32_t a = (uint32_t)__shfl((int)(uint32_t)v, src, 64), b = (uint32_t)__shfl((int)(uint32_t)(v >> 32), src, 64);
  return reinterpret_cast<const unsigned char *>(((uint64_t)b << 32) | a);
}
// Table entry of key 32 j + (lane & 31) of a request with `lim` keys (-1: none), and the key's row (kZeroRow: none).
__device__ __forceinline__ int key_entry(const PagedParams &p, const int32_t *table, int j, int lim) {
  const int key = 32 * j + (lane_id() & 31);
  return key < lim ? table[(uint32_t)key / (uint32_t)p.block] : -1;
}
__device__ __forceinline__ const unsigned char *key_row(const PagedParams &p, int j, int entry, int row_bytes) {
  const uint32_t key = 32u * (uint32_t)j + (uint32_t)(lane_id() & 31);
  const int64_t slot = (int64_t)entry * p.block + (key - key / (uint32_t)p.block * (uint32_t)p.block);
  return entry >= 0 && entry < p.num_blocks ? p.cache + slot * row_bytes : reinterpret_cast<const unsigned char *>(kZeroRow);
}

constexpr int kWindow = 1024;  // table entries of a request that a workgroup has in LDS
// vmcnt(n) alone
constexpr int vmcnt_only(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }

int paged_wide_keys();  // keys of a step
int launch_paged_wide(const PagedParams &p, int tiles16, bool fp4, hipStream_t st);
int launch_paged_few(const PagedParams &p, bool fp4, hipStream_t st);

// The blocks of all units can be numbered in 32 bits, whatever the lengths.
bool paged_countable(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk);
size_t paged_workspace(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v);
int launch_paged_fwd(PagedParams p, int64_t d_qk, int64_t d_v, bool fp4, unsigned char *ws, hipStream_t st);

}  // namespace dsa
