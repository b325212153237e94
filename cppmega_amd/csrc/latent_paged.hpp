// Parameter block of latent attention over a paged cache.
#pragma once

#include "dsa_common.hpp"
#include "latent_cache.hpp"
#include "requests.hpp"

namespace dsa {

struct PagedParams {
  const unsigned char *q;        // [T, H, d_qk] bf16
  const unsigned char *cache;    // [num_blocks][block] rows
  const int32_t *table;          // [R, W] pages, others mask their keys
  Requests req;                  // starts [R + 1] or null (one token each), lengths [R], a request's new tokens' keys among them
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
  // sparse attention: every token a request of its picks (block 1), in token_units units of unit_blocks blocks
  Picks picks;
  int token_units, unit_blocks;
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

// Blocks of a workgroup's range: at least min_blocks, so that a piece is worth its prologue.
__device__ __forceinline__ int range_blocks(const PagedParams &p, int total) {
  const int per = (int)(((uint32_t)total + (uint32_t)p.nwg - 1u) / (uint32_t)p.nwg);
  return per > p.min_blocks ? per : p.min_blocks;
}
// A wave-uniform value as a scalar.
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// All units and their blocks.
template <bool SPARSE>
__device__ __forceinline__ void all_units(const PagedParams &p, int &units, int &total) {
  if constexpr (SPARSE) {
    units = (int)p.T * p.token_units;
    total = units * p.unit_blocks;
  } else {
    units = uni(p.unit0[p.R]);
    total = uni(p.unit_at[units]);
  }
}
// First block of unit u.
template <bool SPARSE>
__device__ __forceinline__ int unit_begin(const PagedParams &p, int u) {
  if constexpr (SPARSE) return u * p.unit_blocks;
  else return uni(p.unit_at[u]);
}

// A piece of a unit: blocks [b0, b1) of it, from a workgroup's range of all blocks.
struct PagedPiece {
  int b0, b1, first, n, kv, nrows, slot;  // first row within the request; partial result's place
  bool whole;                             // the unit entire
  int64_t row0;                           // first row in q, out and lse
  const int32_t *table;
  int token, req, seen;                   // sparse: the token, its request and the positions that it sees
};
// The workgroup's place among the ranges of blocks.  Sparse: neighbouring ranges, which may be a token's units and read the
// same rows, on one XCD.
template <bool SPARSE>
__device__ __forceinline__ int range_of() {
  return SPARSE ? (int)xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;
}
// Piece at block `at` of unit u, for a range that ends at `end`; at moves past it.
template <bool SPARSE = false>
__device__ __forceinline__ PagedPiece next_piece(const PagedParams &p, int u, int &at, int end) {
  const int ub = unit_begin<SPARSE>(p, u), ue = unit_begin<SPARSE>(p, u + 1);
  PagedPiece x;
  x.b0 = at - ub;
  x.b1 = (ue < end ? ue : end) - ub;
  x.whole = x.b0 == 0 && ub + x.b1 == ue;
  x.slot = range_of<SPARSE>() * 2 + (x.b0 == 0 ? 1 : 0);
  at = ub + x.b1;
  if constexpr (SPARSE) {
    x.token = uni(u / p.token_units);
    x.req = uni(p.picks.req.of(x.token));
    x.seen = uni(p.picks.req.keys_of(x.token, x.req));
    x.first = (u - x.token * p.token_units) * p.unit_rows;
    x.n = 1;
    x.kv = x.seen < 0 ? 0 : p.picks.topk;
    x.nrows = x.seen < 0 ? 0 : min(p.H - x.first, p.unit_rows);  // (a token of no request: no rows)
    x.row0 = (int64_t)x.token * p.H + x.first;
    x.table = nullptr;
  } else {
    const int req = uni(p.unit_req[u]);
    x.first = uni(p.unit_first[u]);
    x.n = uni(p.req.tokens(req));
    x.kv = uni(p.req.kv(req));
    x.nrows = min(x.n * p.H - x.first, p.unit_rows);
    x.row0 = (int64_t)uni(p.req.start(req)) * p.H + x.first;
    x.table = p.table + (int64_t)req * p.W;
  }
  return x;
}

// The last unit that begins at or before block `at` (the whole wave: 64 units are looked at in a step).
template <bool SPARSE = false>
__device__ __forceinline__ int unit_of(const PagedParams &p, int units, int at) {
  if constexpr (SPARSE) return at / p.unit_blocks;
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
int launch_paged_wide(const PagedParams &p, int tiles16, bool fp4, bool sparse, hipStream_t st);
int launch_paged_few(const PagedParams &p, bool fp4, hipStream_t st);

// The blocks of all units can be numbered in 32 bits, whatever the lengths.
bool paged_countable(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk);
size_t paged_workspace(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v);
int launch_paged_fwd(PagedParams p, int64_t d_qk, int64_t d_v, bool fp4, unsigned char *ws, hipStream_t st);
int launch_paged_combine(const PagedParams &p, int64_t d_v, bool sparse, hipStream_t st);

// Attention over the cached rows that indices [T, topk] name by their positions in p.table's requests; p as for launch_paged_fwd.
bool paged_sparse_countable(int64_t T, int64_t topk, int64_t H, int64_t d_qk);
size_t paged_sparse_workspace(int64_t T, int64_t topk, int64_t H, int64_t d_qk, int64_t d_v);
int launch_paged_sparse(PagedParams p, const int32_t *indices, int64_t topk, int64_t d_qk, int64_t d_v, bool fp4,
                        unsigned char *ws, hipStream_t st);

}  // namespace dsa
