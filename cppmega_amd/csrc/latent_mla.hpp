// Dense latent attention (LatentMLA, absorbed and expanded forms): parameter
// block, row windows, and the LDS tiles its forward and backward share.
#pragma once

#include "dsa_common.hpp"
#include "sparse_mla_wide_tile.hpp"
#include "wave_ops.hpp"

namespace dsa {

// Rows are (token, head of the group) pairs in that order: row r of kv group g is
// token r / hpg, head g * hpg + r % hpg.  Absorbed: one kv row per token serves the
// hpg heads of a group, V its first D_v channels.  Expanded: hpg = 1, a group is a
// head; K = [k_nope of the head, k_pe of the token].
struct LatentParams {
  const unsigned char *q;              // [B, S, H, DK] bf16
  const unsigned char *k, *kpe, *v;    // bf16; kpe, v: expanded only
  int64_t k_b, k_t, k_g, pe_b, pe_t, v_b, v_t, v_g;  // strides in bytes: batch, token, group
  uint16_t *out, *out_lo;              // [B, S, H, DV]; what rounding took from out, or null
  float *lse;                          // [B, S, H]
  const int32_t *starts, *ends;        // [B, S] key windows, or null
  int64_t B, S, S_kv, H, G, rows;      // rows = S * hpg
  int hpg, causal;
  float sl2, scale;                    // sm_scale * log2(e), sm_scale
  // backward
  const unsigned char *o, *o_lo, *dO;  // (o_lo may be null)
  const float *lse_in;
  uint16_t *dq, *dk, *dkpe, *dv;       // absorbed: dk = dkv [B, S_kv, G, DK]
  float *stat;                         // [B * G][nt64][4][64]: -lse2 / sl2, -delta, lo, hi (int bits) of a row
  int32_t *info;                       // [B * G][2 nt64][4]: least lo, largest hi, largest lo, least hi of 32 rows
  int64_t nt64;                        // 64-row tiles of a (batch, group)
  float *part;                         // [nsplit][B * G][S_kv][width] partial sums of the key gradients
  int32_t *used;                       // [nsplit][B * G][key blocks]: a partial was written
  int nsplit, tiles_per_split, nkb;
  int64_t items;                       // key-major workgroups of a (batch, group)
};

constexpr int kKeyTile = 64;           // keys (or, in the key-major kernel, rows) of an LDS tile
constexpr uint32_t kTileRecords = 0x80000000u;  // a tile's resource: kMaskedOff lies past it, its rows below it
constexpr int kNoLo = 0x7fffffff;
constexpr float kLeastScale = 0x1p-100f;  // of sm_scale: the backward's lse2 / (sm_scale log2 e) stays finite

// Keys [lo, hi) of token t of batch b, within [0, S_kv); an empty row has lo = hi = 0.
__device__ __forceinline__ void latent_window(const LatentParams &p, int64_t b, int64_t t, int &lo, int &hi) {
  const int sk = (int)p.S_kv;
  lo = 0;
  hi = sk;
  if (p.starts != nullptr) {
    lo = p.starts[b * p.S + t];
    hi = p.ends[b * p.S + t];
    lo = lo > 0 ? lo : 0;
    hi = hi < sk ? hi : sk;
  } else if (p.causal) {
    const int64_t e = t + 1 + p.S_kv - p.S;
    hi = e < 0 ? 0 : (e < sk ? (int)e : sk);
  }
  if (hi <= lo) lo = hi = 0;
}

// Workgroups reach the XCDs in turn (blockIdx % 8).  Of n groups with `per` items each, item id's group and index:
// where the groups divide among the XCDs, a group's items stay on one (they share its tensors in that L2), group after
// group; else index after index, so that every XCD gets long and short ones alike.
__device__ __forceinline__ void spread_items(int64_t id, int64_t n, int64_t per, int64_t &group, int64_t &index) {
  if (n % 8 == 0) {
    const int64_t j = id >> 3, round = j / per;
    group = round * 8 + (id & 7);
    index = j - round * per;
  } else {
    index = id / n;
    group = id - index * n;
  }
}

// What a set of rows admits: the union [lo, hi) of their windows and the keys
// [lo_max, hi_min) that every one of them admits (none where a row is empty).
struct RowSpan {
  int lo, hi, lo_max, hi_min;
};
__device__ __forceinline__ RowSpan no_rows() { return RowSpan{kNoLo, 0, 0, kNoLo}; }
__device__ __forceinline__ void span_add(RowSpan &s, int lo, int hi) {
  const bool any = hi > lo;
  s.lo = min(s.lo, any ? lo : kNoLo);
  s.hi = max(s.hi, hi);
  s.lo_max = max(s.lo_max, any ? lo : kNoLo);
  s.hi_min = min(s.hi_min, hi);
}
// The span over all lanes (all values are non-negative: unsigned order is theirs).
__device__ __forceinline__ RowSpan span_wave(RowSpan s) {
  s.lo = (int)wv::wave_reduce((uint32_t)s.lo, wv::MinU());
  s.hi = (int)wv::wave_reduce((uint32_t)s.hi, wv::MaxU());
  s.lo_max = (int)wv::wave_reduce((uint32_t)s.lo_max, wv::MaxU());
  s.hi_min = (int)wv::wave_reduce((uint32_t)s.hi_min, wv::MinU());
  return s;
}

// A tile is 64 rows as two sub-tiles of 32, each stored by panels of 64 columns as
// DmaTile stores its 32 rows (chunk c of row r of a panel at tile_byte(r, c)).
// Fetch panels [P0, P0 + NP) of the NPT-panel tile at LDS byte address lds, the NW
// waves sharing the 8-row groups; off(row) is the byte offset of tile row `row` in
// rs (kMaskedOff: zeros).
template <int NPT, int P0, int NP, int NW, class Off>
__device__ __forceinline__ void tile_fetch(uint32_t lds, i32x4 rs, int w, Off off) {
  const int lane = lane_id();
#pragma unroll
  for (int i = 0; i < 8 / NW; ++i) {
    const int rg = w + NW * i, row = 8 * rg + (lane >> 3);
    const uint32_t src = off(row) + (uint32_t)(((lane & 7) ^ row_swz(row & 31)) * 16);
#pragma unroll
    for (int pn = 0; pn < NP; ++pn)
      lds_dma_16(lds + (uint32_t)((rg >> 2) * NPT * 4096 + (P0 + pn) * 4096 + (rg & 3) * 1024), src, rs, (uint32_t)(pn * 128));
  }
}

// 32x32x16 operand with the tile's rows as its M/N index: row l32, k-step ks (16 columns).
struct RowRead {
  int a[4];
  __device__ __forceinline__ RowRead() {
    const int lane = lane_id();
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = tile_byte(lane & 31, 2 * u + (lane >> 5));
  }
  __device__ __forceinline__ i32x4 operator()(const unsigned char *sub, int ks) const {
    return *reinterpret_cast<const i32x4 *>(sub + a[ks & 3] + (ks >> 2) * 4096);
  }
};

// 32x32x16 operand with the tile's columns as its M index and 16 of its rows as K:
// column tile dt (32 columns: chunk pairs 2 (dt & 1) and 2 (dt & 1) + 4 of panel
// dt / 2, which puts the rows of one read on distinct banks), rows 16 u .. 16 u + 15
// in accumulator order: element e = 4 h + j of lane half gg is row 16 u + 8 h + 4 gg + j.
struct ColRead {
  int a[2][2];  // [h][dt & 1]
  __device__ __forceinline__ ColRead() {
    const int lane = lane_id();
    const int k = lane & 15, j = k >> 2, q = k & 3, cb = (lane >> 4) & 1, gg = lane >> 5;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int odd = 0; odd < 2; ++odd)
        a[h][odd] = tile_byte(8 * h + 4 * gg + j, 2 * odd + 4 * cb + (q >> 1)) + (q & 1) * 8;
  }
  __device__ __forceinline__ i32x4 operator()(const unsigned char *sub, int dt, int u) const {
    const unsigned char *base = sub + (dt >> 1) * 4096 + u * 2048;
    const i32x2 r0 = ds_read_tr16(base + a[0][dt & 1]);
    const i32x2 r1 = ds_read_tr16(base + a[1][dt & 1]);
    return i32x4{r0[0], r0[1], r1[0], r1[1]};
  }
};
// Column of accumulator register i (0..15) of column tile dt; registers 4 m .. 4 m + 3 are consecutive columns.
__device__ __forceinline__ int acc_col(int dt, int i, int g32) {
  return (dt >> 1) * 64 + (dt & 1) * 16 + (i >> 3) * 32 + ((i >> 2) & 1) * 8 + 4 * g32 + (i & 3);
}
// Row (key) of accumulator register i within its 32.
__device__ __forceinline__ int acc_row(int i, int g32) { return 8 * (i >> 2) + 4 * g32 + (i & 3); }

// A 32x32 accumulator as the B operand of the next product: 16 of its rows per k-step.
__device__ __forceinline__ void pack_operand(const f32x16 &x, i32x4 (&b)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
    b[u] = i32x4{(int)pack_bf16x2(x[8 * u], x[8 * u + 1]), (int)pack_bf16x2(x[8 * u + 2], x[8 * u + 3]),
                 (int)pack_bf16x2(x[8 * u + 4], x[8 * u + 5]), (int)pack_bf16x2(x[8 * u + 6], x[8 * u + 7])};
}

// Keeps a wave-uniform branch a branch: what it holds is then not computed, and selected from, where it is not taken.
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// The operands of N products read from LDS, kGroup at a time, a group ahead of its use:
// use(i, operand) for i in order.  The first group was loaded by the caller (while
// something else ran); the barriers keep the compiler from sinking a load to its use.
constexpr int kGroup = 4;
template <int G>
struct OperandsOf {
  i32x4 x[G];
};
using Operands = OperandsOf<kGroup>;
template <int N, int G, class Load>
__device__ __forceinline__ void load_group(OperandsOf<G> &o, int g, Load load) {
#pragma unroll
  for (int i = 0; i < G; ++i)
    if (g * G + i < N) o.x[i] = load(g * G + i);
}
template <int N, int G, class Load, class Use>
__device__ __forceinline__ void stream_operands(const OperandsOf<G> &first, Load load, Use use) {
  constexpr int NG = (N + G - 1) / G;
  OperandsOf<G> cur = first;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    OperandsOf<G> nxt;
    if (g + 1 < NG) load_group<N>(nxt, g + 1, load);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < G; ++i)
      if (g * G + i < N) use(g * G + i, cur.x[i]);
    __builtin_amdgcn_sched_barrier(0);
    if (g + 1 < NG) cur = nxt;
  }
}

// Whether a lane of the workgroup's NW waves has x: by the first NW words of LDS at `words`, free before and after
// (__syncthreads_or takes 256 bytes of its own beside what a kernel asks for).
template <int NW>
__device__ __forceinline__ bool any_wave(bool x, unsigned char *words) {
  int *at = reinterpret_cast<int *>(words);
  const int mine = wv::ballot(x) != 0ull;
  if (lane_id() == 0) at[wave_id()] = mine;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) any |= at[i];
  __syncthreads();  // read: they may be written again
  return __builtin_amdgcn_readfirstlane(any) != 0;
}
constexpr int kLdsOfCu = 160 * 1024, kAnyBytes = 256;  // LDS of a CU; what __syncthreads_or takes of it

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
// Tile dt of a row per lane pair (l, l + 32) as bf16, v[m] its columns acc_col(dt, 4 m, l / 32) .. + 3 (m and m + 1: 16 that lie together):
// halves exchanged, so that a lane stores 16 bytes (8 at a time, the forward's results took a tenth of its time).
__device__ __forceinline__ void store_tile(uint16_t *row, int dt, const i32x2 (&v)[4], int g32) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const auto a = __builtin_amdgcn_permlane32_swap((uint32_t)v[2 * u][0], (uint32_t)v[2 * u + 1][0], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v[2 * u][1], (uint32_t)v[2 * u + 1][1], false, false);
    *reinterpret_cast<i32x4 *>(row + acc_col(dt, 8 * u, 0) + 8 * g32) = i32x4{(int)a[0], (int)b[0], (int)a[1], (int)b[1]};
  }
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// The product of one sub-tile without matrix instructions, for a tile in which some
// (row, column) pairs are masked and a masked one may hold Inf or NaN, which a weight
// of zero does not remove: acc[dt][column of lane] += x[row of sub] * sub[row][column]
// over the sub-tile rows r with admit(r).  Taken only by a workgroup whose first run
// left something that is not finite.
template <int NDT, class Admit>
__device__ __forceinline__ void careful_product(f32x16 (&acc)[NDT], const f32x16 &x, const unsigned char *sub, Admit admit) {
  const int g32 = lane_id() >> 5;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const float mine = x[i], other = xor32(mine);
#pragma unroll 1
    for (int hf = 0; hf < 2; ++hf) {
      const int r = 8 * (i >> 2) + 4 * hf + (i & 3);
      const float xv = g32 == hf ? mine : other;
      const bool ok = admit(r);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int a = 0; a < 16; ++a) {
          const int col = acc_col(dt, a, g32);
          const uint32_t raw =
              *reinterpret_cast<const uint16_t *>(sub + (col >> 6) * 4096 + tile_byte(r, (col & 63) >> 3) + (col & 7) * 2);
          const float t = fmaf(xv, bf16_bits_to_f32(raw), acc[dt][a]);
          acc[dt][a] = ok ? t : acc[dt][a];
          if ((a & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // few loads in flight: the registers are the fast path's
        }
    }
  }
}

// The resource of 64 keys from key0 and the offsets of their rows.
__device__ __forceinline__ i32x4 tile_rsrc(const unsigned char *base) { return make_buffer_words(base, kTileRecords); }

int launch_latent_fwd(const LatentParams &p, int64_t d_qk, int64_t d_v, bool expanded, hipStream_t st);
int launch_latent_bwd(const LatentParams &p, int64_t d_qk, int64_t d_v, bool expanded, unsigned char *ws, hipStream_t st);
size_t latent_bwd_workspace(LatentParams p, int64_t d_qk, int64_t d_v, bool expanded);  // (the sizes of p)

}  // namespace dsa
