// Dense latent attention backward on gfx950 MFMA (bf16).  With p = 2^(sl2 q.k - lse2),
// delta = out . dO and ds = p (dO . v - delta) scale:
//   dq = sum_keys ds k     dk = sum_rows ds q     dv = sum_rows p dO
// (absorbed: dkv = dk + [dv, 0], summed over the group's heads, which are rows).
//
//   latent_bwd_q_kernel    row-major, as the forward: a wave keeps 32 rows of Q
//     and dO, S^T = K Q^T and dP^T = V dO^T leave one row per lane, dQ^T[d][row] +=
//     K^T dS^T.  It also leaves every row's lse2, delta * scale and window, and the
//     windows' spans per 32 rows, for the next kernel.
//   latent_bwd_kv_kernel   key-major: a wave keeps 32 keys of K (and V) and streams
//     LDS tiles of 64 rows of Q and dO: S = Q K^T and dP = dO V^T leave one key per
//     lane, dK^T[d][key] += Q^T dS, dV^T[d][key] += dO^T P (absorbed: into the same
//     accumulators).  Row tiles that no key of the workgroup is admitted by are passed
//     over.  Where (batch, group, key block) triples leave the GPU idle, the rows are
//     split over nsplit workgroups, whose fp32 partial sums
//   latent_bwd_reduce_kernel adds in split order (and k_pe's over the heads).
// No float atomics: the order of every sum follows from the shapes, so results repeat
// bit for bit.  P and dS are rounded to bf16 (nearest even) for the matrix products;
// sums are fp32.  Both kernels form S and dP (the reading and the rounding of a stored
// P and dS, 4 bytes a pair, would take longer than the two products).
//
// Bound by the MFMAs, with the exponentials and the packing of P and dS beside them.
// Causal, 4096 tokens: 128 / 64 absorbed, batch 2, 32 heads: rows 340 us (1010 TFLOP/s of
// its three products), keys 525 (785 of its four), reduction 17; 192 / 128 expanded, 128
// heads: 1325 (830), 1990 (690), 28.  The wider form has registers for one wave a SIMD, so
// that nothing runs beside its softmax.  delta is a sum over out: where out_lo is given,
// over out + out_lo, since the rounding of out alone shows in dq and dk of rows with few
// keys (packed documents: relative error 0.0026 against 0.0024).
#include <type_traits>

#include "latent_mla.hpp"

namespace dsa {

constexpr float kNoRow = 1.0e30f;  // in place of the lse2 of a row without weights: 2^(x - it) = 0

template <int DK, int DN, int DV, int RT, int NW>
struct LatentBwdQ {
  static constexpr bool SHARED = DN == DK;
  static constexpr int KP = DK / 64, NP = DN / 64, VP = DV / 64;
  static constexpr int K_BYTES = 2 * KP * 4096, V_BYTES = SHARED ? 0 : 2 * VP * 4096;
  static constexpr int BUF = K_BYTES + V_BYTES;
  static constexpr int ROWS = NW * RT * 32;
  static constexpr int OFF_SPAN = 2 * BUF;
  static constexpr int BYTES = OFF_SPAN + NW * 16 + 16;
};

template <int DK, int DN, int DV, int RT, int NW, int OCC>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC))) latent_bwd_q_kernel(const LatentParams p) {
  using C = LatentBwdQ<DK, DN, DV, RT, NW>;
  constexpr int KS = DK / 16, VS = DV / 16, NDT = DK / 32;
  static_assert(NW == 4 && OCC * (C::BYTES + kAnyBytes) <= kLdsOfCu, "a wave a SIMD and workgroup; LDS of all of them");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const int nblk = (int)((p.rows + C::ROWS - 1) / C::ROWS);
  int64_t bg, index;
  spread_items(blockIdx.x, p.B * p.G, nblk, bg, index);
  const int64_t b = bg / p.G, g = bg - b * p.G;
  const int blk = nblk - 1 - (int)index;
  int *span_lds = reinterpret_cast<int *>(smem + C::OFF_SPAN);

  int lo[RT], hi[RT];
  int64_t orow[RT];
  i32x4 q[RT][KS], dO[RT][VS];
  float lse[RT], delta[RT];  // delta * scale
  RowSpan span = no_rows();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int64_t row = (int64_t)blk * C::ROWS + (w * RT + rt) * 32 + l32;
    lo[rt] = hi[rt] = 0;
    orow[rt] = -1;
    RowSpan mine = no_rows();
    if (row < p.rows) {
      const int64_t t = (int64_t)((uint32_t)row / (uint32_t)p.hpg);
      orow[rt] = (b * p.S + t) * p.H + g * p.hpg + (row - t * p.hpg);
      latent_window(p, b, t, lo[rt], hi[rt]);
      span_add(mine, lo[rt], hi[rt]);
      span_add(span, lo[rt], hi[rt]);
    } else {
      span_add(mine, 0, 0);  // no row admits nothing: its weight 0 must not meet a key that is not finite
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[rt][ks] = i32x4{0, 0, 0, 0};
      if (orow[rt] >= 0) q[rt][ks] = ld_global_16(p.q + (orow[rt] * DK + 16 * ks + 8 * g32) * 2);
    }
    float dl = 0.0f;
#pragma unroll
    for (int vs = 0; vs < VS; ++vs) {
      dO[rt][vs] = i32x4{0, 0, 0, 0};
      if (orow[rt] >= 0) {
        dO[rt][vs] = ld_global_16(p.dO + (orow[rt] * DV + 16 * vs + 8 * g32) * 2);
        auto dot = [&](const unsigned char *o) {
          const i32x4 ov = ld_global_16(o + (orow[rt] * DV + 16 * vs + 8 * g32) * 2);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a = (uint32_t)ov[e], c = (uint32_t)dO[rt][vs][e];
            dl = fmaf(__uint_as_float(a << 16), __uint_as_float(c << 16), dl);
            dl = fmaf(__uint_as_float(a & 0xffff0000u), __uint_as_float(c & 0xffff0000u), dl);
          }
        };
        dot(p.o);
        if (p.o_lo != nullptr) dot(p.o_lo);
      }
    }
    // a row with weights: one without keys, or with scores of -Inf alone (lse2 -Inf), has no gradient
    const float lse_row = hi[rt] > lo[rt] ? p.lse_in[orow[rt]] : -INFINITY;
    const bool any = lse_row != -INFINITY;
    dl = sum_halves(dl);
    delta[rt] = any ? dl * p.scale : 0.0f;
    lse[rt] = any ? lse_row : kNoRow;
    // what the key-major kernel needs of these rows
    const int64_t r32 = (int64_t)blk * (C::ROWS / 32) + w * RT + rt, t64 = r32 >> 1;
    if (t64 < p.nt64) {
      const RowSpan s = span_wave(mine);
      float *st = p.stat + (bg * p.nt64 + t64) * 256 + (r32 & 1) * 32 + l32;
      if (g32 == 0) {
        st[0] = -lse[rt] / p.sl2;
        st[64] = any ? -dl : 0.0f;
      } else {
        st[128] = __int_as_float(lo[rt]);
        st[192] = __int_as_float(hi[rt]);
      }
      if (lane == 0) *reinterpret_cast<i32x4 *>(p.info + (bg * p.nt64 * 2 + r32) * 4) = i32x4{s.lo, s.hi, s.lo_max, s.hi_min};
    }
  }
  span = span_wave(span);
  if (lane == 0) {
    span_lds[2 * w] = span.lo;
    span_lds[2 * w + 1] = span.hi;
  }
  __syncthreads();
  int klo = kNoLo, khi = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    klo = min(klo, span_lds[2 * i]);
    khi = max(khi, span_lds[2 * i + 1]);
  }
  klo = __builtin_amdgcn_readfirstlane(klo);
  khi = __builtin_amdgcn_readfirstlane(khi);
  const int t0 = khi > klo ? klo / kKeyTile : 0, t1 = khi > klo ? (khi + kKeyTile - 1) / kKeyTile : 0;

  const uint32_t lds0 = lds_address(smem);
  const unsigned char *kb = p.k + b * p.k_b + g * p.k_g;
  auto fetch = [&](int tile, int buf) {
    const int64_t k0 = (int64_t)tile * kKeyTile;
    const int n = (int)(p.S_kv - k0 < kKeyTile ? p.S_kv - k0 : kKeyTile);
    const uint32_t at = lds0 + (uint32_t)(buf * C::BUF);
    const uint32_t kt = (uint32_t)p.k_t;
    tile_fetch<C::KP, 0, C::NP, NW>(at, tile_rsrc(kb + k0 * p.k_t), w,
                                    [&](int r) { return r < n ? (uint32_t)r * kt : kMaskedOff; });
    if constexpr (!C::SHARED) {
      const uint32_t pt = (uint32_t)p.pe_t, vt = (uint32_t)p.v_t;
      tile_fetch<C::KP, C::NP, C::KP - C::NP, NW>(at, tile_rsrc(p.kpe + b * p.pe_b + k0 * p.pe_t), w,
                                                  [&](int r) { return r < n ? (uint32_t)r * pt : kMaskedOff; });
      tile_fetch<C::VP, 0, C::VP, NW>(at + C::K_BYTES, tile_rsrc(p.v + b * p.v_b + g * p.v_g + k0 * p.v_t), w,
                                      [&](int r) { return r < n ? (uint32_t)r * vt : kMaskedOff; });
    }
  };

  const RowRead row_read;
  const ColRead col_read;
  f32x16 acc[RT][NDT];
  auto pass = [&](auto careful_t) {
    constexpr bool careful = decltype(careful_t)::value;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc[rt][dt] = zero16();
    if (t0 < t1) fetch(t0, 0);
    for (int tile = t0; tile < t1; ++tile) {
      const int buf = (tile - t0) & 1, k0 = tile * kKeyTile;
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's share of the tile
      __syncthreads();
      if (tile + 1 < t1) fetch(tile + 1, buf ^ 1);
      const unsigned char *Kt = smem + buf * C::BUF, *Vt = C::SHARED ? Kt : Kt + C::K_BYTES;
      if (k0 >= span.hi || k0 + kKeyTile <= span.lo) continue;  // wave-uniform
      // operands 0 .. KS - 1: K; absorbed: the first VS of them V too; expanded: V after them
      constexpr int NR = C::SHARED ? KS : KS + VS;
      auto rows_of = [&](int sub) {
        return [=](int i) { return i < KS ? row_read(Kt + sub * C::KP * 4096, i) : row_read(Vt + sub * C::VP * 4096, i - KS); };
      };
      Operands ka;
      load_group<NR>(ka, 0, rows_of(0));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int ks0 = k0 + 32 * s;
        const bool whole = span.lo_max <= ks0 && span.hi_min >= ks0 + 32;
        const unsigned char *Ks = Kt + s * C::KP * 4096;
        auto cols = [&](int i) { return col_read(Ks, i >> 1, i & 1); };
        f32x16 sc[RT], dp[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt] = dp[rt] = zero16();
        stream_operands<NR>(ka, rows_of(s), [&](int i, i32x4 a) {
          const int vs = C::SHARED ? i : i - KS;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if (i < KS)
              sc[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(q[rt][i < KS ? i : 0]), sc[rt], 0, 0, 0);
            if (vs >= 0 && vs < VS)
              dp[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(dO[rt][vs >= 0 && vs < VS ? vs : 0]), dp[rt], 0, 0, 0);
          }
        });
        // in flight beside the softmax: the first operands of its product with K, and of the next keys
        Operands ca;
        load_group<2 * NDT>(ca, 0, cols);
        if (s == 0) load_group<NR>(ka, 0, rows_of(1));
        __builtin_amdgcn_sched_barrier(0);
        i32x4 db[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[rt][i] = exp2_fast(fmaf(sc[rt][i], p.sl2, -lse[rt])) * fmaf(dp[rt][i], p.scale, -delta[rt]);
          if (!whole) {
            keep_branch();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = ks0 + acc_row(i, g32);
              sc[rt][i] = key >= lo[rt] && key < hi[rt] ? sc[rt][i] : 0.0f;
            }
          }
          pack_operand(sc[rt], db[rt]);
        }
        if (!careful || whole) {
          stream_operands<2 * NDT>(ca, cols, [&](int i, i32x4 a) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              acc[rt][i >> 1] =
                  __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(db[rt][i & 1]), acc[rt][i >> 1], 0, 0, 0);
          });
        } else {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            careful_product<NDT>(acc[rt], sc[rt], Ks, [&](int r) { return ks0 + r >= lo[rt] && ks0 + r < hi[rt]; });
        }
      }
    }
    __syncthreads();  // the buffers are free again
  };
  pass(std::false_type{});
  bool bad = false;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) bad |= not_finite(acc[rt][dt][i]);
  if (__syncthreads_or(bad)) pass(std::true_type{});  // a masked Inf or NaN may have reached a row: once more, without it
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
    if (orow[rt] >= 0) {
      const bool empty = lse[rt] == kNoRow;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const f32x16 &x = acc[rt][dt];
        i32x2 v[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          v[m] = i32x2{(int)pack_bf16x2(x[4 * m], x[4 * m + 1]), (int)pack_bf16x2(x[4 * m + 2], x[4 * m + 3])};
          if (empty) v[m] = i32x2{0, 0};
        }
        store_tile(p.dq + orow[rt] * DK, dt, v, g32);
      }
    }
}

// Key blocks that the rows of a split reach: all, or up to its last token's under the causal mask.
__host__ __device__ inline int split_blocks(const LatentParams &p, int split, int keys) {
  if (!p.causal || p.nsplit == 1) return p.nkb;  // unsplit: every key block is written, if with zeros
  const int64_t row1 = (int64_t)(split + 1) * p.tiles_per_split * 64, end = row1 < p.rows ? row1 : p.rows;
  const int64_t key1 = (end + p.hpg - 1) / p.hpg + p.S_kv - p.S;  // one past the last key
  const int64_t n = key1 <= 0 ? 0 : (key1 + keys - 1) / keys;
  return (int)(n < p.nkb ? n : p.nkb);
}

template <int DK, int DN, int DV, int CT, int NW>
struct LatentBwdKv {
  static constexpr bool SHARED = DN == DK;
  static constexpr int KP = DK / 64, VP = DV / 64;
  static constexpr int Q_BYTES = 2 * KP * 4096, D_BYTES = 2 * VP * 4096;
  static constexpr int OFF_STAT = Q_BYTES + D_BYTES;
  static constexpr int BUF = OFF_STAT + 1024;
  static constexpr int KEYS = NW * CT * 32;
  static constexpr int BYTES = 2 * BUF;
  // columns of a partial row: absorbed DK; expanded, split: [k_nope, k_pe, v]; expanded, unsplit: k_pe
  static constexpr int WIDE = SHARED ? DK : DK + DV;
};

template <int DK, int DN, int DV, int CT, int NW, int OCC>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC))) latent_bwd_kv_kernel(const LatentParams p) {
  using C = LatentBwdKv<DK, DN, DV, CT, NW>;
  constexpr int KS = DK / 16, VS = DV / 16, NDK = DK / 32, NDV = DV / 32;
  static_assert(NW == 4 && OCC * (C::BYTES + kAnyBytes) <= kLdsOfCu, "a wave a SIMD and workgroup; LDS of all of them");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  // Unsplit: by spread_items (windows leave key blocks that follow each other alike in length).  Else item -> (batch and
  // group, row split, key block): the splits from the last (the causal mask's with most key blocks), each with the key
  // blocks that its rows reach; consecutive items, which share rows, on one XCD.
  int64_t bg, index;
  int split = 0;
  if (p.nsplit == 1) {
    if ((int64_t)blockIdx.x >= p.B * p.G * p.items) return;
    spread_items(blockIdx.x, p.B * p.G, p.items, bg, index);
  } else {
    const int64_t item = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    bg = item / p.items;
    index = item - bg * p.items;
    if (bg >= p.B * p.G) return;
    split = p.nsplit - 1;
  }
  const int64_t b = bg / p.G, g = bg - b * p.G;
  int kblk = (int)index;
  for (int n = split_blocks(p, split, C::KEYS); kblk >= n; n = split_blocks(p, split, C::KEYS)) {
    kblk -= n;
    --split;
  }
  const int key_lo = kblk * C::KEYS, key_hi = key_lo + C::KEYS < p.S_kv ? key_lo + C::KEYS : (int)p.S_kv;
  const int wkey = key_lo + w * CT * 32;  // this wave's first key

  int key[CT];
  i32x4 kr[CT][KS], vr[C::SHARED ? 1 : CT][VS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    key[ct] = wkey + ct * 32 + l32;
    const bool in = key[ct] < p.S_kv;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kr[ct][ks] = i32x4{0, 0, 0, 0};
      if (in) {
        const int64_t kk = key[ct];
        kr[ct][ks] = ks < DN / 16 ? ld_global_16(p.k + b * p.k_b + kk * p.k_t + g * p.k_g + (16 * ks + 8 * g32) * 2)
                                  : ld_global_16(p.kpe + b * p.pe_b + kk * p.pe_t + (16 * (ks - DN / 16) + 8 * g32) * 2);
      }
    }
    if constexpr (!C::SHARED) {
#pragma unroll
      for (int vs = 0; vs < VS; ++vs) {
        vr[ct][vs] = i32x4{0, 0, 0, 0};
        if (in) vr[ct][vs] = ld_global_16(p.v + b * p.v_b + (int64_t)key[ct] * p.v_t + g * p.v_g + (16 * vs + 8 * g32) * 2);
      }
    }
  }

  // the next row tile at or after t (below c1) that a key of this workgroup is admitted by
  const int32_t *info = p.info + bg * p.nt64 * 8;
  const int c0 = split * p.tiles_per_split;
  const int c1 = c0 + p.tiles_per_split < p.nt64 ? c0 + p.tiles_per_split : (int)p.nt64;
  int hits_at = 0;       // tiles hits_at .. + 63 that do: bit by bit
  uint64_t hits = 0;
  auto scan = [&](int t) {
    bool hit = false;
    if (t + lane < c1) {
      const i32x4 a = *reinterpret_cast<const i32x4 *>(info + (int64_t)(t + lane) * 8);
      const i32x4 c = *reinterpret_cast<const i32x4 *>(info + (int64_t)(t + lane) * 8 + 4);
      hit = (a[0] < key_hi && a[1] > key_lo) || (c[0] < key_hi && c[1] > key_lo);
    }
    hits_at = t;
    hits = wv::ballot(hit);
  };
  auto next = [&](int t) {  // t in [hits_at, hits_at + 64]
    while (t < c1) {
      if (t >= hits_at + 64) scan(t);
      const uint64_t m = hits >> (t - hits_at);
      if (m != 0ull) return t + (int)__builtin_ctzll(m);
      t = hits_at + 64;
    }
    return c1;
  };
  // the two spans of a row tile, read a tile ahead
  struct Spans {
    i32x4 s[2];
  };
  auto spans = [&](int t) {
    const int tt = t < c1 ? t : c1 - 1;  // (a tile there is: c0 < c1 wherever this is asked)
    return Spans{*reinterpret_cast<const i32x4 *>(info + (int64_t)tt * 8), *reinterpret_cast<const i32x4 *>(info + (int64_t)tt * 8 + 4)};
  };

  const uint32_t lds0 = lds_address(smem);
  const uint32_t hpg = (uint32_t)p.hpg;
  auto fetch = [&](int tile, int buf) {
    const uint32_t at = lds0 + (uint32_t)(buf * C::BUF);
    const int64_t r0 = (int64_t)tile * 64, tok0 = (int64_t)((uint32_t)r0 / hpg);
    const uint32_t h0 = (uint32_t)(r0 - tok0 * p.hpg);
    const int n = (int)(p.rows - r0 < 64 ? p.rows - r0 : 64);
    const int64_t base = (b * p.S + tok0) * p.H + g * p.hpg;  // row (token tok0, first head)
    const uint32_t H = (uint32_t)p.H;
    auto at_row = [&](int r) {  // rows from base: tokens tok0 .. (one group: they lie together; one head a group: a token apart)
      const uint32_t x = h0 + (uint32_t)r;
      if (hpg == H) return x;
      if (hpg == 1) return x * H;
      const uint32_t dt = x / hpg;
      return dt * H + (x - dt * hpg);
    };
    tile_fetch<C::KP, 0, C::KP, NW>(at, tile_rsrc(p.q + base * DK * 2), w,
                                    [&](int r) { return r < n ? at_row(r) * (DK * 2) : kMaskedOff; });
    tile_fetch<C::VP, 0, C::VP, NW>(at + C::Q_BYTES, tile_rsrc(p.dO + base * DV * 2), w,
                                    [&](int r) { return r < n ? at_row(r) * (DV * 2) : kMaskedOff; });
    if (w == 0)
      lds_dma_16(at + C::OFF_STAT, (uint32_t)lane * 16, tile_rsrc(reinterpret_cast<const unsigned char *>(p.stat + (bg * p.nt64 + tile) * 256)), 0);
  };

  const RowRead row_read;
  const ColRead col_read;
  f32x16 dk[CT][NDK], dv[C::SHARED ? 1 : CT][NDV];
  scan(c0);
  const int first = next(c0);
  auto pass = [&](auto careful_t) {
    constexpr bool careful = decltype(careful_t)::value;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int dt = 0; dt < NDK; ++dt) dk[ct][dt] = zero16();
      if constexpr (!C::SHARED) {
#pragma unroll
        for (int dt = 0; dt < NDV; ++dt) dv[ct][dt] = zero16();
      }
    }
    int tile = first, buf = 0;
    Spans now{}, then{};
    if (careful) scan(c0);
    if (tile < c1) {
      fetch(tile, 0);
      now = spans(tile);
    }
    while (tile < c1) {
      const int nxt = next(tile + 1);
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's share of the tile
      __syncthreads();
      if (nxt < c1) fetch(nxt, buf ^ 1);
      then = spans(nxt);
      const unsigned char *Qt = smem + buf * C::BUF, *Dt = Qt + C::Q_BYTES;
      const float *st = reinterpret_cast<const float *>(Qt + C::OFF_STAT);
      // operands 0 .. KS - 1: Q, then the VS of dO
      auto rows_of = [&](int sub) {
        return [=](int i) { return i < KS ? row_read(Qt + sub * C::KP * 4096, i) : row_read(Dt + sub * C::VP * 4096, i - KS); };
      };
      // the accumulators begin at -lse2 / sl2 and -delta of their rows
      f32x16 sc[CT], dp[CT];
      auto begin = [&](int sub) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int r = 32 * sub + 8 * m + 4 * g32;  // registers 4 m .. are rows r ..
          const f32x4 ls = *reinterpret_cast<const f32x4 *>(st + r), de = *reinterpret_cast<const f32x4 *>(st + 64 + r);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sc[ct][4 * m + e] = ls[e];
              dp[ct][4 * m + e] = de[e];
            }
        }
      };
      OperandsOf<3> qa;  // (four at a time: 4% more at two waves a SIMD, whose registers they fill)
      load_group<KS + VS>(qa, 0, rows_of(0));
      begin(0);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bool whole = __builtin_amdgcn_readfirstlane(now.s[s][2]) <= wkey &&
                           __builtin_amdgcn_readfirstlane(now.s[s][3]) >= wkey + CT * 32;
        const unsigned char *Qs = Qt + s * C::KP * 4096, *Ds = Dt + s * C::VP * 4096;
        // operands 0 .. 2 NDV - 1: dO^T, then the 2 NDK of Q^T
        auto cols = [&](int i) { return i < 2 * NDV ? col_read(Ds, i >> 1, i & 1) : col_read(Qs, (i - 2 * NDV) >> 1, i & 1); };
        stream_operands<KS + VS>(qa, rows_of(s), [&](int i, i32x4 a) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            if (i < KS) {
              sc[ct] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(kr[ct][i < KS ? i : 0]), sc[ct], 0, 0, 0);
            } else {
              const i32x4 &bv = C::SHARED ? kr[ct][i < KS ? 0 : i - KS] : vr[C::SHARED ? 0 : ct][i < KS ? 0 : i - KS];
              dp[ct] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(bv), dp[ct], 0, 0, 0);
            }
          }
        });
        // in flight beside the softmax: the first operands of its products, and of the next rows
        OperandsOf<3> ca;
        load_group<2 * NDV + 2 * NDK>(ca, 0, cols);
        if (s == 0) load_group<KS + VS>(qa, 0, rows_of(1));
        __builtin_amdgcn_sched_barrier(0);
        i32x4 pb[CT][2], db[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            sc[ct][i] = exp2_fast(sc[ct][i] * p.sl2);
            dp[ct][i] *= sc[ct][i] * p.scale;
          }
        if (!whole) {
          keep_branch();
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const int r = 32 * s + 8 * m + 4 * g32;
            const i32x4 lo = *reinterpret_cast<const i32x4 *>(st + 128 + r), hi = *reinterpret_cast<const i32x4 *>(st + 192 + r);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool ok = key[ct] >= lo[e] && key[ct] < hi[e];
                sc[ct][4 * m + e] = ok ? sc[ct][4 * m + e] : 0.0f;
                dp[ct][4 * m + e] = ok ? dp[ct][4 * m + e] : 0.0f;
              }
          }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          pack_operand(sc[ct], pb[ct]);
          pack_operand(dp[ct], db[ct]);
        }
        if (!careful || whole) {
          if (s == 0) begin(1);
          stream_operands<2 * NDV + 2 * NDK>(ca, cols, [&](int i, i32x4 a) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              const int j = i < 2 * NDV ? 0 : (i - 2 * NDV) >> 1, jv = i < 2 * NDV ? i >> 1 : 0;
              if (i < 2 * NDV) {
                f32x16 &t = C::SHARED ? dk[ct][jv] : dv[C::SHARED ? 0 : ct][jv];
                t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(pb[ct][i & 1]), t, 0, 0, 0);
              } else {
                dk[ct][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(db[ct][i & 1]), dk[ct][j], 0, 0, 0);
              }
            }
          });
        } else {
          const int *sti = reinterpret_cast<const int *>(st);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            auto admit = [&](int r) { return key[ct] >= sti[128 + 32 * s + r] && key[ct] < sti[192 + 32 * s + r]; };
            if constexpr (C::SHARED) {
              f32x16 part[NDV];
#pragma unroll
              for (int dt = 0; dt < NDV; ++dt) part[dt] = dk[ct][dt];
              careful_product<NDV>(part, sc[ct], Ds, admit);
#pragma unroll
              for (int dt = 0; dt < NDV; ++dt) dk[ct][dt] = part[dt];
            } else {
              careful_product<NDV>(dv[C::SHARED ? 0 : ct], sc[ct], Ds, admit);
            }
            careful_product<NDK>(dk[ct], dp[ct], Qs, admit);
          }
          if (s == 0) begin(1);
        }
      }
      tile = nxt;
      now = then;
      buf ^= 1;
    }
    __syncthreads();
  };
  pass(std::false_type{});
  bool bad = false;
  {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int dt = 0; dt < NDK; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) bad |= not_finite(dk[ct][dt][i]);
      if constexpr (!C::SHARED) {
#pragma unroll
        for (int dt = 0; dt < NDV; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) bad |= not_finite(dv[ct][dt][i]);
      }
    }
  }
  if (__syncthreads_or(bad)) pass(std::true_type{});

  const int64_t bgs = p.B * p.G;
  const bool split_rows = p.nsplit > 1;
  if (split_rows && threadIdx.x == 0) p.used[((int64_t)split * bgs + bg) * p.nkb + kblk] = first < c1;
  if (split_rows && first >= c1) return;
  const int width = split_rows ? C::WIDE : 64;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (key[ct] >= p.S_kv) continue;
    float *row = p.part + (((int64_t)split * bgs + bg) * p.S_kv + key[ct]) * width;
    auto put = [&](const f32x16 &x, int dt, uint16_t *out, float *part) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int col = acc_col(dt, 4 * m, g32);
        if (out != nullptr)
          *reinterpret_cast<i32x2 *>(out + col) =
              i32x2{(int)pack_bf16x2(x[4 * m], x[4 * m + 1]), (int)pack_bf16x2(x[4 * m + 2], x[4 * m + 3])};
        else
          *reinterpret_cast<f32x4 *>(part + col) = f32x4{x[4 * m], x[4 * m + 1], x[4 * m + 2], x[4 * m + 3]};
      }
    };
    const int64_t orow = (b * p.S_kv + key[ct]) * p.G + g;
#pragma unroll
    for (int dt = 0; dt < NDK; ++dt) {
      if (dt * 32 < DN)
        put(dk[ct][dt], dt, split_rows ? nullptr : p.dk + orow * DN, row);
      else  // k_pe: summed over the heads by the reduction
        put(dk[ct][dt], dt, nullptr, split_rows ? row : row - DN);
    }
    if constexpr (!C::SHARED) {
#pragma unroll
      for (int dt = 0; dt < NDV; ++dt) put(dv[ct][dt], dt, split_rows ? nullptr : p.dv + orow * DV, row + DK);
    }
  }
}

// 2^lg threads per 4 columns, each a run of the terms: partial rows in split order (k_pe: group by group, each group's
// splits in order), then the threads' sums in order, rounded once.
struct LatentReduce {
  int keys, width, dn, dr, dvw, lg;  // keys of a block; width of a partial row: dn + dr + dvw, or dr
};
__global__ void __launch_bounds__(256) latent_bwd_reduce_kernel(const LatentParams p, const LatentReduce r) {
  __shared__ f32x4 sums[256];
  const int64_t bgs = p.B * p.G;
  const int own = (r.width - r.dr) / 4;  // columns of the group's own rows
  const int64_t n_own = bgs * p.S_kv * own, n_pe = p.B * p.S_kv * (r.dr / 4);
  const int items = 256 >> r.lg, part = (int)threadIdx.x >> (8 - r.lg);
  const int64_t id = (int64_t)blockIdx.x * items + ((int)threadIdx.x & (items - 1));
  f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
  // groups bg .. bg + n - 1, each with its splits: the flags of eight terms are read together, then what they say is there
  auto add = [&](int64_t bg, int64_t n, int64_t key, int col) {
    constexpr int kTerms = 8;
    const int kb = (int)((uint32_t)key / (uint32_t)r.keys);
    const int terms = (int)n * p.nsplit, per = (terms + (1 << r.lg) - 1) >> r.lg;
    const int end = min(terms, (part + 1) * per);
    int gr = part * per / p.nsplit, s = part * per - gr * p.nsplit;
    for (int i0 = part * per; i0 < end; i0 += kTerms) {
      int64_t at[kTerms];  // row s * bgs + group of the partial sums
      int there[kTerms];
#pragma unroll
      for (int i = 0; i < kTerms; ++i) {
        const bool in = i0 + i < end;
        at[i] = in ? s * bgs + bg + gr : bg;
        there[i] = in && (p.nsplit == 1 || kb < split_blocks(p, s, r.keys)) ? (p.nsplit == 1 ? 1 : p.used[at[i] * p.nkb + kb]) : 0;
        if (in && ++s == p.nsplit) {
          s = 0;
          ++gr;
        }
      }
      f32x4 x[kTerms];
#pragma unroll
      for (int i = 0; i < kTerms; ++i) {
        x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (there[i]) x[i] = *reinterpret_cast<const f32x4 *>(p.part + (at[i] * p.S_kv + key) * r.width + col);
      }
#pragma unroll
      for (int i = 0; i < kTerms; ++i) sum += x[i];
    }
  };
  uint16_t *dst = nullptr;
  if (id < n_own) {
    const int64_t row = id / own, bg = row / p.S_kv, key = row - bg * p.S_kv;
    const int c = (int)(id - row * own) * 4;
    const int64_t b = bg / p.G, orow = (b * p.S_kv + key) * p.G + (bg - b * p.G);
    const bool is_k = c < r.dn;
    add(bg, 1, key, is_k ? c : c + r.dr);
    dst = is_k ? p.dk + orow * r.dn + c : p.dv + orow * r.dvw + (c - r.dn);
  } else if (id < n_own + n_pe) {
    const int64_t x = id - n_own, row = x / (r.dr / 4), b = row / p.S_kv, key = row - b * p.S_kv;
    const int c = (int)(x - row * (r.dr / 4)) * 4;
    add(b * p.G, p.G, key, (r.width == r.dr ? 0 : r.dn) + c);
    dst = p.dkpe + (b * p.S_kv + key) * r.dr + c;
  }
  if (r.lg > 0) {
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (part > 0) return;
    for (int i = 1; i < 1 << r.lg; ++i) sum += sums[threadIdx.x + i * items];
  }
  if (dst != nullptr) *reinterpret_cast<i32x2 *>(dst) = i32x2{(int)pack_bf16x2(sum[0], sum[1]), (int)pack_bf16x2(sum[2], sum[3])};
}

// Waves per SIMD of the key-major kernel: two where its 32 keys a wave and their gradients leave the registers for it.
constexpr int kv_waves(int64_t d_qk, bool expanded) { return !expanded && d_qk == 128 ? 2 : 1; }

// Row splits of the key-major kernel: what takes least of the rounds of its workgroups on the card (1.3 us a row tile,
// 8 tiles' time for a workgroup's beginning and end) and of the partial sums' way to memory and back.
struct BwdKvPlan {
  int keys, nkb, nsplit, tiles_per_split, width;
  int64_t items;  // workgroups of a (batch, group)
};
static BwdKvPlan kv_plan(LatentParams p, int64_t d_qk, int64_t d_v, bool expanded) {
  BwdKvPlan r{};
  r.keys = 4 * 32;
  p.nkb = r.nkb = (int)((p.S_kv + r.keys - 1) / r.keys);
  const int64_t tiles = (p.rows + 63) / 64, bgs = p.B * p.G, slots = kv_waves(d_qk, expanded) * 256;
  const double row_us = (double)(bgs * p.S_kv * (expanded ? d_qk + d_v : d_qk)) * 8 / 4.9e6 * (p.causal ? 0.5 : 1.0);
  double least = 0;
  for (int64_t n = 1; n <= 64 && (n == 1 || n * 4 <= tiles); ++n) {
    p.tiles_per_split = tiles > 0 ? (int)((tiles + n - 1) / n) : 1;
    p.nsplit = tiles > 0 ? (int)((tiles + p.tiles_per_split - 1) / p.tiles_per_split) : 1;
    int64_t items = 0;
    for (int s = 0; s < p.nsplit; ++s) items += split_blocks(p, s, r.keys);
    const double us = (double)((bgs * items + slots - 1) / slots) * 1.3 * (double)(p.tiles_per_split + 8) +
                      (p.nsplit > 1 ? 6.0 + row_us * (double)p.nsplit : 0.0);
    if (n == 1 || us < least) {
      least = us;
      r.nsplit = p.nsplit;
      r.tiles_per_split = p.tiles_per_split;
      r.items = items;
    }
  }
  r.width = expanded ? (r.nsplit > 1 ? (int)(d_qk + d_v) : 64) : (int)d_qk;
  return r;
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
struct BwdSections {
  size_t stat, info, used, part, total;
};
static BwdSections bwd_sections(const BwdKvPlan &k, const LatentParams &p, bool expanded) {
  const size_t nt64 = (size_t)((p.rows + 63) / 64), bgs = (size_t)(p.B * p.G);
  BwdSections s;
  s.stat = 0;
  s.info = s.stat + bgs * nt64 * 1024;
  s.used = s.info + up256(bgs * nt64 * 32);
  s.part = s.used + (k.nsplit > 1 ? up256((size_t)k.nsplit * bgs * (size_t)k.nkb * 4) : 0);
  s.total = s.part + (k.nsplit > 1 || expanded ? (size_t)k.nsplit * bgs * (size_t)p.S_kv * (size_t)k.width * 4 : 0);
  return s;
}
size_t latent_bwd_workspace(LatentParams p, int64_t d_qk, int64_t d_v, bool expanded) {
  // the larger of the two masks' plans: the query does not know the mask
  size_t most = 0;
  for (p.causal = 0; p.causal < 2; ++p.causal) {
    const size_t n = bwd_sections(kv_plan(p, d_qk, d_v, expanded), p, expanded).total;
    most = n > most ? n : most;
  }
  return most;
}

template <int DK, int DN, int DV, int RT, int OQ>
static int launch(LatentParams p, unsigned char *ws, hipStream_t st) {
  constexpr int NW = 4, CT = 1, OK = kv_waves(DK, DN != DK);
  using Q = LatentBwdQ<DK, DN, DV, RT, NW>;
  using K = LatentBwdKv<DK, DN, DV, CT, NW>;
  constexpr bool expanded = DN != DK;
  const BwdKvPlan k = kv_plan(p, DK, DV, expanded);
  const BwdSections s = bwd_sections(k, p, expanded);
  p.nt64 = (p.rows + 63) / 64;
  p.stat = reinterpret_cast<float *>(ws + s.stat);
  p.info = reinterpret_cast<int32_t *>(ws + s.info);
  p.used = reinterpret_cast<int32_t *>(ws + s.used);
  p.part = reinterpret_cast<float *>(ws + s.part);
  p.nsplit = k.nsplit;
  p.tiles_per_split = k.tiles_per_split;
  p.nkb = k.nkb;
  p.items = k.items;
  const auto qk = latent_bwd_q_kernel<DK, DN, DV, RT, NW, OQ>;
  const auto kk = latent_bwd_kv_kernel<DK, DN, DV, CT, NW, OK>;
  hipError_t e = hipFuncSetAttribute((const void *)qk, hipFuncAttributeMaxDynamicSharedMemorySize, Q::BYTES);
  if (e == hipSuccess) e = hipFuncSetAttribute((const void *)kk, hipFuncAttributeMaxDynamicSharedMemorySize, K::BYTES);
  if (e != hipSuccess) return set_error(DSA_ERR_HIP, "dsa_latent_mla_bwd: LDS attribute: %s", hipGetErrorString(e));
  const int64_t bgs = p.B * p.G;
  const int64_t nq = (p.rows + Q::ROWS - 1) / Q::ROWS * bgs, nk = (k.items * bgs + 7) / 8 * 8;
  DSA_REQUIRE(nq < (1ll << 31) && nk < (1ll << 31), "dsa_latent_mla_bwd: grid too large");
  int rc = DSA_OK;
  if (nq > 0) {  // no rows: the key gradients below are zeros
    hipLaunchKernelGGL(qk, dim3((unsigned)nq), dim3(64 * NW), Q::BYTES, st, p);
    rc = check_launch("dsa_latent_mla_bwd (rows)");
  }
  if (rc || nk == 0) return rc;
  hipLaunchKernelGGL(kk, dim3((unsigned)nk), dim3(64 * NW), K::BYTES, st, p);
  rc = check_launch("dsa_latent_mla_bwd (keys)");
  if (rc || (!expanded && k.nsplit == 1)) return rc;
  // threads of an output: one for every eight terms, up to eight (32 splits of 512 rows: 18 us with one, 6.6 with four; where
  // rows are many, one and two are alike)
  LatentReduce r{k.keys, k.width, DN, DK - DN, expanded ? DV : 0, 0};
  const int64_t terms = k.nsplit > 1 ? k.nsplit : p.G;
  while (r.lg < 3 && (8 << r.lg) < terms) ++r.lg;
  const int64_t n = bgs * p.S_kv * ((r.width - r.dr) / 4) + p.B * p.S_kv * (r.dr / 4), wgs = (n + (256 >> r.lg) - 1) / (256 >> r.lg);
  DSA_REQUIRE(wgs < (1ll << 31), "dsa_latent_mla_bwd: grid too large");
  hipLaunchKernelGGL(latent_bwd_reduce_kernel, dim3((unsigned)wgs), dim3(256), 0, st, p, r);
  return check_launch("dsa_latent_mla_bwd (reduction)");
}

int launch_latent_bwd(const LatentParams &p, int64_t d_qk, int64_t d_v, bool expanded, unsigned char *ws, hipStream_t st) {
  if (!expanded) {
    if (d_qk == 128 && d_v == 64) return launch<128, 128, 64, 1, 2>(p, ws, st);
    if (d_qk == 128 && d_v == 128) return launch<128, 128, 128, 1, 2>(p, ws, st);
    if (d_qk == 192 && d_v == 128) return launch<192, 192, 128, 1, 1>(p, ws, st);
  } else {
    if (d_qk == 192 && d_v == 128) return launch<192, 128, 128, 1, 1>(p, ws, st);
    if (d_qk == 128 && d_v == 64) return launch<128, 64, 64, 1, 2>(p, ws, st);
  }
  return set_error(DSA_ERR_UNSUPPORTED, "dsa_latent_mla_bwd: no %s kernel for d_qk=%lld d_v=%lld",
                   expanded ? "expanded" : "absorbed", (long long)d_qk, (long long)d_v);
}

}  // namespace dsa
