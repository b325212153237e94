// Latent attention over a paged cache, rows of 128 channels (64 latent), for units of 16
// rows: bound by reading the cache, so nothing is shared that would make a wave wait for
// another.
//
// The four waves of a workgroup take the unit's 32-key blocks in turn, each in its own
// LDS tile, with the rows' Q and O in its registers:
//   S^T[key][row] = K Q^T    on 16x16x32 MFMAs (lane = row, 8 of the keys)
//   running maximum and sum per lane (two exchanges a block), P^T the operand as it stands
//   O^T[d][row] += V^T P^T   (V^T by transposed reads of the tile)
// No barrier until a piece's end, where the waves' O are brought to one maximum and added
// through LDS in wave order.  A wave's next rows are asked for while the others compute,
// of three workgroups a CU: bf16 rows by LDS-DMA loads, MXFP4 rows into registers a block
// ahead, converted when the tile is free.
// 64 requests of 301 .. 16384 keys, 16 heads, joining and plan included: 40 us for 137 MB
// in bf16 (3.4 TB/s), 37 us for 94 MB in MXFP4.
#include "latent_paged.hpp"
#include "sparse_mla_wide_tile.hpp"
#include "wave_ops.hpp"

namespace dsa {

template <bool FP4>
struct PagedFew {
  static constexpr int D_QK = 128, D_V = 64;
  using Row = CacheRow<D_QK, D_V, FP4>;
  static constexpr int NW = 4, ROWS = 16;
  static constexpr int KS = D_QK / 32, NDT = D_V / 16;    // k-steps, 16-channel tiles of O
  static constexpr int PANELS = D_QK / 64, TILE = PANELS * 4096;
  static constexpr int O_ROW = D_V + 4;                   // floats of an O row in LDS
  static constexpr int NB = D_V / 32;                     // 32-channel blocks of a row
  static constexpr int CPL = NB / 2;                      // 16-byte pieces of codes per lane
  static constexpr int OFF_ML = NW * TILE;                // [NW][ROWS][2]
  static constexpr int BYTES = OFF_ML + NW * ROWS * 8;
  static_assert(ROWS * O_ROW * 4 <= TILE, "a wave's O over its tile");
};

template <bool FP4>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) paged_few_kernel(const PagedParams p) {
  using C = PagedFew<FP4>;
  using Row = typename C::Row;
  constexpr int D_QK = C::D_QK, D_V = C::D_V;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = lane_id(), w = wave_id(), g16 = lane >> 4, l16 = lane & 15;
  unsigned char *K = smem + w * C::TILE;
  float *ML = reinterpret_cast<float *>(smem + C::OFF_ML);
  const uint32_t k_lds = lds_address(K);
  const unsigned char *zero = reinterpret_cast<const unsigned char *>(kZeroRow);
  // MXFP4: chunks are also permuted by their panel, as neighbouring lanes write one row's blocks, a panel to two of them
  auto panel_swz = [](int panel) { return FP4 ? (panel & 7) << 4 : 0; };
  // operand rows: key 8 (m >> 2) + 4 h + (m & 3) is row m of S^T's tile h, so that lane group g16 holds keys 8 g16 + 4 h + i
  int ka[2][2], va[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int u = 0; u < 2; ++u) ka[h][u] = tile_byte(8 * (l16 >> 2) + 4 * h + (l16 & 3), 4 * u + g16);
#pragma unroll
    for (int u = 0; u < 4; ++u) va[h][u] = tile_byte(8 * g16 + 4 * h + (l16 >> 2), 2 * u + ((l16 & 3) >> 1)) + (l16 & 1) * 8;
  }

  const int units = uni(p.unit0[p.R]), total = uni(p.unit_at[units]), per = uni(range_blocks(p, total));
  if ((int64_t)blockIdx.x * per >= total) return;
  int at = (int)blockIdx.x * per;
  const int end = per < total - at ? at + per : total;
  for (int u = uni(unit_of(p, units, at)); at < end; ++u) {
    const PagedPiece x = next_piece(p, u, at, end);
    const int b0 = x.b0, b1 = x.b1, first = x.first, n = x.n, kv = x.kv, nrows = x.nrows;
    const bool whole_unit = x.whole;
    const int64_t piece = x.slot, row0 = x.row0;
    const int tok0 = first / p.H, tok1 = (first + nrows - 1) / p.H;
    const int32_t *table = x.table;

    i32x4 q[C::KS];
    const unsigned char *src = (l16 < nrows ? p.q + (row0 + l16) * D_QK * 2 : zero) + 16 * g16;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) q[ks] = ld_row_16(src + 64 * ks);

    // Tokens [ta, tb] with the keys cut at tb's: all at once, or, where that left something that is not finite, one by
    // one, since a weight of zero does not remove the Inf or NaN of a later token's key.
    int ta = tok0, tb = tok1;
    bool probe = tok0 != tok1;
    while (true) {
      const int lim = token_keys(kv, n, tb), lim_min = token_keys(kv, n, ta);
      const int j1 = min(b1, (lim + 31) / 32);
      const int my_lim = token_keys(kv, n, min((first + l16) / p.H, tb));
      float m_run = kLeastMax, l_run = 0.0f;
      f32x4 o[C::NDT];
#pragma unroll
      for (int dt = 0; dt < C::NDT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      // MXFP4, a block ahead in registers: code pieces (row, blk), their rows' exponent bytes, the rope part
      i32x4 codes[FP4 ? C::CPL : 1], rope[FP4 ? 4 : 1];
      uint32_t expo[FP4 ? C::CPL : 1];
      auto load_raw = [&](const unsigned char *mine) {
        if constexpr (FP4) {
          // piece x: row x (64 / NB) + lane / NB, block lane % NB: a row's codes from neighbouring lanes
#pragma unroll
          for (int x = 0; x < C::CPL; ++x) {
            const unsigned char *src = shfl_ptr(mine, x * (64 / C::NB) + lane / C::NB);
            codes[x] = ld_row_16(src + (lane % C::NB) * 16);
            expo[x] = ld_row_1(src + Row::OFF_EXP + lane % C::NB);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) rope[i] = ld_row_16(shfl_ptr(mine, 8 * i + (lane >> 3)) + Row::OFF_ROPE + (lane & 7) * 16);
        }
      };
      auto put_block = [&](int row, int blk, i32x4 c, uint32_t e) {  // 32 channels of a row
        const float s = e8m0_scale(e);
        unsigned char *dst = K + (blk >> 1) * 4096;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          i32x4 v = e2m1x8_to_bf16((uint32_t)c[x], s);
          if (e == 255u) v = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
          *reinterpret_cast<i32x4 *>(dst + (tile_byte(row, 4 * (blk & 1) + x) ^ panel_swz(blk >> 1))) = v;
        }
      };
      auto put_raw = [&] {
        if constexpr (FP4) {
#pragma unroll
          for (int x = 0; x < C::CPL; ++x) put_block(x * (64 / C::NB) + lane / C::NB, lane % C::NB, codes[x], expo[x]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<i32x4 *>(K + (D_V / 64) * 4096 + (tile_byte(8 * i + (lane >> 3), lane & 7) ^ panel_swz(D_V / 64))) = rope[i];
        }
      };
      auto fetch = [&](const unsigned char *mine) {  // bf16
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
          const int row = 8 * rg + (lane >> 3);
          const unsigned char *src = shfl_ptr(mine, row) + ((lane & 7) ^ row_swz(row)) * 16;
#pragma unroll
          for (int pn = 0; pn < C::PANELS; ++pn) dma_16_at(k_lds + (uint32_t)(pn * 4096 + rg * 1024), src + pn * 128);
        }
      };

      int j = b0 + w;
      const unsigned char *mine = key_row(p, j, key_entry(p, table, j, lim), Row::BYTES);
      int e_nxt = key_entry(p, table, j + C::NW, lim);
      if (FP4 && j < j1) load_raw(mine);
      for (; j < j1; j += C::NW) {
        const uint32_t vm = (uint32_t)wv::ballot(mine != zero);
        if constexpr (FP4) put_raw(); else fetch(mine);
        mine = key_row(p, j + C::NW, e_nxt, Row::BYTES);
        e_nxt = key_entry(p, table, j + 2 * C::NW, lim);
        if constexpr (FP4) {
          load_raw(mine);  // (past the last block: zeros)
          wave_lds_sync();
        } else {
          __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the tile
          wave_lds_sync();
        }
        f32x4 s[2]{{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int ks = 0; ks < C::KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const i32x4 a = *reinterpret_cast<const i32x4 *>(K + (ka[h][ks & 1] ^ panel_swz(ks >> 1)) + (ks >> 1) * 4096);
            s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(q[ks]), s[h], 0, 0, 0);
          }
        if (vm != 0xffffffffu || 32 * j + 32 > lim_min) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = 8 * g16 + 4 * h + i;
              if (!((vm >> k) & 1u) || 32 * j + k >= my_lim) s[h][i] = -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = max_halves(mx) * p.sl2;
        if (wv::ballot(mx > m_run + 8.0f) != 0ull) {
          const float m_new = fmaxf(m_run, mx), alpha = exp2_fast(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int dt = 0; dt < C::NDT; ++dt) o[dt] *= alpha;
        }
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t[i] = exp2_fast(fmaf(s[i >> 2][i & 3], p.sl2, -m_run));
          l_run += t[i];
        }
        const i32x4 pb{(int)pack_bf16x2(t[0], t[1]), (int)pack_bf16x2(t[2], t[3]), (int)pack_bf16x2(t[4], t[5]),
                       (int)pack_bf16x2(t[6], t[7])};
#pragma unroll
        for (int dt = 0; dt < C::NDT; ++dt) {
          const i32x2 r0 = ds_read_tr16(K + (va[0][dt & 3] ^ panel_swz(dt >> 2)) + (dt >> 2) * 4096);
          const i32x2 r1 = ds_read_tr16(K + (va[1][dt & 3] ^ panel_swz(dt >> 2)) + (dt >> 2) * 4096);
          const i32x4 a{r0[0], r0[1], r1[0], r1[1]};
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(pb), o[dt], 0, 0, 0);
        }
        wave_lds_sync();  // the tile is read: it may be written again
      }

      if (probe) {
        bool bad = false;
#pragma unroll
        for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= (__float_as_uint(o[dt][e]) & 0x7f800000u) == 0x7f800000u;
        if (__syncthreads_or(bad)) {
          probe = false;
          ta = tb = tok0;
          continue;
        }
      }
      // the waves' sums, by row
      l_run += __shfl_xor(l_run, 16, 64);
      l_run = sum_halves(l_run);
      if (g16 == 0) {
        ML[(w * C::ROWS + l16) * 2] = m_run;
        ML[(w * C::ROWS + l16) * 2 + 1] = l_run;
      }
      const int rlo = ta * p.H - first, rhi = min((tb + 1) * p.H - first, nrows);  // rows of tokens [ta, tb]
      float *mine_o = reinterpret_cast<float *>(K);
#pragma unroll
      for (int dt = 0; dt < C::NDT; ++dt) *reinterpret_cast<f32x4 *>(mine_o + l16 * C::O_ROW + dt * 16 + 4 * g16) = o[dt];
      __syncthreads();  // every wave's O tile and sums
      constexpr int QUADS = C::ROWS * D_V / 4;
      for (int x = (int)threadIdx.x; x < QUADS; x += 256) {
        const int ur = x / (D_V / 4), d = (x - ur * (D_V / 4)) * 4;
        if (ur < rlo || ur >= rhi) continue;
        float m = kLeastMax, l = 0.0f;
#pragma unroll
        for (int k = 0; k < C::NW; ++k)
          if (ML[(k * C::ROWS + ur) * 2 + 1] != 0.0f) m = fmaxf(m, ML[(k * C::ROWS + ur) * 2]);
        f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < C::NW; ++k) {
          const float lk = ML[(k * C::ROWS + ur) * 2 + 1];
          if (lk == 0.0f) continue;  // the wave saw no key of the row (a NaN sum joins)
          const float a = exp2_fast(ML[(k * C::ROWS + ur) * 2] - m);
          l += lk * a;
          sum += a * *reinterpret_cast<const f32x4 *>(smem + k * C::TILE + (ur * C::O_ROW + d) * 4);
        }
        if (whole_unit) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          *reinterpret_cast<i32x2 *>(p.out + (row0 + ur) * D_V + d) =
              i32x2{(int)pack_bf16x2(sum[0] * inv, sum[1] * inv), (int)pack_bf16x2(sum[2] * inv, sum[3] * inv)};
          if (d == 0) p.lse[row0 + ur] = l == 0.0f ? -INFINITY : log2f(l) + m;
        } else {
          if (l != 0.0f) *reinterpret_cast<f32x4 *>(p.part_o + (piece * C::ROWS + ur) * D_V + d) = sum;
          if (d == 0) {
            p.part_ml[(piece * C::ROWS + ur) * 2] = m;
            p.part_ml[(piece * C::ROWS + ur) * 2 + 1] = l;
          }
        }
      }
      __syncthreads();  // read: the tiles may be written again
      if (tb == tok1) break;
      ta = ++tb;
    }
  }
}

template <bool FP4>
static int launch(const PagedParams &p, hipStream_t st) {
  using C = PagedFew<FP4>;
  static_assert(C::BYTES <= 64 * 1024, "LDS of an ordinary launch");
  hipLaunchKernelGGL((paged_few_kernel<FP4>), dim3((unsigned)p.nwg), dim3(256), C::BYTES, st, p);
  return check_launch("dsa_paged_latent_mla_fwd");
}

int launch_paged_few(const PagedParams &p, bool fp4, hipStream_t st) {
  return fp4 ? launch<true>(p, st) : launch<false>(p, st);
}

}  // namespace dsa
