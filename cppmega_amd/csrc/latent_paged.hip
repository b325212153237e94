// Latent attention over a paged cache on gfx950 (absorbed form, bf16 or MXFP4 rows):
// decoding, speculative tokens and prefill chunks of ragged requests.
//
// A request's rows are its (new token, head) pairs in that order; a unit is up to 128 of
// them with the keys 0 .. of its last token.  The units' blocks of keys, one after the
// other, are split evenly over the grid's workgroups (stream-wise, so a long request is
// shared and short ones are packed), whose ends may fall inside a unit: such a piece
// leaves its unnormalised fp32 O, maximum and sum, and paged_combine_kernel adds a unit's
// pieces in order.  The plan (units and their first blocks) is made on the device from
// the lengths: the host knows neither.
//
// Three kernels take the units: latent_paged_wide.hip rows of 576 channels,
// latent_paged_few.hip few rows of 128, paged_rows_kernel below many.  Keys past a
// request's last, and keys whose table entry is no page, read as zeros and have no weight.
#include "latent_mla.hpp"
#include "latent_paged.hpp"

namespace dsa {

// blocks of a unit (at least one: a unit without keys still writes its rows)
__device__ __forceinline__ int unit_blocks(const PagedParams &p, int kv, int n, int first, int rows, int unit_rows) {
  const int last = min(first + unit_rows, rows) - 1;
  return max((token_keys(kv, n, last / p.H) + p.step_keys - 1) / p.step_keys, 1);
}

// The plan, one workgroup: unit_req[u], unit_first[u] (first row), unit_at[u] (first block,
// unit_at[units] = all), unit0[r] (first unit of request r; unit0[R] = all).
__global__ void __launch_bounds__(1024) paged_plan_kernel(const PagedParams p) {
  __shared__ uint32_t tmp[16];
  const uint32_t most = (uint32_t)p.max_units;
  uint32_t total, at = 0;
  for (int r0 = 0; r0 < p.R; r0 += 1024) {
    const int r = r0 + (int)threadIdx.x;
    // (starts that do not ascend may ask for more units than there are: cut)
    const int n = r < p.R ? min((p.req.tokens(r) * p.H + p.unit_rows - 1) / p.unit_rows, p.max_units) : 0;
    const uint32_t x = add_sat(at, block_scan<1024>((uint32_t)n, tmp, total));
    if (r < p.R) p.unit0[r] = (int)min(x, most);
    at = min(add_sat(at, total), most);
  }
  const int units = (int)at;
  if (threadIdx.x == 0) p.unit0[p.R] = units;
  __syncthreads();
  at = 0;
  for (int u0 = 0; u0 < units; u0 += 1024) {
    const int u = u0 + (int)threadIdx.x;
    int nb = 0;
    if (u < units) {
      int lo = 0, hi = p.R - 1;  // the last request whose first unit is at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.unit0[mid] <= u) lo = mid; else hi = mid - 1;
      }
      const int first = (u - p.unit0[lo]) * p.unit_rows, n = p.req.tokens(lo);
      nb = unit_blocks(p, p.req.kv(lo), n, first, n * p.H, p.unit_rows);
      p.unit_req[u] = lo;
      p.unit_first[u] = first;
    }
    const uint32_t x = at + block_scan<1024>((uint32_t)nb, tmp, total);  // (all of them below 2^31: paged_countable)
    if (u < units) p.unit_at[u] = (int)x;
    at += total;
  }
  if (threadIdx.x == 0) p.unit_at[units] = (int)at;
}

// Many rows of 128 channels: four waves, NT of them 32 rows each, by 4 / NT key groups; steps of 64 keys, two ahead of
// the one that is worked on, shared by the waves in three LDS buffers, one barrier a step; three workgroups a CU.
//   S^T = K Q^T, O^T += V^T P^T on 32x32x16 MFMAs, lane = row.
// Bound by the MFMAs and the softmax beside them: prefill of 6 requests, 40 .. 512 tokens each on 1024 .. 4096 keys, 32
// heads, MXFP4: 83 us, 430 TFLOP/s (two workgroups a CU: 112).  Widening the codes costs a sixth (decode of 128 heads: 76 us
// against 64 in bf16).
template <int NT, bool FP4>
struct Paged {
  static constexpr int D_QK = 128, D_V = 64;
  using Row = CacheRow<D_QK, D_V, FP4>;
  static constexpr int NW = 4, KG = NW / NT, ROWS = 32 * NT;  // waves: NT row tiles x KG key groups
  static constexpr int TILES = 2, SUB = TILES / KG, KEYS = 32 * TILES;  // 32-key tiles of a step, of a wave; keys of a step
  static constexpr int NBUF = 3, AHEAD = NBUF - 1;            // steps in LDS, fetched ahead
  static constexpr int KS = D_QK / 16, NDT = D_V / 32;
  static constexpr int PANELS = D_QK / 64, TILE = PANELS * 4096, STEP = TILES * TILE;
  static constexpr int DMA = TILES * PANELS;                  // bf16: loads of a wave per step (an 8-row group a tile)
  static constexpr int NB = D_V / 32, CODES = KEYS * NB;      // MXFP4: code pieces of a row, of a step (one to a thread)
  static constexpr int OFF_T = NBUF * STEP;                   // table entries, then words of any_wave
  static constexpr int WINDOW = 1024 - 16, OFF_ANY = OFF_T + WINDOW * 4;
  static constexpr int BYTES = OFF_ANY + 16 * 4;
  static constexpr int O_BYTES = D_V * 32 * 4;                // a wave's O
  static constexpr int OFF_ML = (NW / 2) * O_BYTES;           // [NW / 2][32][2], behind the O that lie over the tiles
  static constexpr int WGS = 3;                               // workgroups a CU (LDS by blocks of at most 2 KiB)
  static_assert(WGS * ((BYTES + 2047) / 2048 * 2048) <= kLdsOfCu && OFF_ML + (NW / 2) * 32 * 8 <= OFF_T, "LDS");
  static_assert(KEYS * (AHEAD + 2) < WINDOW, "the steps that are asked for lie in the window, also where pages have one row");
  static_assert(CODES % 64 == 0 && CODES <= 256, "code pieces by whole waves");
};

template <int NT, bool FP4>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Paged<NT, FP4>::WGS))) paged_rows_kernel(const PagedParams p) {
  using C = Paged<NT, FP4>;
  using Row = typename C::Row;
  constexpr int D_QK = C::D_QK, D_V = C::D_V, KS = C::KS, NDT = C::NDT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const int rt = w % NT, kg = w / NT;
  int *window = reinterpret_cast<int *>(smem + C::OFF_T);
  float *ML = reinterpret_cast<float *>(smem + C::OFF_ML);
  const uint32_t lds0 = lds_address(smem);
  const unsigned char *zero = reinterpret_cast<const unsigned char *>(kZeroRow);
  // MXFP4: chunks are also permuted by their panel, as neighbouring lanes write one row's blocks, a panel to two of them
  auto panel_swz = [](int panel) { return FP4 ? (panel & 7) << 4 : 0; };
  const RowRead row_at;
  const ColRead col_at;
  auto row_read = [&](const unsigned char *tile, int ks) {
    return *reinterpret_cast<const i32x4 *>(tile + (row_at.a[ks & 3] ^ panel_swz(ks >> 2)) + (ks >> 2) * 4096);
  };
  auto col_read = [&](const unsigned char *tile, int dt, int u) {
    const unsigned char *base = tile + (dt >> 1) * 4096 + u * 2048;
    const i32x2 r0 = ds_read_tr16(base + (col_at.a[0][dt & 1] ^ panel_swz(dt >> 1)));
    const i32x2 r1 = ds_read_tr16(base + (col_at.a[1][dt & 1] ^ panel_swz(dt >> 1)));
    return i32x4{r0[0], r0[1], r1[0], r1[1]};
  };
  auto page_of = [&](int key) { return p.block_shift >= 0 ? key >> p.block_shift : (int)((uint32_t)key / (uint32_t)p.block); };

  const int units = uni(p.unit0[p.R]), total = uni(p.unit_at[units]), per = uni(range_blocks(p, total));
  if ((int64_t)blockIdx.x * per >= total) return;
  int at = (int)blockIdx.x * per;
  const int end = per < total - at ? at + per : total;
  for (int u = uni(unit_of(p, units, at)); at < end; ++u) {
    const PagedPiece x = next_piece(p, u, at, end);
    const int tok0 = x.first / p.H, tok1 = (x.first + x.nrows - 1) / p.H;
    const int row = 32 * rt + l32;  // of the unit
    i32x4 q[KS];
    {
      const unsigned char *src = (row < x.nrows ? p.q + (x.row0 + row) * D_QK * 2 : zero) + 16 * g32;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q[ks] = ld_row_16(src + 32 * ks);
    }
    // Tokens [ta, tb] with the keys cut at tb's: all at once, or, where that left something that is not finite, one by
    // one, since a weight of zero does not remove the Inf or NaN of a later token's key.
    int ta = tok0, tb = tok1;
    bool probe = tok0 != tok1;
    while (true) {
      const int lim = token_keys(x.kv, x.n, tb), lim_min = token_keys(x.kv, x.n, ta);
      const int j1 = min(x.b1, (lim + C::KEYS - 1) / C::KEYS);  // steps past it hold no key
      const int t = (x.first + row) / p.H, my_lim = token_keys(x.kv, x.n, t < tb ? t : tb);
      int base = 0;          // first page in the window
      bool all_there = true;
      auto refill = [&](int first_page) {
        base = first_page;
        const int pages = lim > 0 ? page_of(lim - 1) + 1 : 0;
        bool ok = true;
        __syncthreads();  // the window's readers are done
        for (int i = (int)threadIdx.x; i < C::WINDOW; i += 256) {
          const int pg = base + i;
          int e = -1;
          if (pg < pages) {
            e = x.table[pg];
            if (e < 0 || e >= p.num_blocks) {
              e = -1;
              ok = false;
            }
          }
          window[i] = e;
        }
        all_there = !any_wave<C::NW>(!ok, smem + C::OFF_ANY);  // (its barriers stand behind the entries too)
      };
      // row of a key, by the window
      auto key_at = [&](int key) -> const unsigned char * {
        const int pg = page_of(key), e = key < lim ? window[pg - base] : -1;
        const int64_t slot = (int64_t)e * p.block + (key - pg * p.block);
        return e >= 0 ? p.cache + slot * Row::BYTES : zero;
      };
      // the wave's 8-row groups of a step's tiles (bf16: their rows; MXFP4: their rope part)
      auto fetch = [&](int j, int buf) {
        constexpr int P0 = FP4 ? D_V / 64 : 0;
#pragma unroll
        for (int i = 0; i < C::TILES; ++i) {
          const int grp = w + 4 * i, r = 8 * (grp & 3) + (lane >> 3);
          const unsigned char *src = key_at(j * C::KEYS + 8 * grp + (lane >> 3)) + (FP4 ? Row::OFF_ROPE : 0) +
                                     ((((lane & 7) ^ row_swz(r)) * 16) ^ panel_swz(P0));
#pragma unroll
          for (int pn = P0; pn < C::PANELS; ++pn)
            dma_16_at(lds0 + (uint32_t)(buf * C::STEP + (grp >> 2) * C::TILE + pn * 4096 + (grp & 3) * 1024), src + (pn - P0) * 128);
        }
      };
      // MXFP4: code pieces of a step, a row's from neighbouring threads
      i32x4 codes{0, 0, 0, 0};
      uint32_t expo = 0;
      const int my_key = (int)threadIdx.x / C::NB, my_blk = (int)threadIdx.x % C::NB;
      auto load_codes = [&](int j) {
        if (w * 64 >= C::CODES) return;  // wave-uniform
        const unsigned char *src = key_at(j * C::KEYS + my_key);
        codes = ld_row_16(src + my_blk * 16);
        expo = ld_row_1(src + Row::OFF_EXP + my_blk);
      };
      auto store_codes = [&](int buf) {
        if (w * 64 >= C::CODES) return;
        const float sc = e8m0_scale(expo);
        unsigned char *dst = smem + buf * C::STEP + (my_key >> 5) * C::TILE + (my_blk >> 1) * 4096;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          i32x4 v = e2m1x8_to_bf16((uint32_t)codes[c], sc);
          if (expo == 255u) v = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
          *reinterpret_cast<i32x4 *>(dst + (tile_byte(my_key & 31, 4 * (my_blk & 1) + c) ^ panel_swz(my_blk >> 1))) = v;
        }
      };

      float m_run = kLeastMax, l_run = 0.0f;
      f32x16 o[NDT];
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] = zero16();

      // one 32-key tile from key0 at LDS tile K
      auto tile_step = [&](const unsigned char *K, int key0) {
        auto rows = [&](int ks) { return row_read(K, ks); };
        auto cols = [&](int i) { return col_read(K, i >> 1, i & 1); };
        f32x16 acc = zero16();
        Operands ka;
        load_group<KS>(ka, 0, rows);
        stream_operands<KS>(ka, rows, [&](int ks, i32x4 a) {
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(q[ks]), acc, 0, 0, 0);
        });
        Operands va;
        load_group<2 * NDT>(va, 0, cols);
        __builtin_amdgcn_sched_barrier(0);
        if (!all_there || key0 + 32 > lim_min) {
          keep_branch();
          const uint32_t there = (uint32_t)wv::ballot(key0 + l32 < lim && window[page_of(key0 + l32) - base] >= 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = acc_row(i, g32);
            if (!((there >> k) & 1u) || key0 + k >= my_lim) acc[i] = -INFINITY;
          }
        }
        float mx = acc[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, acc[i]);
        mx = max_halves(mx) * p.sl2;
        if (wv::ballot(mx > m_run + 8.0f) != 0ull) {
          const float m_new = fmaxf(m_run, mx), alpha = exp2_fast(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[i] = exp2_fast(fmaf(acc[i], p.sl2, -m_run));
          l_run += acc[i];
        }
        i32x4 pb[2];
        pack_operand(acc, pb);
        stream_operands<2 * NDT>(va, cols, [&](int i, i32x4 a) {
          o[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(pb[i & 1]), o[i >> 1], 0, 0, 0);
        });
      };

      refill(page_of(x.b0 * C::KEYS));
      if (x.b0 < j1) {
        if constexpr (FP4) {
          load_codes(x.b0);
          fetch(x.b0, 0);
          store_codes(0);
          load_codes(x.b0 + 1);
        } else {
#pragma unroll
          for (int i = 0; i < C::AHEAD; ++i) fetch(x.b0 + i, i);
        }
      }
      int buf = 0;
      for (int j = x.b0; j < j1; ++j) {
        // what is asked for in this step lies in the window, and what is masked in it
        if (page_of((j + C::AHEAD + 2) * C::KEYS - 1) >= base + C::WINDOW && page_of(lim - 1) >= base + C::WINDOW) refill(page_of(j * C::KEYS));
        const unsigned char *S = smem + buf * C::STEP;
        const int nxt = buf + 1 == C::NBUF ? 0 : buf + 1;
        if constexpr (FP4) {
          __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
          __syncthreads();          // step j is whole; the step before it is consumed
          store_codes(nxt);         // step j + 1
          fetch(j + 1, nxt);
          load_codes(j + 2);
        } else {
          __builtin_amdgcn_s_waitcnt(vmcnt_only((C::AHEAD - 1) * C::DMA));  // this wave's share of step j
          __syncthreads();
          fetch(j + C::AHEAD, buf == 0 ? C::NBUF - 1 : buf - 1);           // (past the last step: zeros)
        }
#pragma unroll
        for (int sub = 0; sub < C::SUB; ++sub) {
          const int tl = kg * C::SUB + sub, key0 = j * C::KEYS + tl * 32;
          if (key0 < lim) tile_step(S + tl * C::TILE, key0);
        }
        buf = nxt;
      }
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // what was fetched past the last step has landed
      if (probe) {
        bool bad = false;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) bad |= not_finite(o[dt][i]);
        if (any_wave<C::NW>(bad, smem + C::OFF_ANY)) {
          probe = false;
          ta = tb = tok0;
          continue;
        }
      }
      l_run = sum_halves(l_run);
      // the key groups' sums, pairwise: waves of the upper half of them leave theirs for the lower half
#pragma unroll
      for (int half = C::KG / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (kg >= half && kg < 2 * half) {
          const int slot = (kg - half) * NT + rt;
          unsigned char *dst = smem + slot * C::O_BYTES;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int m = 0; m < 4; ++m)
              *reinterpret_cast<f32x4 *>(dst + ((dt * 4 + m) * 64 + lane) * 16) =
                  f32x4{o[dt][4 * m], o[dt][4 * m + 1], o[dt][4 * m + 2], o[dt][4 * m + 3]};
          if (g32 == 0) {
            ML[(slot * 32 + l32) * 2] = m_run;
            ML[(slot * 32 + l32) * 2 + 1] = l_run;
          }
        }
        __syncthreads();
        if (kg < half) {
          const int slot = kg * NT + rt;
          const unsigned char *src = smem + slot * C::O_BYTES;
          const float m2 = ML[(slot * 32 + l32) * 2], l2 = ML[(slot * 32 + l32) * 2 + 1];
          // (a group without a key of the row has l = 0 and O = 0)
          const float m_new = l2 == 0.0f ? m_run : (l_run == 0.0f ? m2 : fmaxf(m_run, m2));
          const float a1 = l_run == 0.0f ? 0.0f : exp2_fast(m_run - m_new), a2 = l2 == 0.0f ? 0.0f : exp2_fast(m2 - m_new);
          m_run = m_new;
          l_run = l_run * a1 + l2 * a2;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const f32x4 y = *reinterpret_cast<const f32x4 *>(src + ((dt * 4 + m) * 64 + lane) * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[dt][4 * m + e] = o[dt][4 * m + e] * a1 + y[e] * a2;
            }
        }
      }
      const int rlo = ta * p.H - x.first, rhi = min((tb + 1) * p.H - x.first, x.nrows);  // rows of tokens [ta, tb]
      if (kg == 0 && row >= rlo && row < rhi) {
        const bool none = my_lim <= x.b0 * C::KEYS || l_run == 0.0f;  // no key of this piece
        const float inv = none ? 0.0f : 1.0f / l_run;
        const int64_t part = (int64_t)x.slot * C::ROWS + row;
        if (g32 == 0) {
          if (x.whole) {
            p.lse[x.row0 + row] = none ? -INFINITY : log2f(l_run) + m_run;
          } else {
            p.part_ml[part * 2] = m_run;
            p.part_ml[part * 2 + 1] = none ? 0.0f : l_run;
          }
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const f32x4 v{o[dt][4 * m], o[dt][4 * m + 1], o[dt][4 * m + 2], o[dt][4 * m + 3]};
            const int col = acc_col(dt, 4 * m, g32);
            if (x.whole) {
              // a row without keys: 0, whatever its neighbours' keys left
              *reinterpret_cast<i32x2 *>(p.out + (x.row0 + row) * D_V + col) =
                  none ? i32x2{0, 0} : i32x2{(int)pack_bf16x2(v[0] * inv, v[1] * inv), (int)pack_bf16x2(v[2] * inv, v[3] * inv)};
            } else if (!none) {
              *reinterpret_cast<f32x4 *>(p.part_o + part * D_V + col) = v;
            }
          }
      }
      __syncthreads();  // LDS is free for the next piece
      if (tb == tok1) break;
      ta = ++tb;
    }
  }
}

// Workgroup (w, y): where the first of a unit's blocks that is not in the piece of the
// workgroup that began it is in range w + 1, some rows of that unit, a row to 64 lanes
// (64 channels: to 16), one after the other: its pieces brought to their largest maximum
// and added in order, read AHEAD at a time.
template <int D_V, bool SPARSE>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedParams p) {
  constexpr int NCH = D_V / 4, LANES = NCH < 64 ? NCH : 64, CPL = NCH / LANES, AT_ONCE = 256 / LANES, AHEAD = 4;
  const int ln = lane_id() % LANES;
  int units, total;
  all_units<SPARSE>(p, units, total);
  const int per = uni(range_blocks(p, total));
  const int64_t cut = ((int64_t)blockIdx.x + 1) * per;
  if (cut >= total) return;
  const int u = uni(unit_of<SPARSE>(p, units, (int)cut)), ub = unit_begin<SPARSE>(p, u), ue = unit_begin<SPARSE>(p, u + 1);
  const int w0 = ub / per, pieces = (ue - 1) / per - w0 + 1;
  if (ub == cut || w0 != (int)blockIdx.x) return;  // no unit is cut here, or it was cut before
  int at_unit = ub;
  const PagedPiece x_u = next_piece<SPARSE>(p, u, at_unit, ue);
  const int nrows = x_u.nrows;
  const int64_t row0 = x_u.row0;
  const int rows = p.unit_rows / (int)gridDim.y;
  for (int ur = (int)blockIdx.y * rows + (int)threadIdx.x / LANES; ur < min(((int)blockIdx.y + 1) * rows, nrows); ur += AT_ONCE) {
    const int64_t row = row0 + ur;
    // piece k's row of partial results: in the second place of the workgroup that began the unit, the first of the others
    auto at = [&](int k) { return (int64_t)((w0 + k) * 2 + (k == 0 ? 1 : 0)) * p.unit_rows + ur; };
    float m = kLeastMax;
    for (int k = ln; k < pieces; k += LANES)
      if (p.part_ml[at(k) * 2 + 1] != 0.0f) m = fmaxf(m, p.part_ml[at(k) * 2]);
#pragma unroll
    for (int x = LANES / 2; x >= 1; x /= 2) m = fmaxf(m, __shfl_xor(m, x, 64));
    float l = 0.0f;
    f32x4 o[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < pieces; k0 += AHEAD) {
      f32x4 x[AHEAD][CPL];
      float lk[AHEAD], mk[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t r = at(min(k0 + i, pieces - 1));
        mk[i] = p.part_ml[r * 2];
        lk[i] = k0 + i < pieces ? p.part_ml[r * 2 + 1] : 0.0f;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
          x[i][c] = *reinterpret_cast<const f32x4 *>(p.part_o + r * D_V + (ln + LANES * c) * 4);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (lk[i] == 0.0f) continue;  // no key of the row in the piece, which left no O (a NaN sum joins)
        const float a = exp2_fast(mk[i] - m);
        l += lk[i] * a;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
          o[c] += a * x[i][c];
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < CPL; ++c)
      *reinterpret_cast<i32x2 *>(p.out + row * D_V + (ln + LANES * c) * 4) =
          i32x2{(int)pack_bf16x2(o[c][0] * inv, o[c][1] * inv), (int)pack_bf16x2(o[c][2] * inv, o[c][3] * inv)};
    if (ln == 0) p.lse[row] = l == 0.0f ? -INFINITY : log2f(l) + m;
  }
}

// How a call is run, from its sizes alone: by the rows that share keys, a request's (token, head) pairs on average.
// Times of a step of 64 requests, 301 .. 16384 keys, us, the chosen one's first:
//   576, bf16   up to 64 rows    units of 64: 16 heads 143, 64 heads 159; of 128: 189, 204
//               more             units of 128: 128 heads 229; of 64: 260
//   576, MXFP4  up to 32 rows    units of 32: 16 heads 103, 32 heads 107; of 64: 144, 146
//               more             units of 64: 64 heads 158, 128 heads 274; of 32: 177, 309
//   128, bf16   up to 16 rows    waves that split the keys, 16 rows: 16 heads 40; units of 64: 49
//               up to 64         units of 64: 32 heads 50, 64 heads 53; of 128: 54, 56; 16 rows: 59, 97
//               more             units of 128: 128 heads 64; of 64: 73
//   128, MXFP4  up to 32 rows    16 rows: 16 heads 37, 32 heads 49; units of 128: 63, 65
//               more             units of 128: 64 heads 69, 128 heads 76; 16 rows: 78, 129
struct PagedPlan {
  int wide;       // 576 / 512: 16-row tiles of a unit
  bool few;       // 128 / 64: 16 rows a unit, whose waves split the keys
  int nt;         // 128 / 64: else 32-row tiles of a unit
  int unit_rows, step_keys, max_units, nwg, min_blocks;
};
static PagedPlan paged_plan(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, bool fp4) {
  PagedPlan r{};
  const int64_t rows = (T + R - 1) / R * H;
  if (d_qk == 576) {
    r.wide = fp4 ? (rows <= 32 ? 2 : 4) : (rows <= 64 ? 4 : 8);
    r.unit_rows = 16 * r.wide;
    r.step_keys = paged_wide_keys();
  } else if (rows <= (fp4 ? 32 : 16)) {
    r.few = true;
    r.unit_rows = 16;
    r.step_keys = 32;
  } else {
    r.nt = fp4 || rows > 64 ? 4 : 2;
    r.unit_rows = 32 * r.nt;
    r.step_keys = 64;
  }
  r.min_blocks = 256 / r.step_keys;  // keys that are worth a piece's beginning and end
  r.max_units = (int)(T * H / r.unit_rows + R);
  const int64_t blocks = (int64_t)r.max_units * ((W * block + r.step_keys - 1) / r.step_keys);
  const int64_t n = (blocks + r.min_blocks - 1) / r.min_blocks;
  const int64_t most = 256 * (d_qk == 128 ? Paged<4, true>::WGS : 1);  // resident workgroups (few rows: as many fit)
  r.nwg = (int)(n < 1 ? 1 : (n < most ? n : most));
  return r;
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
struct PagedSections {
  size_t unit0, unit_req, unit_first, unit_at, part_ml, part_o, total;
};
static PagedSections paged_sections(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v, bool fp4) {
  const PagedPlan k = paged_plan(T, R, W, block, H, d_qk, fp4);
  const size_t units = (size_t)k.max_units, pieces = (size_t)k.nwg * 2 * (size_t)k.unit_rows;
  PagedSections s;
  s.unit0 = 0;
  s.unit_req = s.unit0 + up256(((size_t)R + 1) * 4);
  s.unit_first = s.unit_req + up256(units * 4);
  s.unit_at = s.unit_first + up256(units * 4);
  s.part_ml = s.unit_at + up256((units + 1) * 4);
  s.part_o = s.part_ml + pieces * 8;
  s.total = s.part_o + pieces * (size_t)d_v * 4;
  return s;
}
bool paged_countable(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk) {
  bool ok = true;
  for (int fp4 = 0; fp4 < 2; ++fp4) {
    const PagedPlan k = paged_plan(T, R, W, block, H, d_qk, fp4 != 0);
    ok = ok && (T * H / k.unit_rows + R) * ((W * block + k.step_keys - 1) / k.step_keys) < (1ll << 31);
  }
  return ok;
}
size_t paged_workspace(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v) {
  // the larger of the two formats': the query does not know it
  const size_t a = paged_sections(T, R, W, block, H, d_qk, d_v, false).total, b = paged_sections(T, R, W, block, H, d_qk, d_v, true).total;
  return a > b ? a : b;
}

template <int NT, bool FP4>
static int launch(const PagedParams &p, hipStream_t st) {
  using C = Paged<NT, FP4>;
  hipLaunchKernelGGL((paged_rows_kernel<NT, FP4>), dim3((unsigned)p.nwg), dim3(256), C::BYTES, st, p);
  return check_launch("dsa_paged_latent_mla_fwd");
}

int launch_paged_combine(const PagedParams &p, int64_t d_v, bool sparse, hipStream_t st) {
  if (p.nwg == 1) return DSA_OK;  // one workgroup: no unit has several pieces
  const dim3 grid((unsigned)(p.nwg - 1), (unsigned)(p.unit_rows / (p.unit_rows < 64 ? 4 : 16)));
  if (sparse) hipLaunchKernelGGL((paged_combine_kernel<512, true>), grid, dim3(256), 0, st, p);
  else if (d_v == 512) hipLaunchKernelGGL((paged_combine_kernel<512, false>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_combine_kernel<64, false>), grid, dim3(256), 0, st, p);
  return check_launch("dsa_paged_latent_mla_fwd (combine)");
}

int launch_paged_fwd(PagedParams p, int64_t d_qk, int64_t d_v, bool fp4, unsigned char *ws, hipStream_t st) {
  const PagedSections s = paged_sections(p.T, p.R, p.W, p.block, p.H, d_qk, d_v, fp4);
  const PagedPlan k = paged_plan(p.T, p.R, p.W, p.block, p.H, d_qk, fp4);
  p.unit_rows = k.unit_rows;
  p.max_units = k.max_units;
  p.nwg = k.nwg;
  p.min_blocks = k.min_blocks;
  p.step_keys = k.step_keys;
  p.unit0 = (int32_t *)(ws + s.unit0);
  p.unit_req = (int32_t *)(ws + s.unit_req);
  p.unit_first = (int32_t *)(ws + s.unit_first);
  p.unit_at = (int32_t *)(ws + s.unit_at);
  p.part_ml = (float *)(ws + s.part_ml);
  p.part_o = (float *)(ws + s.part_o);
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(1024), 0, st, p);
  int rc = check_launch("dsa_paged_latent_mla_fwd (plan)");
  if (rc) return rc;
  if (k.wide) rc = launch_paged_wide(p, k.wide, fp4, false, st);
  else if (k.few) rc = launch_paged_few(p, fp4, st);
  else if (k.nt == 4) rc = fp4 ? launch<4, true>(p, st) : launch<4, false>(p, st);
  else rc = launch<2, false>(p, st);
  return rc ? rc : launch_paged_combine(p, d_v, false, st);
}

}  // namespace dsa
