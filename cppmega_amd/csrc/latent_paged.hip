// Latent attention over a paged cache on gfx950 (absorbed form, bf16 or MXFP4 rows):
// decoding, speculative tokens and prefill chunks of ragged requests.
//
// A request's rows are its (new token, head) pairs in that order; a unit is NT * 32 of
// them with the keys 0 .. of its last token.  The units' 32-key blocks, one after the
// other, are split evenly over the grid's workgroups (stream-wise, so a long request is
// shared and short ones are packed), whose ends may fall inside a unit: such a piece
// leaves its unnormalised fp32 O, maximum and sum, and paged_combine_kernel adds a unit's
// pieces in order.  The plan (units and their first blocks) is made on the device from
// the lengths: the host knows neither.
//
// A block's products follow the wide SparseMLA forward: S^T partial sums over parts of
// the channels meet through LDS, the softmax of block j runs beside the PV products of
// block j - 1 (two barriers a block), and block j + 1's rows arrive by LDS-DMA loads from
// 64-bit addresses that the block table gives (MXFP4: as codes in registers, written to
// the tile as exact bf16 values).  Keys past a request's last, and keys whose table entry
// is no page, read as zeros and have no weight.
#include "latent_paged.hpp"
#include "sparse_mla_wide_tile.hpp"
#include "wave_ops.hpp"

namespace dsa {

// blocks of a unit (at least one: a unit without keys still writes its rows)
__device__ __forceinline__ int unit_blocks(const PagedParams &p, int kv, int n, int first, int rows, int unit_rows) {
  const int last = min(first + unit_rows, rows) - 1;
  return max((token_keys(kv, n, last / p.H) + 31) / 32, 1);
}

// Exclusive prefix over the workgroup of one value per thread; total in every thread.
template <int NTHR>
__device__ __forceinline__ int block_scan(int x, int *tmp, int &total) {
  const int lane = lane_id(), w = (int)(threadIdx.x >> 6);
  const int v = (int)wv::wave_incl_scan((uint32_t)x);
  __syncthreads();
  if (lane == 63) tmp[w] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NTHR / 64; ++i) {
    const int t = tmp[i];
    if (i < w) before += t;
    total += t;
  }
  return before + v - x;
}

// The plan, one workgroup: unit_req[u], unit_first[u] (first row), unit_at[u] (first block,
// unit_at[units] = all), unit0[r] (first unit of request r; unit0[R] = all).
__global__ void __launch_bounds__(1024) paged_plan_kernel(const PagedParams p) {
  __shared__ int tmp[16];
  int total, at = 0;
  for (int r0 = 0; r0 < p.R; r0 += 1024) {
    const int r = r0 + (int)threadIdx.x;
    // (starts that do not ascend may ask for more units than there are: cut)
    const int n = r < p.R ? min((request_tokens(p, r) * p.H + p.unit_rows - 1) / p.unit_rows, p.max_units) : 0;
    const int x = at + block_scan<1024>(n, tmp, total);
    if (r < p.R) p.unit0[r] = min(x, p.max_units);
    at = min(at + total, p.max_units);
  }
  const int units = at;
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
      const int first = (u - p.unit0[lo]) * p.unit_rows, n = request_tokens(p, lo);
      nb = unit_blocks(p, request_kv(p, lo), n, first, n * p.H, p.unit_rows);
      p.unit_req[u] = lo;
      p.unit_first[u] = first;
    }
    const int x = at + block_scan<1024>(nb, tmp, total);
    if (u < units) p.unit_at[u] = x;
    at += total;
  }
  if (threadIdx.x == 0) p.unit_at[units] = at;
}

template <int D_QK, int D_V, int NT, int NW_, bool FP4>
struct Paged {
  static constexpr int NW = NW_, NTHR = 64 * NW, KP = NW / NT;
  static constexpr int FW = NW / 2;                          // waves that fetch by DMA
  using T = DmaTile<D_QK, FW>;
  using Row = CacheRow<D_QK, D_V, FP4>;
  static constexpr int KS = D_QK / 16 / KP;
  static constexpr int NDT = D_V / 16, DTW = (NDT + NW - 1) / NW;
  static constexpr int ROWS = 32 * NT, HW = ROWS / NW;       // rows per wave in the softmax
  static constexpr int LPH = 64 / HW, SPL4 = 8 / LPH;
  static constexpr int SP_W = 32 * 32;
  static constexpr int PT_BYTES = 32 * 32 * 2;
  static constexpr int CODES = 32 * (D_V / 32);              // 16-byte pieces of codes in a block
  static constexpr int CPT = (CODES + NTHR - 1) / NTHR;      // per thread
  static constexpr int OFF_K = 0;
  static constexpr int OFF_SP = OFF_K + 3 * T::BYTES;
  static constexpr int OFF_P = OFF_SP + NW * SP_W * 4;
  static constexpr int OFF_AL = OFF_P + 2 * NT * PT_BYTES;
  static constexpr int OFF_FL = OFF_AL + 3 * ROWS * 4;
  static constexpr int BYTES = OFF_FL + 2 * NW * 4;
  static_assert(D_QK / 16 % KP == 0 && (KP == 2 || KP == 4) && (HW == 8 || HW == 16), "wave split");
  static_assert(BYTES <= 159 * 1024, "LDS");
};

template <int D_QK, int D_V, int NT, int NW, bool FP4>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW / 4))) paged_fwd_kernel(const PagedParams p) {
  using C = Paged<D_QK, D_V, NT, NW, FP4>;
  using T = typename C::T;
  using Row = typename C::Row;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  // Lane-dependent values are formed from lane_here() where they are used: kept across a unit's blocks they would
  // take the registers of O and Q.
  const int w = wave_id();
  unsigned char *K = smem + C::OFF_K;
  float *Sp = reinterpret_cast<float *>(smem + C::OFF_SP);
  unsigned char *P = smem + C::OFF_P;
  float *AL = reinterpret_cast<float *>(smem + C::OFF_AL);
  int *FL = reinterpret_cast<int *>(smem + C::OFF_FL);
  const uint32_t k_lds = lds_address(K);
  const unsigned char *zero = reinterpret_cast<const unsigned char *>(kZeroRow);
  // MXFP4: chunks are also permuted by their panel, as neighbouring lanes write one row's blocks, a panel to two of them
  auto panel_swz = [](int panel) { return FP4 ? (panel & 7) << 4 : 0; };
  const int ht = w / C::KP, kq = w % C::KP;
  constexpr int kPh = 4 / C::KP;
  const int et = w * C::HW / 32;  // row tile of this wave's softmax rows

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

    // this wave's part of Q: row lane % 32 of tile ht, k-steps KP i + kq; and where its operands of K are
    i32x4 q[C::KS];
    int ka[kPh];
    {
      const int ln = lane_here(), r = 32 * ht + (ln & 31), g32 = ln >> 5;
#pragma unroll
      for (int i = 0; i < C::KS; ++i) {
        q[i] = i32x4{0, 0, 0, 0};
        if (r < nrows) q[i] = ld_global_16(p.q + ((row0 + r) * D_QK + 16 * (C::KP * i + kq) + 8 * g32) * 2);
      }
#pragma unroll
      for (int v = 0; v < kPh; ++v) ka[v] = tile_byte(ln & 31, 2 * (C::KP * v + kq) + g32);
    }

    // Runs the piece with the tokens' keys cut at those of token tlim and writes the rows of tokens
    // [tok, tlim].  All tokens at once; where that leaves something that is not finite, token by
    // token, since a row's weight of zero does not remove the Inf or NaN of a later token's key.
    auto run = [&](int tok, int tlim, bool probe) -> bool {
      const int lim = token_keys(kv, n, tlim);           // keys that are read
      const int lim_min = token_keys(kv, n, tok);        // keys that every row sees
      auto row_keys = [&](int r) {                       // of row r
        const int t = (first + r) / p.H;
        return token_keys(kv, n, t < tlim ? t : tlim);
      };
      const int j1 = min(b1, (lim + 31) / 32);           // blocks past it hold no key
      auto entry = [&](int j) { return key_entry(p, table, j, lim); };
      auto row_at = [&](int j, int e) { return key_row(p, j, e, Row::BYTES); };
      auto there = [&](int e) { return (uint32_t)wv::ballot(e >= 0 && e < p.num_blocks); };
      // bf16: the rows; MXFP4: their rope part, into its panels
      auto fetch = [&](int tile, const unsigned char *mine) {
        const int ln = lane_here();
        constexpr int P0 = FP4 ? D_V / 64 : 0, SRC = FP4 ? Row::OFF_ROPE : 0;
#pragma unroll
        for (int i = 0; i < T::RG; ++i) {
          const int rg = w + T::NW * i, row = 8 * rg + (ln >> 3);
          const unsigned char *src = shfl_ptr(mine, row) + SRC + ((((ln & 7) ^ row_swz(row)) * 16) ^ panel_swz(P0));
#pragma unroll
          for (int pn = P0; pn < T::PANELS; ++pn) {
            __builtin_amdgcn_sched_barrier(0);  // an address at a time
            dma_16_at(k_lds + (uint32_t)(tile * T::BYTES + pn * T::PANEL + rg * 1024), src + (pn - P0) * 128);
          }
        }
      };
      // MXFP4 latent: 16 bytes of codes (one 32-channel block of a row) and its exponent per piece
      i32x4 codes[FP4 ? C::CPT : 1];
      uint32_t expo[FP4 ? C::CPT : 1];
      auto piece_of = [&](int i, int &row, int &blk) {  // a row's codes from neighbouring lanes
        const int y = (w + NW * i) * 64 + lane_here();
        row = y / (D_V / 32);
        blk = y % (D_V / 32);
      };
      auto load_codes = [&](const unsigned char *mine) {
        if constexpr (FP4) {
#pragma unroll
          for (int i = 0; i < C::CPT; ++i) {
            int row, blk;
            piece_of(i, row, blk);
            const bool in = C::CODES % C::NTHR == 0 || (w + NW * i) * 64 < C::CODES;
            const unsigned char *src = shfl_ptr(mine, row & 31);
            codes[i] = i32x4{0, 0, 0, 0};
            expo[i] = 127;
            if (in && src != zero) {
              codes[i] = ld_global_16(src + blk * 16);
              expo[i] = src[Row::OFF_EXP + blk];
            }
          }
        }
      };
      auto store_codes = [&](int tile) {
        if constexpr (FP4) {
#pragma unroll
          for (int i = 0; i < C::CPT; ++i) {
            if (!(C::CODES % C::NTHR == 0 || (w + NW * i) * 64 < C::CODES)) continue;
            int row, blk;
            piece_of(i, row, blk);
            const float s = e8m0_scale(expo[i]);
            unsigned char *dst = K + tile * T::BYTES + (blk >> 1) * T::PANEL;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              i32x4 v = e2m1x8_to_bf16((uint32_t)codes[i][c], s);
              if (expo[i] == 255u) v = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
              *reinterpret_cast<i32x4 *>(dst + (tile_byte(row, 4 * (blk & 1) + c) ^ panel_swz(blk >> 1))) = v;
            }
          }
        }
      };

      float m_run = kNegBig, l_run = 0.0f;
      f32x4 o[C::DTW][2 * NT];
#pragma unroll
      for (int i = 0; i < C::DTW; ++i)
#pragma unroll
        for (int h = 0; h < 2 * NT; ++h) o[i][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

      auto pv_step = [&](const unsigned char *Kb, int buf) {
        const int ln = lane_here(), c16 = ln & 15, cg = ln >> 4;
        if (wv::ballot(FL[buf * NW + (ln & (NW - 1))] != 0) != 0ull) {
#pragma unroll
          for (int h = 0; h < 2 * NT; ++h) {
            const float a = AL[buf * C::ROWS + 16 * h + c16];
#pragma unroll
            for (int i = 0; i < C::DTW; ++i) o[i][h] *= a;
          }
        }
        if (C::NDT < NW && w >= C::NDT) return;
        // V^T of d tile w + NW i: rows 8 cg + (lane % 16) / 4 (+ 4), columns 4 (lane % 4) .. of the tile
        int vt[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int c = c16 & 3;
          vt[v] = tile_byte(8 * cg + 4 * v + (c16 >> 2), 2 * (w & 3) + (c >> 1)) + (c & 1) * 8;
        }
        // P[row][key]: 64-byte rows, 16-byte chunk c of row r at c ^ ((r >> 2) & 3)
        const int p_rd = buf * NT * C::PT_BYTES + c16 * 64 + ((cg ^ ((c16 >> 2) & 3)) * 16);
        i32x4 av[C::DTW];
#pragma unroll
        for (int i = 0; i < C::DTW; ++i) {
          const int pn = (w >> 2) + i * (NW / 4);
          const i32x2 r0 = ds_read_tr16(Kb + (vt[0] ^ panel_swz(pn)) + pn * T::PANEL);
          const i32x2 r1 = ds_read_tr16(Kb + (vt[1] ^ panel_swz(pn)) + pn * T::PANEL);
          av[i] = i32x4{r0[0], r0[1], r1[0], r1[1]};
        }
#pragma unroll
        for (int h = 0; h < 2 * NT; ++h) {
          const i32x4 bv = *reinterpret_cast<const i32x4 *>(P + p_rd + (h >> 1) * C::PT_BYTES + (h & 1) * 1024);
#pragma unroll
          for (int i = 0; i < C::DTW; ++i)
            o[i][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(av[i]), as_bf16x8(bv), o[i][h], 0, 0, 0);
        }
      };

      int e_nxt = entry(b0);  // table entry of the block that is fetched next
      uint32_t vm = there(e_nxt);
      if (b0 < j1) {
        const unsigned char *mine = row_at(b0, e_nxt);
        if (w < C::FW) fetch(0, mine);
        load_codes(mine);
        store_codes(0);
        e_nxt = entry(b0 + 1);
        if constexpr (FP4) load_codes(row_at(b0 + 1, e_nxt));
      }
      int kb = 0, kp = 0;
      for (int j = b0; j < j1; ++j) {
        const int kn = kb == 2 ? 0 : kb + 1, cur = (j - b0) & 1;
        const unsigned char *Kj = K + kb * T::BYTES;
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): block j's rows, issued a block ago
        __syncthreads();                     // block j's rows and block j - 1's P are whole; block j - 2's rows are consumed
        const uint32_t vm_nxt = there(e_nxt);
        if (w < C::FW) fetch(kn, row_at(j + 1, e_nxt));  // block j + 1 (past the last: zeros)
        store_codes(kn);
        e_nxt = entry(j + 2);
        f32x16 acc;
#pragma unroll
        for (int a = 0; a < 16; ++a) acc[a] = 0.0f;
#pragma unroll
        for (int i = 0; i < C::KS; ++i) {
          const i32x4 a = *reinterpret_cast<const i32x4 *>(Kj + (ka[i % kPh] ^ panel_swz(i / kPh)) + (i / kPh) * T::PANEL);
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(q[i]), acc, 0, 0, 0);
        }
        put_partial(Sp + w * C::SP_W, acc);
        __syncthreads();  // partial tiles whole
        if constexpr (FP4) load_codes(row_at(j + 2, e_nxt));
        // softmax: row eh of tile et, 4-key groups (i, eg) with i = ei .. ei + SPL4 - 1: keys 8 i + 4 eg ..
        const int ln = lane_here(), eh = (w * C::HW) % 32 + (ln & (C::HW - 1)), sr = et * 32 + eh;
        const int eq = ln / C::HW, eg = eq & 1, ei = (eq >> 1) * C::SPL4;
        f32x4 s[C::SPL4];
        {
          const float *sp = Sp + et * C::KP * C::SP_W + ((ei * 2 + eg) * 32 + eh) * 4;
#pragma unroll
          for (int x = 0; x < C::SPL4; ++x) {
            s[x] = *reinterpret_cast<const f32x4 *>(sp + x * 256);
#pragma unroll
            for (int k = 1; k < C::KP; ++k) s[x] += *reinterpret_cast<const f32x4 *>(sp + k * C::SP_W + x * 256);
          }
        }
        if (j > b0) pv_step(K + kp * T::BYTES, cur ^ 1);

        // online softmax (log2 domain, lazy rescale); key 32 j + 8 (ei + x) + 4 eg + e
        if (vm != 0xffffffffu || 32 * j + 32 > lim_min) {
          const int my_lim = row_keys(sr);
#pragma unroll
          for (int x = 0; x < C::SPL4; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = 8 * (ei + x) + 4 * eg + e;
              if (!((vm >> k) & 1u) || 32 * j + k >= my_lim) s[x][e] = -INFINITY;
            }
        }
        float mloc = kNegBig;
#pragma unroll
        for (int x = 0; x < C::SPL4; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) mloc = fmaxf(mloc, s[x][e]);
#pragma unroll
        for (int off = C::HW; off < 32; off <<= 1) mloc = fmaxf(mloc, __shfl_xor(mloc, off, 64));
        mloc = max_halves(mloc) * p.sl2;
        const bool moved = wv::ballot(mloc > m_run + 8.0f) != 0ull;
        float alpha = 1.0f;
        if (moved) {
          const float m_new = fmaxf(m_run, mloc);
          alpha = exp2_fast(m_run - m_new);
          l_run *= alpha;
          m_run = m_new;
        }
        if (eq == 0) AL[cur * C::ROWS + sr] = alpha;
        if (ln == 0) FL[cur * NW + w] = moved ? 1 : 0;
#pragma unroll
        for (int x = 0; x < C::SPL4; ++x) {
          float t[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            t[e] = exp2_fast(fmaf(s[x][e], p.sl2, -m_run));
            l_run += t[e];
          }
          *reinterpret_cast<i32x2 *>(P + (cur * NT + et) * C::PT_BYTES + eh * 64 + (((ei + x) ^ ((eh >> 2) & 3)) * 16) + eg * 8) =
              i32x2{(int)pack_bf16x2(t[0], t[1]), (int)pack_bf16x2(t[2], t[3])};
        }
        vm = vm_nxt;
        kp = kb;
        kb = kn;
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);  // what was fetched past the last block has landed
#pragma unroll
      for (int off = C::HW; off < 32; off <<= 1) l_run += __shfl_xor(l_run, off, 64);
      l_run = sum_halves(l_run);
      const int ln = lane_here(), sr = w * C::HW + (ln & (C::HW - 1)), eq = ln / C::HW;  // this lane's softmax row
      const bool none = row_keys(sr) <= 32 * b0 || l_run == 0.0f;  // no key of this piece
      if (eq == 0) AL[2 * C::ROWS + sr] = none ? 0.0f : 1.0f / l_run;
      __syncthreads();
      if (b0 < j1) pv_step(K + kp * T::BYTES, (j1 - b0 - 1) & 1);

      if (probe) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < C::DTW; ++i)
#pragma unroll
          for (int h = 0; h < 2 * NT; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= (__float_as_uint(o[i][h][e]) & 0x7f800000u) == 0x7f800000u;
        if (__syncthreads_or(bad)) return false;
      }
      const int rlo = tok * p.H - first, rhi = min((tlim + 1) * p.H - first, nrows);  // rows of tokens [tok, tlim]
      if (!whole_unit) {
        if (eq == 0 && sr >= rlo && sr < rhi) {
          p.part_ml[(piece * C::ROWS + sr) * 2] = m_run;
          p.part_ml[(piece * C::ROWS + sr) * 2 + 1] = none ? 0.0f : l_run;
        }
      } else if (eq == 0 && sr >= rlo && sr < rhi) {
        p.lse[row0 + sr] = none ? -INFINITY : log2f(l_run) + m_run;
      }
#pragma unroll
      for (int h = 0; h < 2 * NT; ++h) {
        const int r = 16 * h + (ln & 15);
        const float inv = AL[2 * C::ROWS + r];
        if (r >= rlo && r < rhi) {
#pragma unroll
          for (int i = 0; i < C::DTW; ++i)
            if (C::NDT % NW == 0 || w + NW * i < C::NDT) {
              const int d = (w + NW * i) * 16 + 4 * (ln >> 4);
              if (whole_unit) {
                // an empty row's O is zeros (or what a neighbour's key left): 0
                const f32x4 x = inv == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o[i][h] * inv;
                *reinterpret_cast<i32x2 *>(p.out + (row0 + r) * D_V + d) =
                    i32x2{(int)pack_bf16x2(x[0], x[1]), (int)pack_bf16x2(x[2], x[3])};
              } else if (inv != 0.0f) {
                *reinterpret_cast<f32x4 *>(p.part_o + (piece * C::ROWS + r) * D_V + d) = o[i][h];
              }
            }
        }
      }
      __syncthreads();  // LDS is free for the next piece
      return true;
    };
    int ta = tok0, tb = tok1;
    bool probe = tok0 != tok1;
    while (true) {
      if (!run(ta, tb, probe)) {
        probe = false;
        ta = tb = tok0;
        __syncthreads();
        continue;
      }
      if (tb == tok1) break;
      ta = ++tb;
    }
  }
}

// One wave per row of q: the pieces of its unit, where it has several, brought to their
// largest maximum and added in order.
template <int D_V>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedParams p) {
  constexpr int NCH = D_V / 4, CPL = (NCH + 63) / 64;
  const int lane = lane_id();
  const int64_t row = (int64_t)blockIdx.x * 4 + wave_id();
  if (row >= p.T * p.H) return;
  const int tok = (int)(row / p.H);
  int r = tok;
  if (p.query_starts != nullptr) {
    int lo = 0, hi = p.R - 1;  // the last request that starts at or before the token
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (request_start(p, mid) <= tok) lo = mid; else hi = mid - 1;
    }
    r = lo;
    if (tok < request_start(p, r) || tok >= request_start(p, r) + request_tokens(p, r)) return;  // behind the last request
  } else if (r >= p.R) {
    return;
  }
  const int in_req = (int)(row - (int64_t)request_start(p, r) * p.H);
  const int u = p.unit0[r] + in_req / p.unit_rows, ur = in_req % p.unit_rows;
  const int units = p.unit0[p.R];
  if (u >= units) return;
  const int per = range_blocks(p, p.unit_at[units]);
  const int64_t w0 = p.unit_at[u] / per, w1 = (p.unit_at[u + 1] - 1) / per;
  if (w0 == w1) return;  // one piece: its workgroup wrote the row
  auto at = [&](int64_t w) { return (w * 2 + (w == w0 ? 1 : 0)) * p.unit_rows + ur; };
  float m = kNegBig;
  for (int64_t w = w0; w <= w1; ++w)
    if (p.part_ml[at(w) * 2 + 1] != 0.0f) m = fmaxf(m, p.part_ml[at(w) * 2]);
  float l = 0.0f;
  f32x4 o[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t w = w0; w <= w1; ++w) {
    const float lw = p.part_ml[at(w) * 2 + 1];
    if (lw == 0.0f) continue;  // no key of the row in the piece, which left no O (a NaN sum joins)
    const float a = exp2_fast(p.part_ml[at(w) * 2] - m);
    l += lw * a;
#pragma unroll
    for (int c = 0; c < CPL; ++c)
      if (lane + 64 * c < NCH) o[c] += a * *reinterpret_cast<const f32x4 *>(p.part_o + at(w) * D_V + (lane + 64 * c) * 4);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < CPL; ++c)
    if (lane + 64 * c < NCH)
      *reinterpret_cast<i32x2 *>(p.out + row * D_V + (lane + 64 * c) * 4) =
          i32x2{(int)pack_bf16x2(o[c][0] * inv, o[c][1] * inv), (int)pack_bf16x2(o[c][2] * inv, o[c][3] * inv)};
  if (lane == 0) p.lse[row] = l == 0.0f ? -INFINITY : log2f(l) + m;
}

// How a call is run, from its sizes alone.  Rows that share keys: a request's (token, head) pairs, on average.
struct PagedPlan {
  int few;        // 16-row tiles of a unit whose waves split the keys, or 0
  int nt;         // else 32-row tiles of a unit whose waves share them
  int unit_rows, max_units, nwg, min_blocks;
};
static PagedPlan paged_plan(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk) {
  PagedPlan r{};
  const int64_t rows = (T + R - 1) / R * H;
  if (rows <= (d_qk == 576 ? 16 : 32)) {
    r.few = rows <= 16 ? 1 : 2;
    r.unit_rows = 16 * r.few;
  } else {
    r.nt = rows > 64 && d_qk == 576 ? 4 : (rows > 32 ? 2 : 1);
    r.unit_rows = 32 * r.nt;
  }
  r.min_blocks = r.few ? 8 : 4;
  r.max_units = (int)(T * H / r.unit_rows + R);
  const int64_t blocks = (int64_t)r.max_units * ((W * block + 31) / 32), n = (blocks + r.min_blocks - 1) / r.min_blocks;
  const int64_t most = r.few && d_qk == 128 ? 768 : 256;  // resident workgroups
  r.nwg = (int)(n < 1 ? 1 : (n < most ? n : most));
  return r;
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
struct PagedSections {
  size_t unit0, unit_req, unit_first, unit_at, part_ml, part_o, total;
};
static PagedSections paged_sections(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v) {
  const PagedPlan k = paged_plan(T, R, W, block, H, d_qk);
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
size_t paged_workspace(int64_t T, int64_t R, int64_t W, int64_t block, int64_t H, int64_t d_qk, int64_t d_v) {
  return paged_sections(T, R, W, block, H, d_qk, d_v).total;
}

template <int D_QK, int D_V, int NT, int NW, bool FP4>
static int launch(const PagedParams &p, hipStream_t st) {
  using C = Paged<D_QK, D_V, NT, NW, FP4>;
  const auto kernel = paged_fwd_kernel<D_QK, D_V, NT, NW, FP4>;
  const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
  if (e != hipSuccess) return set_error(DSA_ERR_HIP, "dsa_paged_latent_mla_fwd: LDS attribute: %s", hipGetErrorString(e));
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.nwg), dim3(C::NTHR), C::BYTES, st, p);
  return check_launch("dsa_paged_latent_mla_fwd");
}

template <bool FP4>
static int launch_nt(const PagedParams &p, int64_t d_qk, int nt, hipStream_t st) {
  if (d_qk == 128) return launch<128, 64, 2, 4, FP4>(p, st);
  if (nt == 1) return launch<576, 512, 1, 4, FP4>(p, st);
  return nt == 4 ? launch<576, 512, 4, 8, FP4>(p, st) : launch<576, 512, 2, 8, FP4>(p, st);
}

int launch_paged_fwd(PagedParams p, int64_t d_qk, int64_t d_v, bool fp4, unsigned char *ws, hipStream_t st) {
  const PagedSections s = paged_sections(p.T, p.R, p.W, p.block, p.H, d_qk, d_v);
  const PagedPlan k = paged_plan(p.T, p.R, p.W, p.block, p.H, d_qk);
  p.unit_rows = k.unit_rows;
  p.max_units = k.max_units;
  p.nwg = k.nwg;
  p.min_blocks = k.min_blocks;
  p.unit0 = (int32_t *)(ws + s.unit0);
  p.unit_req = (int32_t *)(ws + s.unit_req);
  p.unit_first = (int32_t *)(ws + s.unit_first);
  p.unit_at = (int32_t *)(ws + s.unit_at);
  p.part_ml = (float *)(ws + s.part_ml);
  p.part_o = (float *)(ws + s.part_o);
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(1024), 0, st, p);
  int rc = check_launch("dsa_paged_latent_mla_fwd (plan)");
  if (rc) return rc;
  rc = k.few ? launch_paged_few(p, d_qk, k.few, fp4, st) : (fp4 ? launch_nt<true>(p, d_qk, k.nt, st) : launch_nt<false>(p, d_qk, k.nt, st));
  if (rc || p.nwg == 1) return rc;  // one workgroup: no unit has several pieces
  const dim3 grid((unsigned)((p.T * p.H + 3) / 4));
  if (d_v == 512) hipLaunchKernelGGL(paged_combine_kernel<512>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(paged_combine_kernel<64>, grid, dim3(256), 0, st, p);
  return check_launch("dsa_paged_latent_mla_fwd (combine)");
}

}  // namespace dsa
