// Latent attention over a paged cache, rows of 576 channels (512 latent): every wave holds
// 16 rows' Q (72 registers) and O (128), so two waves share a SIMD.
//
//   S^T[key][row] = K Q^T    on 16x16x32 MFMAs (lane = row, its keys in the registers)
//   running maximum and sum per lane (two exchanges a tile), P^T the operand as it stands
//   O^T[d][row] += V^T P^T   (V^T by transposed LDS reads)
// Steps of 64 keys (two 32-key tiles), one ahead in LDS, one barrier a step:
//   RG 8 (128 rows, bf16): all eight waves fetch and compute;
//   RG 4, 2: four waves compute (RG row groups x KG = 4 / RG key groups), the other four
//     bring the rows;
//   RG 1 (sparse attention): two key groups by two halves of V's channels, both with all of S.
// bf16 rows come by LDS-DMA loads; MXFP4 rows (a third of the bytes) by registers, two
// more steps ahead, converted to exact bf16 values as they are written to LDS.  At a
// piece's end the key groups' O are brought to one maximum and added pairwise through LDS.
//
// What bounds it: bf16 with up to 64 rows the reading of the cache, 143 us with plan and
// joining for 64 requests of 301 .. 16384 keys, 630 MB (4.8 TB/s in this kernel).  MXFP4
// with up to 32 rows the computing waves, one a SIMD: for 96 requests, 338 MB, the kernel
// takes 124 us, its loads alone 65, these with the conversion 84, the products alone 108.
// At 128 rows a wave reads every tile's K and V whole (70 KiB), which is 2176 cycles of LDS
// reads and as many of MFMAs a tile, against 135 us for the loads alone: 203 to 214 us.
// Two steps ahead in flight made that 248 us, the loads after the products 228.
#include "latent_mla.hpp"
#include "latent_paged.hpp"

namespace dsa {

constexpr int kWideKeys = 64;  // keys of a step

template <int RG_, bool FP4, bool SPARSE = false>
struct PagedWide {
  using Row = CacheRow<576, 512, FP4>;
  static constexpr int RG = RG_, ROWS = 16 * RG;
  static constexpr bool ROLES = RG < 8;                      // waves 4..7 bring the rows
  static constexpr int DG = RG == 1 ? 2 : 1;                 // groups of V's channels
  static constexpr int CW = ROLES ? 4 : 8, LW = ROLES ? 4 : 8, KG = CW / (RG * DG);  // computing, loading waves; key groups
  static constexpr int SUB = 2 / KG;                         // tiles of a computing wave
  static constexpr int PANELS = 9, TILE = PANELS * 4096, STEP = 2 * TILE;
  // Operands read at once (3, 4: registers spill among a step's products).  2: none does there; around a piece's joining, the
  // window's refill and a step with masked keys, MXFP4 with RG 2 spills 22, sparse 28, sparse bf16 with RG 2 22, sparse MXFP4 with
  // RG 4 and sparse bf16 with RG 8 2.
  static constexpr int GROUP = 2;
  static constexpr int KS = 18, NDT = 32 / DG;               // 16-channel tiles of O in a wave
  static constexpr int TPR = 4, CPT = 16 / TPR, RPT = 8 / TPR;  // MXFP4: threads of a row; their code pieces, rope chunks
  static constexpr int OFF_T = 2 * STEP;
  static constexpr int WINDOW = SPARSE ? 2 * kWindow : kWindow;
  static constexpr int OFF_ML = OFF_T + WINDOW * 4;          // [2][16][2]
  static constexpr int BYTES = OFF_ML + 2 * 16 * 8;
  static constexpr int O_BYTES = NDT * 16 * 16 * 4;
  static_assert(BYTES <= 159 * 1024 && (KG == 1 || RG * DG * O_BYTES <= OFF_T), "LDS");
  static_assert(!FP4 || (ROLES && 64 * LW == kWideKeys * TPR), "MXFP4 rows: by the loading waves");
};

template <int RG, bool FP4, bool SPARSE>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) paged_wide_kernel(const PagedParams p) {
  using C = PagedWide<RG, FP4, SPARSE>;
  using Row = typename C::Row;
  constexpr int KEYS = kWideKeys, KS = C::KS, NDT = C::NDT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int w = wave_id();
  const int rg = w % RG, kg = C::ROLES ? (w & 3) / RG % C::KG : 0, dg = C::DG > 1 ? (w & 3) / (RG * C::KG) : 0;
  const bool computes = !C::ROLES || w < 4;  // wave-uniform
  const int lw = C::ROLES ? w - 4 : w;       // loading wave
  int *window = reinterpret_cast<int *>(smem + C::OFF_T);
  float *ML = reinterpret_cast<float *>(smem + C::OFF_ML);
  const uint32_t lds0 = lds_address(smem);
  const unsigned char *zero = reinterpret_cast<const unsigned char *>(kZeroRow);
  // MXFP4: chunks are also permuted by their panel, as neighbouring lanes write one row's blocks, a panel to two of them
  auto panel_swz = [](int panel) { return FP4 ? (panel & 7) << 4 : 0; };
  // (sparse: a pick is its own page)
  auto page_of = [&](int key) { return SPARSE ? key : p.block_shift >= 0 ? key >> p.block_shift : (int)((uint32_t)key / (uint32_t)p.block); };

  int units, total;
  all_units<SPARSE>(p, units, total);
  const int per = uni(range_blocks(p, total));
  const int range = range_of<SPARSE>();
  if ((int64_t)range * per >= total) return;
  int at = range * per;
  const int end = per < total - at ? at + per : total;
  for (int u = uni(unit_of<SPARSE>(p, units, at)); at < end; ++u) {
    const PagedPiece x = next_piece<SPARSE>(p, u, at, end);
    const int tok0 = SPARSE ? 0 : x.first / p.H, tok1 = SPARSE ? 0 : (x.first + x.nrows - 1) / p.H;
    auto my_row = [&] { return 16 * rg + (lane_here() & 15); };  // of the unit
    // Tokens [ta, tb] with the keys cut at tb's: all at once, or, where that left something that is not finite, one by
    // one, since a weight of zero does not remove the Inf or NaN of a later token's key.
    int ta = tok0, tb = tok1;
    bool probe = tok0 != tok1;
    while (true) {
      const int lim = token_keys(x.kv, x.n, tb), lim_min = token_keys(x.kv, x.n, ta);
      int j1 = min(x.b1, (lim + KEYS - 1) / KEYS);  // steps past it hold no key
      auto row_keys = [&](int row) {
        if constexpr (SPARSE) return lim;
        const int t = (x.first + row) / p.H;
        return token_keys(x.kv, x.n, t < tb ? t : tb);
      };
      int base = 0;  // first page in the window
      bool all_there = true;
      auto refill = [&](int first_page) {
        base = first_page;
        const int pages = lim > 0 ? page_of(lim - 1) + 1 : 0;
        bool ok = true;
        __syncthreads();  // the window's readers are done
        if constexpr (SPARSE) {
          // the picks' slots: all positions, then all entries, so that two latencies are waited for
          constexpr int N = C::WINDOW / 512;
          int pos[N], e[N];
#pragma unroll
          for (int k = 0; k < N; ++k) pos[k] = p.picks.position(x.token, base + k * 512 + (int)threadIdx.x, x.seen);
#pragma unroll
          for (int k = 0; k < N; ++k) e[k] = p.picks.entry(x.req, pos[k]);
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int i = k * 512 + (int)threadIdx.x, slot = p.picks.slot(pos[k], e[k]);
            if (base + i < pages && slot < 0) ok = false;
            window[i] = slot;
          }
          all_there = __syncthreads_and(ok) != 0;
          return;
        }
        for (int i = (int)threadIdx.x; i < kWindow; i += 512) {
          int e = -1;
          if (base + i < pages) {
            e = x.table[base + i];
            if (e < 0 || e >= p.num_blocks) {
              e = -1;
              ok = false;
            }
          }
          window[i] = e;
        }
        all_there = __syncthreads_and(ok) != 0;
      };
      auto key_at = [&](int key) -> const unsigned char * {  // row of a key, by the window
        const int pg = page_of(key), e = key < lim ? window[pg - base] : -1;
        const int64_t slot = SPARSE ? e : (int64_t)e * p.block + (key - pg * p.block);
        return e >= 0 ? p.cache + slot * Row::BYTES : zero;
      };
      // bf16: a step's eight 8-row groups
      auto fetch = [&](int j, int buf) {
        const int ln = lane_here();
#pragma unroll
        for (int grp = lw; grp < 8; grp += C::LW) {
          const int r = 8 * grp + (ln >> 3);
          const unsigned char *src = key_at(j * KEYS + r) + ((ln & 7) ^ row_swz(r & 31)) * 16;
#pragma unroll
          for (int pn = 0; pn < C::PANELS; ++pn)
            dma_16_at(lds0 + (uint32_t)(buf * C::STEP + (grp >> 2) * C::TILE + pn * 4096 + (grp & 3) * 1024), src + pn * 128);
        }
      };
      // MXFP4: TPR neighbouring threads have a row: every TPR-th piece of codes (16 bytes, a 32-channel block) and rope
      // chunk of it, and all its exponents
      struct Raw {
        i32x4 codes[C::CPT], rope[C::RPT], expo;
      };
      auto load_raw = [&](Raw &raw, int j) {
        const int th = lw * 64 + lane_here(), key_of = th / C::TPR, part = th % C::TPR;
        const unsigned char *src = key_at(j * KEYS + key_of);
#pragma unroll
        for (int i = 0; i < C::CPT; ++i) raw.codes[i] = ld_row_16(src + (i * C::TPR + part) * 16);
        raw.expo = ld_row_16(src + Row::OFF_EXP);
#pragma unroll
        for (int i = 0; i < C::RPT; ++i) raw.rope[i] = ld_row_16(src + Row::OFF_ROPE + ((i * C::TPR + part) & 7) * 16);
      };
      auto store_raw = [&](const Raw &raw, int buf) {
        const int th = lw * 64 + lane_here(), key_of = th / C::TPR, part = th % C::TPR;
        unsigned char *tile = smem + buf * C::STEP + (key_of >> 5) * C::TILE;
#pragma unroll
        for (int i = 0; i < C::CPT; ++i) {
          const int blk = i * C::TPR + part;
          const uint32_t e = ((uint32_t)raw.expo[i] >> (8 * part)) & 255u;  // byte blk of the exponents
          const float sc = e8m0_scale(e);
          i32x4 v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = e2m1x8_to_bf16((uint32_t)raw.codes[i][c], sc);
          if (wv::ballot(e == 255u) != 0ull) {
            keep_branch();
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (e == 255u) v[c] = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<i32x4 *>(tile + (blk >> 1) * 4096 + (tile_byte(key_of & 31, 4 * (blk & 1) + c) ^ panel_swz(blk >> 1))) = v[c];
        }
#pragma unroll
        for (int i = 0; i < C::RPT; ++i)
          *reinterpret_cast<i32x4 *>(tile + 8 * 4096 + tile_byte(key_of & 31, (i * C::TPR + part) & 7)) = raw.rope[i];
      };

      // steps that are asked for before they are worked on, and their pages in the window
      constexpr int kAsked = FP4 ? 3 : 1;
      auto window_for = [&](int j) {
        if (page_of((j + kAsked + 1) * KEYS - 1) >= base + C::WINDOW && page_of(lim - 1) >= base + C::WINDOW) refill(page_of(j * KEYS));
      };
      refill(page_of(x.b0 * KEYS));
      if constexpr (SPARSE) {
        // behind the last pick that is there: no step (a top-k of few keys), where the window shows it
        if (!all_there && x.b1 * KEYS <= base + C::WINDOW) {
          int last = 0;
          for (int i = lane_here(); i < x.b1 * KEYS - base; i += 64)
            if (window[i] >= 0) last = base + i + 1;
          for (int k = 32; k >= 1; k >>= 1) last = max(last, __shfl_xor(last, k, 64));
          j1 = min(j1, uni((last + KEYS - 1) / KEYS));
        }
      }
      int buf = 0;
      bool again = false;
      if (computes) {  // (the registers of Q and O are these waves' alone)
        i32x4 q[KS];
        {
          const int row = my_row(), g16 = lane_here() >> 4;
          const unsigned char *src = (row < x.nrows ? p.q + (x.row0 + row) * 1152 : zero) + 16 * g16;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) q[ks] = ld_row_16(src + 64 * ks);
        }
        float m_run = kLeastMax, l_run = 0.0f;
        f32x4 o[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

        // this wave's tile K of a step, from key0
        auto tile_step = [&](const unsigned char *K, int key0) {
          // Row m of S^T's 16-key tile h is key 8 (m >> 2) + 4 h + (m & 3), so that lane group g16 holds keys
          // 8 g16 + 4 h + i: what the second product's operand wants of it.
          const int ln = lane_here(), g16 = ln >> 4, l16 = ln & 15;
          int ka[2][2], va[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 2; ++u) ka[h][u] = tile_byte(8 * (l16 >> 2) + 4 * h + (l16 & 3), 4 * u + g16);
          // operands in the order (k-step, h) of the first product, then of V^T's 16-channel tiles
          auto rows = [&](int i) {
            const int ks = i >> 1, h = i & 1;
            return *reinterpret_cast<const i32x4 *>(K + (ka[h][ks & 1] ^ panel_swz(ks >> 1)) + (ks >> 1) * 4096);
          };
          auto cols = [&](int dt) {
            const unsigned char *b = K + dg * (NDT / 4 * 4096) + (dt >> 2) * 4096;
            const i32x2 r0 = ds_read_tr16(b + (va[0][dt & 3] ^ panel_swz(dt >> 2)));
            const i32x2 r1 = ds_read_tr16(b + (va[1][dt & 3] ^ panel_swz(dt >> 2)));
            return i32x4{r0[0], r0[1], r1[0], r1[1]};
          };
          f32x4 s[2]{{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
          OperandsOf<C::GROUP> a0;
          load_group<KS * 2>(a0, 0, rows);
          stream_operands<KS * 2>(a0, rows, [&](int i, i32x4 a) {
            s[i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(q[i >> 1]), s[i & 1], 0, 0, 0);
            asm volatile("" : "+v"(s[i & 1]));  // here, not sunk to where the sum is needed
          });
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              va[h][u] = (tile_byte(8 * g16 + 4 * h + (l16 >> 2), 2 * u + ((l16 & 3) >> 1)) + (l16 & 1) * 8) ^ panel_swz(dg * (NDT / 4));
          load_group<NDT>(a0, 0, cols);
          __builtin_amdgcn_sched_barrier(0);
          if (!all_there || key0 + 32 > lim_min) {
            keep_branch();
            const int kl = key0 + (ln & 31), my_lim = row_keys(16 * rg + l16);
            const uint32_t there = (uint32_t)wv::ballot(kl < lim && window[page_of(kl) - base] >= 0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int k = 8 * g16 + e;
              if (!((there >> k) & 1u) || key0 + k >= my_lim) s[e >> 2][e & 3] = -INFINITY;
            }
          }
          float mx = s[0][0];
#pragma unroll
          for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
          mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = max_halves(mx) * p.sl2;
          if (wv::ballot(mx > m_run + 8.0f) != 0ull) {
            const float m_new = fmaxf(m_run, mx), alpha = exp2_fast(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
          }
          float e2[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            e2[e] = exp2_fast(fmaf(s[e >> 2][e & 3], p.sl2, -m_run));
            l_run += e2[e];
          }
          // the weights in bf16, the product's operand: each off by 2^-8 of itself at most, their sum is of the 32-bit ones (results
          // are 0.0020 of their size from those in 64 bits, whose own rounding to bf16 is 0.0017)
          const i32x4 pb{(int)pack_bf16x2(e2[0], e2[1]), (int)pack_bf16x2(e2[2], e2[3]), (int)pack_bf16x2(e2[4], e2[5]),
                         (int)pack_bf16x2(e2[6], e2[7])};
          stream_operands<NDT>(a0, cols, [&](int dt, i32x4 a) {
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(pb), o[dt], 0, 0, 0);
          });
        };

        auto compute = [&](int j, int buf) {
#pragma unroll
          for (int sub = 0; sub < C::SUB; ++sub) {
            const int tl = kg * C::SUB + sub, key0 = j * KEYS + tl * 32;
            if (key0 < lim) tile_step(smem + buf * C::STEP + tl * C::TILE, key0);
          }
        };
        if constexpr (C::ROLES) {
          for (int j = x.b0; j < j1; ++j) {
            window_for(j);
            __syncthreads();  // step j is whole
            compute(j, buf);
            buf ^= 1;
          }
        } else {
          if (x.b0 < j1) fetch(x.b0, 0);
          for (int j = x.b0; j < j1; ++j) {
            window_for(j);
            __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
            __syncthreads();      // step j is whole, the other buffer consumed
            fetch(j + 1, buf ^ 1);  // (past the last step: zeros)
            compute(j, buf);
            buf ^= 1;
          }
          __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // what was fetched past the last step has landed
        }
        if (probe) {
          bool bad = false;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= not_finite(o[dt][e]);
          again = __syncthreads_or(bad) != 0;
        }
        if (!again) {
          l_run += __shfl_xor(l_run, 16, 64);
          l_run = sum_halves(l_run);
          // the key groups' sums, pairwise: the upper half of them leave theirs for the lower half
#pragma unroll
          for (int half = C::KG / 2; half >= 1; half /= 2) {
            __syncthreads();
            const int lane = lane_here(), g16 = lane >> 4, l16 = lane & 15;
            if (kg >= half && kg < 2 * half) {
              const int slot = ((kg - half) * RG + rg) * C::DG + dg;
              unsigned char *dst = smem + slot * C::O_BYTES;
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<f32x4 *>(dst + (dt * 64 + lane) * 16) = o[dt];
              if (g16 == 0) {
                ML[(slot * 16 + l16) * 2] = m_run;
                ML[(slot * 16 + l16) * 2 + 1] = l_run;
              }
            }
            __syncthreads();
            if (kg < half) {
              const int slot = (kg * RG + rg) * C::DG + dg;
              const unsigned char *src = smem + slot * C::O_BYTES;
              const float m2 = ML[(slot * 16 + l16) * 2], l2 = ML[(slot * 16 + l16) * 2 + 1];
              // (a group without a key of the row has l = 0 and O = 0; a NaN sum joins)
              const float m_new = l2 == 0.0f ? m_run : (l_run == 0.0f ? m2 : fmaxf(m_run, m2));
              const float a1 = l_run == 0.0f ? 0.0f : exp2_fast(m_run - m_new), a2 = l2 == 0.0f ? 0.0f : exp2_fast(m2 - m_new);
              m_run = m_new;
              l_run = l_run * a1 + l2 * a2;
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt) o[dt] = o[dt] * a1 + a2 * *reinterpret_cast<const f32x4 *>(src + (dt * 64 + lane) * 16);
            }
          }
          const int rlo = ta * p.H - x.first, rhi = min((tb + 1) * p.H - x.first, x.nrows);  // rows of tokens [ta, tb]
          const int row = my_row(), g16 = lane_here() >> 4;
          if (kg == 0 && row >= rlo && row < rhi) {
            const bool none = row_keys(row) <= x.b0 * KEYS || l_run == 0.0f;  // no key of this piece
            const float inv = none ? 0.0f : 1.0f / l_run;
            const int64_t part = (int64_t)x.slot * C::ROWS + row;
            if (g16 == 0 && dg == 0) {
              if (x.whole) {
                p.lse[x.row0 + row] = none ? -INFINITY : log2f(l_run) + m_run;
              } else {
                p.part_ml[part * 2] = m_run;
                p.part_ml[part * 2 + 1] = none ? 0.0f : l_run;
              }
            }
            if (x.whole && !FP4) {
              // Two channel tiles at a time, neighbouring lane groups' halves swapped, so that a lane has eight channels of one: 1537
              // tokens, 128 heads, top-64 151 -> 139 us, 32 heads 90 -> 84 (MXFP4: 180 -> 165, but 70 -> 73 and 102 -> 105 with 2048).
              // Dense: 6 prompts of 40 .. 512 tokens on 600 .. 4096 keys, 128 heads 1373 -> 1241, 16 heads 216 -> 202; 32 of 16 .. 64 tokens
              // on 64 .. 200 keys 227 -> 208; 64 single tokens of 301 .. 16384 keys, 16 heads 148, 147.
              unsigned char *dst = reinterpret_cast<unsigned char *>(p.out + (x.row0 + row) * 512 + 16 * dg * NDT + 16 * (g16 & 1) + 8 * (g16 >> 1));
#pragma unroll
              for (int dt = 0; dt < NDT; dt += 2) {
                i32x4 v;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const auto r = __builtin_amdgcn_permlane16_swap(pack_bf16x2(o[dt][2 * c] * inv, o[dt][2 * c + 1] * inv),
                                                                  pack_bf16x2(o[dt + 1][2 * c] * inv, o[dt + 1][2 * c + 1] * inv), false, false);
                  v[c] = (int)r[0];
                  v[c + 2] = (int)r[1];
                }
                // a row without keys: 0, whatever its neighbours' keys left
                *reinterpret_cast<i32x4 *>(dst + 32 * dt) = none ? i32x4{0, 0, 0, 0} : v;
              }
            } else if (x.whole) {
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt)
                *reinterpret_cast<i32x2 *>(p.out + (x.row0 + row) * 512 + 16 * (dg * NDT + dt) + 4 * g16) =
                    none ? i32x2{0, 0} : i32x2{(int)pack_bf16x2(o[dt][0] * inv, o[dt][1] * inv), (int)pack_bf16x2(o[dt][2] * inv, o[dt][3] * inv)};
            } else if (!none) {
#pragma unroll
              for (int dt = 0; dt < NDT; ++dt)
                *reinterpret_cast<f32x4 *>(p.part_o + part * 512 + 16 * (dg * NDT + dt) + 4 * g16) = o[dt];
            }
          }
        }
      } else {
        if constexpr (C::ROLES && FP4) {
          Raw raw0, raw1;  // the steps after the one that is written next, in turn
          load_raw(raw0, x.b0);  // (where there is no step: zeros)
          load_raw(raw1, x.b0 + 1);
          store_raw(raw0, 0);
          load_raw(raw0, x.b0 + 2);
          for (int j = x.b0; j < j1; j += 2) {
            window_for(j);
            __syncthreads();        // step j is whole, the other buffer consumed
            store_raw(raw1, 1);     // step j + 1
            load_raw(raw1, j + 3);
            if (j + 1 >= j1) break;
            window_for(j + 1);
            __syncthreads();
            store_raw(raw0, 0);     // step j + 2
            load_raw(raw0, j + 4);
          }
        } else if constexpr (C::ROLES) {
          if (x.b0 < j1) fetch(x.b0, 0);
          for (int j = x.b0; j < j1; ++j) {
            window_for(j);
            __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
            __syncthreads();        // step j is whole, the other buffer consumed
            buf ^= 1;
            fetch(j + 1, buf);      // (past the last step: zeros)
          }
          __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
        }
        // the computing waves' barriers
        if (probe) again = __syncthreads_or(0) != 0;
        if (!again)
          for (int half = C::KG / 2; half >= 1; half /= 2) {
            __syncthreads();
            __syncthreads();
          }
      }
      __syncthreads();  // LDS is free again
      if (again) {
        probe = false;
        ta = tb = tok0;
        continue;
      }
      if (tb == tok1) break;
      ta = ++tb;
    }
  }
}

template <int RG, bool FP4, bool SPARSE>
static int launch(const PagedParams &p, hipStream_t st) {
  using C = PagedWide<RG, FP4, SPARSE>;
  const char *who = SPARSE ? "dsa_paged_sparse_mla_fwd" : "dsa_paged_latent_mla_fwd";
  const auto kernel = paged_wide_kernel<RG, FP4, SPARSE>;
  const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
  if (e != hipSuccess) return set_error(DSA_ERR_HIP, "%s: LDS attribute: %s", who, hipGetErrorString(e));
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.nwg), dim3(512), C::BYTES, st, p);
  return check_launch(who);
}

int paged_wide_keys() { return kWideKeys; }
int launch_paged_wide(const PagedParams &p, int tiles16, bool fp4, bool sparse, hipStream_t st) {
  if (sparse) {
    if (tiles16 == 1) return fp4 ? launch<1, true, true>(p, st) : launch<1, false, true>(p, st);
    if (tiles16 == 2) return fp4 ? launch<2, true, true>(p, st) : launch<2, false, true>(p, st);
    if (tiles16 == 4) return fp4 ? launch<4, true, true>(p, st) : launch<4, false, true>(p, st);
    return launch<8, false, true>(p, st);
  }
  if (fp4) return tiles16 == 2 ? launch<2, true, false>(p, st) : launch<4, true, false>(p, st);
  return tiles16 == 4 ? launch<4, false, false>(p, st) : launch<8, false, false>(p, st);
}

}  // namespace dsa
