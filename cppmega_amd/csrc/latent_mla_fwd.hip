// Dense latent attention forward on gfx950 MFMA (bf16): out = softmax(scale q k^T) v
// over each row's key window, with the row's log2 sum of exponentials.
//
// A workgroup of NW waves takes NW * RT * 32 rows (token, head) of one kv group and
// walks its keys in LDS tiles of 64, fetched one tile ahead by LDS-DMA loads (one
// barrier a tile).  A wave keeps RT * 32 rows of Q as MFMA operands; per 32 keys:
//   S^T[key][row] = K Q^T      (one row per lane, 16 keys in its registers, so the
//                               row maximum and sum need no lane exchange but one)
//   p = 2^(s - m), running m and l (log2 domain; m moves only when a score passes it
//                               by 2^8, so O is seldom rescaled)
//   O^T[d][row] += V^T P^T     (P rounded to bf16: its registers are the operand as
//                               they stand, V^T by transposed LDS reads)
// Sums, statistics and O are fp32.  P is rounded to nearest even for the matrix
// product; l sums the weights before that rounding.
//
// Bound by the MFMAs and the softmax beside them, which overlap across the two or three
// waves of a SIMD only.  Causal, 4096 tokens: 128 / 64 absorbed, batch 2, 32 heads, 222 us
// (930 TFLOP/s of the admitted pairs); 192 / 128 expanded, 128 heads, 707 us (970; 946 us when
// 336 bytes more of LDS left room for one workgroup a CU); a large product runs at 1173.
// Of these 5 and 20 us go to out_lo, what rounding took from out.
// 32 rows a wave (RT 1): with 64, Q, O, the scores and an operand group take 190 (128 / 64)
// to 290 registers (192 / 128), which leaves a SIMD two waves or one.
#include <type_traits>

#include "latent_mla.hpp"

namespace dsa {

template <int DK, int DN, int DV, int RT, int NW>
struct LatentFwd {
  static constexpr bool SHARED = DN == DK;             // V is the first DV columns of K's tile
  static constexpr int KP = DK / 64, NP = DN / 64, VP = DV / 64;
  static constexpr int K_BYTES = 2 * KP * 4096, V_BYTES = SHARED ? 0 : 2 * VP * 4096;
  static constexpr int BUF = K_BYTES + V_BYTES;
  static constexpr int ROWS = NW * RT * 32;
  static constexpr int BYTES = 2 * BUF;                // (the waves' spans lie in the first buffer before a tile does)
};

// OCC workgroups a CU.
template <int DK, int DN, int DV, int RT, int NW, int OCC>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC))) latent_fwd_kernel(const LatentParams p) {
  using C = LatentFwd<DK, DN, DV, RT, NW>;
  constexpr int KS = DK / 16, NDT = DV / 32;
  static_assert(NW == 4 && OCC * C::BYTES <= kLdsOfCu, "a wave a SIMD and workgroup; LDS of all of them (no static LDS beside it)");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const int nblk = (int)((p.rows + C::ROWS - 1) / C::ROWS);
  int64_t bg, index;
  spread_items(blockIdx.x, p.B * p.G, nblk, bg, index);
  const int64_t b = bg / p.G, g = bg - b * p.G;
  const int blk = nblk - 1 - (int)index;  // the causal mask's longest first
  int *span_lds = reinterpret_cast<int *>(smem);

  // this lane's rows
  int lo[RT], hi[RT];
  int64_t orow[RT];  // (b S + t) H + head, or -1
  i32x4 q[RT][KS];
  RowSpan span = no_rows();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int64_t row = (int64_t)blk * C::ROWS + (w * RT + rt) * 32 + l32;
    lo[rt] = hi[rt] = 0;
    orow[rt] = -1;
    if (row < p.rows) {
      const int64_t t = (int64_t)((uint32_t)row / (uint32_t)p.hpg);
      orow[rt] = (b * p.S + t) * p.H + g * p.hpg + (row - t * p.hpg);
      latent_window(p, b, t, lo[rt], hi[rt]);
      span_add(span, lo[rt], hi[rt]);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[rt][ks] = i32x4{0, 0, 0, 0};
      if (orow[rt] >= 0) q[rt][ks] = ld_global_16(p.q + (orow[rt] * DK + 16 * ks + 8 * g32) * 2);
    }
  }
  span = span_wave(span);  // of the wave: what it may skip and where it needs no mask
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
  __syncthreads();  // read: a tile may lie there
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
  float m_run[RT], l_run[RT];
  f32x16 o[RT][NDT];

  auto pass = [&](auto careful_t) {
    constexpr bool careful = decltype(careful_t)::value;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m_run[rt] = kLeastMax;
      l_run[rt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[rt][dt] = zero16();
    }
    if (t0 < t1) fetch(t0, 0);
    for (int tile = t0; tile < t1; ++tile) {
      const int buf = (tile - t0) & 1, k0 = tile * kKeyTile;
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's share of the tile
      __syncthreads();                     // the tile is whole; the other buffer is consumed
      if (tile + 1 < t1) fetch(tile + 1, buf ^ 1);
      const unsigned char *Kt = smem + buf * C::BUF, *Vt = C::SHARED ? Kt : Kt + C::K_BYTES;
      if (k0 >= span.hi || k0 + kKeyTile <= span.lo) continue;  // wave-uniform
      auto rows_of = [&](int sub) { return [=](int ks) { return row_read(Kt + sub * C::KP * 4096, ks); }; };
      Operands ka;
      load_group<KS>(ka, 0, rows_of(0));
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int ks0 = k0 + 32 * s;
        const bool whole = span.lo_max <= ks0 && span.hi_min >= ks0 + 32;
        const unsigned char *Vs = Vt + s * (C::SHARED ? C::KP : C::VP) * 4096;
        auto cols = [&](int i) { return col_read(Vs, i >> 1, i & 1); };
        f32x16 acc[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt] = zero16();
        stream_operands<KS>(ka, rows_of(s), [&](int ks, i32x4 a) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            acc[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(q[rt][ks]), acc[rt], 0, 0, 0);
        });
        // in flight beside the softmax: the first operands of its product with V, and of the next keys
        Operands va;
        load_group<2 * NDT>(va, 0, cols);
        if (s == 0) load_group<KS>(ka, 0, rows_of(1));
        __builtin_amdgcn_sched_barrier(0);
        if (!whole) {
          keep_branch();
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = ks0 + acc_row(i, g32);
              acc[rt][i] = key >= lo[rt] && key < hi[rt] ? acc[rt][i] : -INFINITY;
            }
        }
        i32x4 pb[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float mx = acc[rt][0];
#pragma unroll
          for (int i = 1; i < 16; ++i) mx = __builtin_elementwise_maximum(mx, acc[rt][i]);  // (fmaxf quiets operands first)
          mx = max_halves(mx) * p.sl2;
          if (wv::ballot(mx > m_run[rt] + 8.0f) != 0ull) {
            const float m_new = fmaxf(m_run[rt], mx), alpha = exp2_fast(m_run[rt] - m_new);
            m_run[rt] = m_new;
            l_run[rt] *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[rt][dt][i] *= alpha;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            acc[rt][i] = exp2_fast(fmaf(acc[rt][i], p.sl2, -m_run[rt]));
            l_run[rt] += acc[rt][i];
          }
          pack_operand(acc[rt], pb[rt]);
        }
        if (!careful || whole) {
          stream_operands<2 * NDT>(va, cols, [&](int i, i32x4 a) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              o[rt][i >> 1] =
                  __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(pb[rt][i & 1]), o[rt][i >> 1], 0, 0, 0);
          });
        } else {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            careful_product<NDT>(o[rt], acc[rt], Vs, [&](int r) { return ks0 + r >= lo[rt] && ks0 + r < hi[rt]; });
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
      for (int i = 0; i < 16; ++i) bad |= not_finite(o[rt][dt][i]);
  if (any_wave<NW>(bad, smem)) pass(std::true_type{});  // a masked Inf or NaN may have reached a row: once more, without it

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = sum_halves(l_run[rt]);
    const bool empty = hi[rt] <= lo[rt] || l == 0.0f;  // no key, or a score of -Inf with each: no weight
    const float inv = empty ? 0.0f : 1.0f / l;
    if (orow[rt] >= 0) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        i32x2 v[4], low[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // an empty row's O is 0 (or what a neighbour's NaN left): 0
            const float x = empty ? 0.0f : o[rt][dt][4 * m + 2 * e] * inv, y = empty ? 0.0f : o[rt][dt][4 * m + 2 * e + 1] * inv;
            const uint32_t two = pack_bf16x2(x, y);
            v[m][e] = (int)two;
            low[m][e] = (int)pack_bf16x2(x - __uint_as_float(two << 16), y - __uint_as_float(two & 0xffff0000u));
          }
        store_tile(p.out + orow[rt] * DV, dt, v, g32);
        if (p.out_lo != nullptr) store_tile(p.out_lo + orow[rt] * DV, dt, low, g32);
      }
      if (g32 == 0) p.lse[orow[rt]] = empty ? -INFINITY : log2f(l) + m_run[rt];
    }
  }
}

template <int DK, int DN, int DV, int RT, int NW, int OCC>
static int launch(const LatentParams &p, hipStream_t st) {
  using C = LatentFwd<DK, DN, DV, RT, NW>;
  const auto kernel = latent_fwd_kernel<DK, DN, DV, RT, NW, OCC>;
  const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, C::BYTES);
  if (e != hipSuccess) return set_error(DSA_ERR_HIP, "dsa_latent_mla_fwd: LDS attribute: %s", hipGetErrorString(e));
  const int64_t n = (p.rows + C::ROWS - 1) / C::ROWS * p.B * p.G;
  DSA_REQUIRE(n < (1ll << 31), "dsa_latent_mla_fwd: grid too large");
  hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(64 * NW), C::BYTES, st, p);
  return check_launch("dsa_latent_mla_fwd");
}

int launch_latent_fwd(const LatentParams &p, int64_t d_qk, int64_t d_v, bool expanded, hipStream_t st) {
  if (!expanded) {
    if (d_qk == 128 && d_v == 64) return launch<128, 128, 64, 1, 4, 3>(p, st);
    if (d_qk == 128 && d_v == 128) return launch<128, 128, 128, 1, 4, 2>(p, st);
    if (d_qk == 192 && d_v == 128) return launch<192, 192, 128, 1, 4, 2>(p, st);
  } else {
    if (d_qk == 192 && d_v == 128) return launch<192, 128, 128, 1, 4, 2>(p, st);
    if (d_qk == 128 && d_v == 64) return launch<128, 64, 64, 1, 4, 3>(p, st);
  }
  return set_error(DSA_ERR_UNSUPPORTED, "dsa_latent_mla_fwd: no %s kernel for d_qk=%lld d_v=%lld",
                   expanded ? "expanded" : "absorbed", (long long)d_qk, (long long)d_v);
}

}  // namespace dsa
