// SparseMLA over the paged latent cache, rows of 128 channels (64 latent), on gfx950.
//
// A unit is a token's 32 heads.  A wave walks 32 of its picks at a time: positions three blocks ahead, page entries two,
// rows one (in registers), so that no load waits for the one that it is reached by; the rows then lie in the wave's own
// LDS tile, MXFP4 ones widened to exact bf16 values:
//   S^T[pick][head] = K Q^T, O^T[channel][head] += V^T P^T   on 32x32x16 MFMAs (lane = head)
// Many tokens: a wave has a unit.  Fewer: the four waves of a workgroup share a unit's picks and are joined through LDS,
// and workgroups may share them as well, whose fp32 sums sparse_narrow_combine_kernel adds in order.
//
// Bound by the chain of a block (LDS, S, softmax, P V) at three waves a SIMD, nothing saturated: 6 prompts of 40 .. 512 tokens,
// 32 heads, top-256, MXFP4 21 us (of a CU's busy time VALU 31 %, MFMA 12 %, LDS 21 %); bf16 the same.  Rows two blocks ahead 27, four
// waves a SIMD (registers spill) 44, S in two accumulators 26, operands read in groups 28.  With a long top-k the same: 1537 tokens,
// 32 heads, top-1000, bf16 55 us; of a replay of 58, the rows' loads and their way into LDS alone 46, all but the loads 47 (VALU
// 35 %, MFMA 15 %, LDS 27 %; of 390 MB of rows 220 come from the L2s); up to 16 heads on 16x16x32 MFMAs at four waves a SIMD took 43 us against 46 here.  One
// token of 777 keys: 6.5.
#include "latent_mla.hpp"
#include "latent_paged.hpp"
#include "paged_sparse.hpp"

namespace dsa {

template <bool FP4>
struct NarrowRows {  // 32 rows on their way
  i32x4 v[FP4 ? 4 : 8];  // bf16: row 4 i + lane / 16, chunk lane % 16; MXFP4: rope chunk lane % 8 of row 8 i + lane / 8
  i32x4 codes;           // MXFP4: of row lane / 2, channels 32 (lane % 2) ..
  uint32_t expo;
};

template <bool FP4, int WPU>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) sparse_narrow_kernel(const SparseParams p) {
  using Row = CacheRow<128, 64, FP4>;
  __shared__ __attribute__((aligned(16))) unsigned char tiles[4][8192];
  __shared__ float ML[WPU > 1 ? 4 : 1][32][2];
  constexpr int UPG = 4 / WPU;  // units of a workgroup
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  unsigned char *K = tiles[w];
  const int64_t item = xcd_remap(blockIdx.x, gridDim.x);
  const int64_t unit = item / p.nsplit * UPG + w / WPU, units = (int64_t)p.picks.req.T * p.htiles;
  if (WPU == 1 && unit >= units) return;
  const int t = __builtin_amdgcn_readfirstlane((int)((unit < units ? unit : units - 1) / p.htiles));
  const int head0 = __builtin_amdgcn_readfirstlane((int)(unit % p.htiles)) * 32;
  const int r = __builtin_amdgcn_readfirstlane(p.picks.req.of(t)), lim = __builtin_amdgcn_readfirstlane(p.picks.req.keys_of(t, r));
  const bool nobody = unit >= units || lim < 0;  // (a token of no request)
  if (WPU == 1 && nobody) return;
  // this wave's blocks of picks
  const int nb = (p.picks.topk + 31) / 32, parts = WPU * p.nsplit;
  const int part = (int)(item % p.nsplit) * WPU + w % WPU;
  const int b0 = (int)((int64_t)nb * part / parts), b1 = nobody ? b0 : (int)((int64_t)nb * (part + 1) / parts);

  auto pick = [&](int b) { return p.picks.position(t, 32 * b + l32, lim); };  // of the lane in block b
  const unsigned char *zero = reinterpret_cast<const unsigned char *>(kZeroRow);
  auto row_at = [&](int slot) { return slot >= 0 ? p.cache + (int64_t)slot * Row::BYTES : zero; };
  auto load = [&](NarrowRows<FP4> &x, int slot) {
    if constexpr (FP4) {
      const unsigned char *src = row_at(__shfl(slot, lane >> 1, 64));
      x.codes = ld_row_16(src + (lane & 1) * 16);
      x.expo = ld_row_1(src + Row::OFF_EXP + (lane & 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = ld_row_16(row_at(__shfl(slot, 8 * i + (lane >> 3), 64)) + Row::OFF_ROPE + (lane & 7) * 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x.v[i] = ld_row_16(row_at(__shfl(slot, 4 * i + (lane >> 4), 64)) + (lane & 15) * 16);
    }
  };
  auto put = [&](const NarrowRows<FP4> &x) {
    if constexpr (FP4) {
      const float s = e8m0_scale(x.expo);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        i32x4 v = e2m1x8_to_bf16((uint32_t)x.codes[c], s);
        if (x.expo == 255u) v = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
        *reinterpret_cast<i32x4 *>(K + tile_byte(lane >> 1, 4 * (lane & 1) + c)) = v;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<i32x4 *>(K + 4096 + tile_byte(8 * i + (lane >> 3), lane & 7)) = x.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<i32x4 *>(K + ((lane >> 3) & 1) * 4096 + tile_byte(4 * i + (lane >> 4), lane & 7)) = x.v[i];
    }
  };

  float m_run = kLeastMax, l_run = 0.0f;
  f32x16 o[2] = {zero16(), zero16()};
  if (b0 < b1) {
    NarrowRows<FP4> rows;
    int pos0 = pick(b0), pos1 = pick(b0 + 1), pos2 = pick(b0 + 2);
    i32x4 q[8];
    {
      const unsigned char *src = (head0 + l32 < p.H ? p.q + ((int64_t)t * p.H + head0 + l32) * 256 : zero) + 16 * g32;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) q[ks] = ld_row_16(src + 32 * ks);
    }
    const int slot0 = p.picks.slot(pos0, p.picks.entry(r, pos0));
    int ent1 = p.picks.entry(r, pos1);
    uint32_t there = (uint32_t)wv::ballot(slot0 >= 0);
    load(rows, slot0);
    const RowRead row_read;
    const ColRead col_read;
    for (int b = b0; b < b1; ++b) {
      put(rows);
      const uint32_t vm = there;
      const int slot = p.picks.slot(pos1, ent1);
      there = (uint32_t)wv::ballot(slot >= 0);
      load(rows, slot);  // (past the last block: rows that are not used)
      pos1 = pos2;
      ent1 = p.picks.entry(r, pos1);
      pos2 = pick(b + 3);
      wave_lds_sync();
      if (vm != 0u) {
        f32x16 acc = zero16();
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(row_read(K, ks)), as_bf16x8(q[ks]), acc, 0, 0, 0);
        if (vm != 0xffffffffu) {
          keep_branch();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!((vm >> acc_row(i, g32)) & 1u)) acc[i] = -INFINITY;
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
          for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[i] = exp2_fast(fmaf(acc[i], p.sl2, -m_run));
          l_run += acc[i];
        }
        i32x4 pb[2];
        pack_operand(acc, pb);  // (weights in bf16, the product's operand: off by 2^-8 of themselves at most; their sum is of the 32-bit ones)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(col_read(K, dt, u)), as_bf16x8(pb[u]), o[dt], 0, 0, 0);
      }
      wave_lds_sync();  // the tile is read: it may be written again
    }
    l_run = sum_halves(l_run);
  }
  const int head = head0 + l32;
  const int64_t row = (int64_t)t * p.H + head;
  if constexpr (WPU == 1) {
    if (head >= p.H) return;
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
      i32x2 v[4];
#pragma unroll
      for (int m = 0; m < 4; ++m)
        v[m] = i32x2{(int)pack_bf16x2(o[dt][4 * m] * inv, o[dt][4 * m + 1] * inv), (int)pack_bf16x2(o[dt][4 * m + 2] * inv, o[dt][4 * m + 3] * inv)};
      store_tile(p.out + row * 64, dt, v, g32);  // (head is the same in both lane halves)
    }
    if (g32 == 0) p.lse[row] = l_run == 0.0f ? -INFINITY : log2f(l_run) + m_run;
  } else {
    // the waves' sums, in order
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int m = 0; m < 4; ++m)
        *reinterpret_cast<f32x4 *>(K + ((dt * 4 + m) * 64 + lane) * 16) = f32x4{o[dt][4 * m], o[dt][4 * m + 1], o[dt][4 * m + 2], o[dt][4 * m + 3]};
    if (g32 == 0) {
      ML[w][l32][0] = m_run;
      ML[w][l32][1] = l_run;
    }
    __syncthreads();
    if (nobody || head >= p.H) return;
    const int w0 = w / WPU * WPU;
    float m = kLeastMax, l = 0.0f, a[WPU];
#pragma unroll
    for (int k = 0; k < WPU; ++k)
      if (ML[w0 + k][l32][1] != 0.0f) m = fmaxf(m, ML[w0 + k][l32][0]);
#pragma unroll
    for (int k = 0; k < WPU; ++k) {
      const float lk = ML[w0 + k][l32][1];
      a[k] = lk == 0.0f ? 0.0f : exp2_fast(ML[w0 + k][l32][0] - m);  // (no pick of the wave: its O is 0; a NaN sum joins)
      l += lk * a[k];
    }
    const bool whole = p.nsplit == 1;
    const int64_t part_row = (unit * p.nsplit + item % p.nsplit) * 32 + l32;
    const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 8 / WPU; ++i) {
      const int dm = 8 / WPU * (w - w0) + i, col = acc_col(dm >> 2, 4 * (dm & 3), g32);
      f32x4 x{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < WPU; ++k) x += a[k] * *reinterpret_cast<const f32x4 *>(tiles[w0 + k] + (dm * 64 + lane) * 16);
      x *= inv;
      if (whole) *reinterpret_cast<i32x2 *>(p.out + row * 64 + col) = i32x2{(int)pack_bf16x2(x[0], x[1]), (int)pack_bf16x2(x[2], x[3])};
      else *reinterpret_cast<f32x4 *>(p.part_o + part_row * 64 + col) = x;
    }
    if (w == w0 && g32 == 0) {
      if (whole) {
        p.lse[row] = l == 0.0f ? -INFINITY : log2f(l) + m;
      } else {
        p.part_ml[part_row * 2] = m;
        p.part_ml[part_row * 2 + 1] = l;
      }
    }
  }
}

// 16 lanes a (token, head): its splits' sums brought to their largest maximum and added in order.
__global__ void __launch_bounds__(256) sparse_narrow_combine_kernel(const SparseParams p) {
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (row >= (int64_t)p.picks.req.T * p.H) return;
  const int64_t t = row / p.H;
  const int head = (int)(row - t * p.H), c = (int)(threadIdx.x & 15) * 4;
  if (p.picks.req.keys_of((int)t, p.picks.req.of_lane((int)t)) < 0) return;
  const int64_t at = (t * p.htiles + head / 32) * p.nsplit * 32 + head % 32;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 *ml = reinterpret_cast<const f32x2 *>(p.part_ml) + at;
  float m = kLeastMax, l = 0.0f;
#pragma unroll 8
  for (int s = 0; s < p.nsplit; ++s) {
    const f32x2 x = ml[32 * s];
    m = x[1] != 0.0f ? fmaxf(m, x[0]) : m;
  }
  f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int s = 0; s < p.nsplit; ++s) {
    const f32x2 x = ml[32 * s];
    const float a = x[1] == 0.0f ? 0.0f : exp2_fast(x[0] - m);
    l += x[1] * a;
    o += a * *reinterpret_cast<const f32x4 *>(p.part_o + (at + 32 * s) * 64 + c);
  }
  o *= l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<i32x2 *>(p.out + row * 64 + c) = i32x2{(int)pack_bf16x2(o[0], o[1]), (int)pack_bf16x2(o[2], o[3])};
  if (c == 0) p.lse[row] = l == 0.0f ? -INFINITY : log2f(l) + m;
}

// How a call is run: waves of a unit, workgroups that share it.  Replays of n tokens, 32 heads, one and four waves a unit, us:
// top-128: n = 768 17, 16; 1000 17, 20; 1300 19, 25; top-256: 768 20, 18; 1000 21, 23; 1300 25, 29; top-512: 1000 31, 28;
// 1300 37, 36; top-1000: 1300 60, 50; top-2048: 64 (four waves of eight workgroups) 76, 21; 1000 82, 62; 1656 100, 103.
// (Two waves a unit: between the two, or behind both.)
struct NarrowPlan {
  int wpu, nsplit;
};
static NarrowPlan narrow_plan(int64_t T, int64_t topk, int64_t H) {
  const int64_t units = T * ((H + 31) / 32), nb = (topk + 31) / 32;
  if (units >= (nb <= 8 ? 900 : 1536)) return {1, 1};
  int64_t ns = 512 / units;               // two workgroups a CU (three, top-2048: 128 tokens 28 us, two 25; 320 44, 39)
  if (ns > nb / 8) ns = nb / 8;           // two blocks a wave at least
  return {4, (int)(ns < 1 ? 1 : ns)};
}
size_t sparse_narrow_workspace(int64_t T, int64_t topk, int64_t H) {
  const NarrowPlan k = narrow_plan(T, topk, H);
  return k.nsplit == 1 ? 0 : (size_t)(T * ((H + 31) / 32)) * (size_t)k.nsplit * 32 * (64 + 2) * 4;
}

template <bool FP4>
static void launch_as(const SparseParams &p, int wpu, int64_t n, hipStream_t st) {
  if (wpu == 1) hipLaunchKernelGGL((sparse_narrow_kernel<FP4, 1>), dim3((unsigned)n), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((sparse_narrow_kernel<FP4, 4>), dim3((unsigned)n), dim3(256), 0, st, p);
}
int launch_sparse_narrow(SparseParams p, bool fp4, unsigned char *ws, hipStream_t st) {
  const NarrowPlan k = narrow_plan(p.picks.req.T, p.picks.topk, p.H);
  p.htiles = (p.H + 31) / 32;
  p.nsplit = k.nsplit;
  const int64_t units = (int64_t)p.picks.req.T * p.htiles, n = (units * k.wpu + 3) / 4 * k.nsplit;
  p.part_o = (float *)ws;
  p.part_ml = p.part_o + units * k.nsplit * 32 * 64;
  if (fp4) launch_as<true>(p, k.wpu, n, st);
  else launch_as<false>(p, k.wpu, n, st);
  const int rc = check_launch("dsa_paged_sparse_mla_fwd");
  if (rc || k.nsplit == 1) return rc;
  hipLaunchKernelGGL(sparse_narrow_combine_kernel, dim3((unsigned)(((int64_t)p.picks.req.T * p.H + 15) / 16)), dim3(256), 0, st, p);
  return check_launch("dsa_paged_sparse_mla_fwd (combine)");
}

}  // namespace dsa
