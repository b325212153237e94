// Layer norm over the last axis, forward and backward, on gfx950 (bf16 or f32 rows).
//
//   y = (x - mean) rstd weight + bias,   rstd = (mean((x - mean)^2) + eps)^-1/2
//   g = dy weight,  xhat = (x - mean) rstd
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  dweight = sum dy xhat,  dbias = sum dy  (over rows)
//
// GL lanes have a row, 8 neighbouring elements a lane and chunk (CH chunks), all in registers, so the variance is that of
// the differences from the mean, the mean's own rounding is taken out of them, and the row is read once; the index keys' 64
// channels take 8 lanes, a hidden state's 4096 a wave forward and a workgroup backward.  Rows need no alignment beyond their
// elements': the loads and stores are 16 bytes wide wherever a row begins.
// The backward adds a lane's columns over the rows that it meets, then its workgroup's lanes in order through LDS, and
// layer_norm_reduce_kernel the workgroups' sums: no atomics, the order depends on the sizes alone.  A lane adds kNormRun rows at
// most before its sum joins the workgroup's, whose roundings are kept beside it: a column of any length is off by 256 steps of
// the sum of its magnitudes at most (128 rows, 32 lanes, 32 and 16 workgroups' sums).  The backward has its next row in flight
// while it works on one, and one exchange between a row's lanes for both of its sums (135 -> 86 us at 4096).
//
// Bound by the bytes moved, or by a launch's own time: 16384 rows of 4096 bf16, forward, backward, sums: 60 us (4.5 TB/s),
// 83 (4.9), 5.6; 2051 rows of 1001 f32: 6.4, 10.7, 4.0; 8192 rows of 64 bf16: 3.2, 4.7, 3.1.  The backward of more than 8192 columns
// spills 119 (bf16) and 171 (f32) registers, part of them read in each row (weights, sums and two rows of 16 elements a lane do not
// fit into 128): 4096 rows of 16384 135 us (3.0 TB/s) and 265 (3.0), of 12288 124 and 230, of 8192 48 (4.2) and 83 (4.9).  Results
// stored past the caches make these calls shorter and what reads the results longer: 16384 rows of 4096, both directions 147 -> 128
// us, but the forward and a kernel that reads y 98 -> 106 (of 32768 rows 195 -> 199).
#include <math.h>

#include "dsa_common.hpp"
#include "wave_ops.hpp"

namespace dsa {

struct NormParams {
  const unsigned char *x, *dy;
  const void *weight, *bias;
  unsigned char *y, *dx;     // dense
  float *mean, *rstd;        // [rows]
  float *part;               // [nwg][2][n] sums of dy xhat and dy, or null
  float *low;                // the same of what their additions rounded away, or null
  void *dweight, *dbias;     // nwg == 1: written at once
  int64_t rows, x_stride, dy_stride;  // strides in elements
  int n, w_f32, nwg;
  float eps, inv_n;
};

// 16 bytes wherever an element may begin
typedef int u16x16b __attribute__((ext_vector_type(4), aligned(2)));
typedef int f32x16b __attribute__((ext_vector_type(4), aligned(4)));

// 8 neighbouring elements as they lie in memory; those past `left` are zeros.
template <bool F32>
struct Raw8 {
  i32x4 v[F32 ? 2 : 1];
};
template <bool F32>
__device__ __forceinline__ Raw8<F32> load_raw(const unsigned char *p, int left) {
  Raw8<F32> r;
  if (left >= 8) {
    if constexpr (F32) {
      r.v[0] = *reinterpret_cast<const f32x16b *>(p);
      r.v[1] = *reinterpret_cast<const f32x16b *>(p + 16);
    } else {
      r.v[0] = *reinterpret_cast<const u16x16b *>(p);
    }
    return r;
  }
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i >> 2][i & 3] = i < left ? reinterpret_cast<const int *>(p)[i] : 0;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < left ? reinterpret_cast<const uint16_t *>(p)[2 * i] : 0u;
      const uint32_t hi = 2 * i + 1 < left ? reinterpret_cast<const uint16_t *>(p)[2 * i + 1] : 0u;
      r.v[0][i] = (int)(lo | hi << 16);
    }
  }
  return r;
}
template <bool F32>
__device__ __forceinline__ void widen(const Raw8<F32> &r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (F32) v[i] = __int_as_float(r.v[i >> 2][i & 3]);
    else v[i] = __uint_as_float((i & 1) ? (uint32_t)r.v[0][i >> 1] & 0xffff0000u : (uint32_t)r.v[0][i >> 1] << 16);
  }
}
template <bool F32>
__device__ __forceinline__ void load_8(const unsigned char *p, int left, float (&v)[8]) {
  widen<F32>(load_raw<F32>(p, left), v);
}
template <bool F32>
__device__ __forceinline__ void store_8(unsigned char *p, int left, const float (&v)[8]) {
  if (left >= 8) {
    if constexpr (F32) {
      *reinterpret_cast<f32x16b *>(p) = f32x16b{__float_as_int(v[0]), __float_as_int(v[1]), __float_as_int(v[2]), __float_as_int(v[3])};
      *reinterpret_cast<f32x16b *>(p + 16) = f32x16b{__float_as_int(v[4]), __float_as_int(v[5]), __float_as_int(v[6]), __float_as_int(v[7])};
    } else {
      *reinterpret_cast<u16x16b *>(p) = u16x16b{(int)pack_bf16x2(v[0], v[1]), (int)pack_bf16x2(v[2], v[3]),
                                                (int)pack_bf16x2(v[4], v[5]), (int)pack_bf16x2(v[6], v[7])};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) {
      if constexpr (F32) reinterpret_cast<float *>(p)[i] = v[i];
      else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)pack_bf16x2(v[i], 0.0f);
    }
}
// weight or bias of 8 columns (none: `value`)
__device__ __forceinline__ void load_param(const void *w, int f32, int col, int left, float value, float (&v)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = value;
  } else if (f32) {
    load_8<true>(static_cast<const unsigned char *>(w) + (int64_t)col * 4, left, v);
  } else {
    load_8<false>(static_cast<const unsigned char *>(w) + (int64_t)col * 2, left, v);
  }
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float(wv::dpp<CTRL>(__float_as_uint(v)));
}
__device__ __forceinline__ float sum_rows16(float x) {  // x(lane) + x(lane ^ 16)
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sums over the GL lanes of a row, in each of them.  GL > 64: the whole workgroup through tmp [N][GL / 64], one barrier.
template <int GL, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float *tmp) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = add_dpp<0xB1>(v[i]);   // quad_perm [1,0,3,2]
    v[i] = add_dpp<0x4E>(v[i]);   // quad_perm [2,3,0,1]
    v[i] = add_dpp<0x141>(v[i]);  // row_half_mirror
    if constexpr (GL >= 16) v[i] = add_dpp<0x140>(v[i]);  // row_mirror
    if constexpr (GL >= 32) v[i] = sum_rows16(v[i]);
    if constexpr (GL >= 64) v[i] = sum_halves(v[i]);
  }
  if constexpr (GL > 64) {
    constexpr int NW = GL / 64;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane_id() == 0) tmp[i * NW + wave_id()] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; ++k) v[i] += tmp[i * NW + k];
    }
  }
}

template <int GL>
struct NormGroup {
  static constexpr int NTHR = GL > 256 ? GL : 256, RPW = NTHR / GL, NW = GL / 64;  // threads; rows at once; waves of a row
};

template <int GL, int CH, bool F32>
__global__ void __launch_bounds__((NormGroup<GL>::NTHR)) layer_norm_fwd_kernel(const NormParams p) {
#pragma clang fp contract(off)  // (the first mean is a rounded one: fused into the differences it would be another there)
  using C = NormGroup<GL>;
  constexpr int ELT = F32 ? 4 : 2;
  __shared__ float tmp[3][GL > 64 ? C::NW : 1];
  const int gl = (int)threadIdx.x % GL;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * C::RPW + (int)threadIdx.x / GL;
  const bool there = row < p.rows;  // (whole rows of lanes)
  float v[CH][8], sum = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = 8 * (gl + GL * c);
    load_8<F32>(p.x + ((there ? row : 0) * p.x_stride + col) * ELT, p.n - col, v[c]);
    float part = 0.0f;  // (chunk by chunk: 64 elements one after the other would lose up to as many steps of the sum)
#pragma unroll
    for (int i = 0; i < 8; ++i) part += v[c][i];
    sum += part;
  }
  float total[1] = {sum};
  row_sums<GL>(total, tmp[0]);
  const float mean0 = total[0] * p.inv_n;
  // mean0's error, some steps of its last bit, would stand in every difference: it is the differences' own mean
  float rest = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[c][i] = 8 * (gl + GL * c) + i < p.n ? v[c][i] - mean0 : 0.0f;
      part += v[c][i];
    }
    rest += part;
  }
  total[0] = rest;
  row_sums<GL>(total, tmp[1]);
  rest = total[0] * p.inv_n;
  const float mean = mean0 + rest;
  float sq = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[c][i] = 8 * (gl + GL * c) + i < p.n ? v[c][i] - rest : 0.0f;
      part = fmaf(v[c][i], v[c][i], part);
    }
    sq += part;
  }
  total[0] = sq;
  row_sums<GL>(total, tmp[2]);
  const float rstd = 1.0f / sqrtf(total[0] * p.inv_n + p.eps);
  if (!there) return;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = 8 * (gl + GL * c), left = p.n - col;
    if (left <= 0) continue;
    float w[8], b[8];
    load_param(p.weight, p.w_f32, col, left, 1.0f, w);
    load_param(p.bias, p.w_f32, col, left, 0.0f, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[c][i] = fmaf(v[c][i] * rstd, w[i], b[i]);
    store_8<F32>(p.y + (row * p.n + col) * ELT, left, v[c]);
  }
  if (gl == 0 && p.mean != nullptr) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
}

__device__ __forceinline__ void put_sum(void *dst, int f32, int col, float v) {
  if (f32) static_cast<float *>(dst)[col] = v;
  else static_cast<uint16_t *>(dst)[col] = (uint16_t)pack_bf16x2(v, 0.0f);
}

constexpr int kNormRun = 128;  // rows that a lane of the backward adds one after the other

template <int GL, int CH, bool F32>
__global__ void __launch_bounds__((NormGroup<GL>::NTHR)) layer_norm_bwd_kernel(const NormParams p) {
  using C = NormGroup<GL>;
  constexpr int ELT = F32 ? 4 : 2;
  __shared__ float tmp[2][GL > 64 ? 2 * C::NW : 1];
  __shared__ float sums[C::RPW * GL * CH * 8];
  const int gl = (int)threadIdx.x % GL, grp = (int)threadIdx.x / GL;
  const int64_t step = (int64_t)p.nwg * C::RPW;
  // a row, fetched while the one before it is worked on
  Raw8<F32> rx[CH], rg[CH];
  float mean, rstd;
  auto fetch = [&](int64_t row) {
    const bool there = row < p.rows;
    const int64_t r = there ? row : 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = 8 * (gl + GL * c), left = there ? p.n - col : 0;
      rx[c] = load_raw<F32>(p.x + (r * p.x_stride + col) * ELT, left);
      rg[c] = load_raw<F32>(p.dy + (r * p.dy_stride + col) * ELT, left);
    }
    mean = p.mean[r];
    rstd = p.rstd[r];
  };
  int64_t row = (int64_t)blockIdx.x * C::RPW + grp;
  fetch(row);
  float w[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = 8 * (gl + GL * c);
    load_param(p.weight, p.w_f32, col, p.n - col, 1.0f, w[c]);
  }
  const bool sums_wanted = p.part != nullptr || p.dweight != nullptr || p.dbias != nullptr;
  int turn = 0;
  for (bool first = true;; first = false) {
    float dw[CH][8], db[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[c][i] = db[c][i] = 0.0f;
    for (int run = 0; run < kNormRun && row - grp < p.rows; ++run, row += step, turn ^= 1) {
      const bool there = row < p.rows;
      const float r = rstd;
      float x[CH][8], g[CH][8], s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        widen<F32>(rx[c], x[c]);
        widen<F32>(rg[c], g[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[c][i] = there && 8 * (gl + GL * c) + i < p.n ? (x[c][i] - mean) * r : 0.0f;
          dw[c][i] = fmaf(g[c][i], x[c][i], dw[c][i]);
          db[c][i] += g[c][i];
          g[c][i] *= w[c][i];
          s[0] += g[c][i];
          s[1] = fmaf(g[c][i], x[c][i], s[1]);
        }
      }
      fetch(row + step);
      if (p.dx == nullptr) continue;  // (uniform)
      row_sums<GL>(s, tmp[turn]);     // (two places in turn: no wait for the readers)
      const float m1 = s[0] * p.inv_n, m2 = s[1] * p.inv_n;
      if (there) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int col = 8 * (gl + GL * c), left = p.n - col;
          if (left <= 0) continue;
#pragma unroll
          for (int i = 0; i < 8; ++i) g[c][i] = r * (g[c][i] - m1 - x[c][i] * m2);
          store_8<F32>(p.dx + (row * p.n + col) * ELT, left, g[c]);
        }
      }
    }
    const bool last = row - grp >= p.rows;  // (uniform)
    if (!sums_wanted) {
      if (last) return;
      continue;
    }
    // the workgroup's sums: its row groups in order
    int th = (int)threadIdx.x;
    asm("" : "+v"(th));  // (its addresses are made here, not held in registers through the rows)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[th / GL * GL * CH * 8 + 8 * (th % GL + GL * c) + i] = which ? db[c][i] : dw[c][i];
      __syncthreads();
      auto column = [&](int col) {
        float v = 0.0f;
        for (int k = 0; k < C::RPW; ++k) v += sums[k * GL * CH * 8 + col];
        return v;
      };
      const int64_t at = ((int64_t)blockIdx.x * 2 + which) * p.n;
      if (p.nwg == 1) {
        if (void *dst = which ? p.dbias : p.dweight)
          for (int col = th; col < p.n; col += C::NTHR) put_sum(dst, p.w_f32, col, column(col));
      } else if (p.low == nullptr) {
        for (int col = th; col < p.n; col += C::NTHR) p.part[at + col] = column(col);
      } else {
        for (int col = th; col < p.n; col += C::NTHR) {  // (a column is one thread's in every run)
          float v = column(col), low = 0.0f;
          if (!first) {
            const float had = p.part[at + col], sum = had + v, grown = sum - had;
            low = p.low[at + col] + ((had - (sum - grown)) + (v - grown));  // what the addition rounded away, exactly
            v = sum;
          }
          p.part[at + col] = v;
          p.low[at + col] = low;
        }
      }
    }
    if (last) return;
  }
}

// dweight (y = 0), dbias (y = 1): the workgroups' sums, 64 columns a workgroup, wave w those of w, w + 16, ..; nwg = 0: zeros.
__global__ void __launch_bounds__(1024) layer_norm_reduce_kernel(const NormParams p) {
  __shared__ float sums[16][64];
  const int lane = lane_id(), w = wave_id(), which = (int)blockIdx.y, col = (int)blockIdx.x * 64 + lane;
  void *dst = which ? p.dbias : p.dweight;
  if (dst == nullptr) return;
  float v = 0.0f;
  if (col < p.n) {
#pragma unroll 8
    for (int k = w; k < p.nwg; k += 16) v += p.part[((int64_t)k * 2 + which) * p.n + col];
    if (p.low != nullptr) {
      float low = 0.0f;
      for (int k = w; k < p.nwg; k += 16) low += p.low[((int64_t)k * 2 + which) * p.n + col];
      if (fabsf(low) < INFINITY) v += low;  // (not of a sum that is not finite)
    }
  }
  sums[w][lane] = v;
  __syncthreads();
  if (w != 0 || col >= p.n) return;
  for (int k = 1; k < 16; ++k) v += sums[k][lane];
  put_sum(dst, p.w_f32, col, v);
}

// Lanes of a row and chunks a lane, by the width.  The forward keeps up to 64 elements a lane, so that a wave has a row of
// 4096 and waits for no other; the backward, whose sums and weights stay in registers too, 16.
struct NormShape {
  int gl, ch;
};
static NormShape norm_shape(int64_t n, bool bwd) {
  if (n <= 512) return {n <= 64 ? 8 : n <= 128 ? 16 : n <= 256 ? 32 : 64, 1};
  if (n <= 1024) return {64, 2};
  if (bwd) return n <= 4096 ? NormShape{256, n <= 2048 ? 1 : 2} : NormShape{1024, n <= 8192 ? 1 : 2};
  if (n <= 4096) return {64, n <= 2048 ? 4 : 8};
  return {256, n <= 8192 ? 4 : 8};
}
constexpr int64_t kNormMost = 16384;
// Workgroups of the backward, whose sums cost 16 bytes a column, a row's step 6 to 12: as few as take no more turns than the most
// would (replays of forward and backward, the most and so, us: 2051 rows of 1001 f32 24.4, 23.0; 600 of 2048 f32 26.4, 24.4; 9000
// of 1001 f32 44.3, 45.1).
struct NormBwdPlan {
  int64_t nwg;
  bool runs;  // lanes add more rows than a run
  size_t bytes;
};
static NormBwdPlan norm_bwd_plan(int64_t rows, int64_t n) {
  const int gl = norm_shape(n, true).gl, rpw = gl > 256 ? 1 : 256 / gl;
  const int64_t steps = (rows + rpw - 1) / rpw, most = gl > 256 ? 256 : 512;
  const int64_t turns = (steps + most - 1) / most;
  NormBwdPlan k;
  k.nwg = steps <= most ? steps : (steps + turns - 1) / turns;
  k.runs = turns > kNormRun;
  k.bytes = k.nwg > 1 ? (size_t)k.nwg * 2 * (size_t)n * 4 * (k.runs ? 2 : 1) : 0;
  return k;
}

template <int GL, int CH>
static void launch_fwd(bool f32, const NormParams &p, hipStream_t st) {
  using C = NormGroup<GL>;
  const int64_t n = (p.rows + C::RPW - 1) / C::RPW, most = 1 << 20;  // (2^32 threads and more: not along one axis)
  const dim3 grid((unsigned)(n < most ? n : most), (unsigned)((n + most - 1) / most)), block(C::NTHR);
  if (f32) hipLaunchKernelGGL((layer_norm_fwd_kernel<GL, CH, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((layer_norm_fwd_kernel<GL, CH, false>), grid, block, 0, st, p);
}
template <int GL, int CH>
static void launch_bwd(bool f32, const NormParams &p, hipStream_t st) {
  const dim3 grid((unsigned)p.nwg), block(NormGroup<GL>::NTHR);
  if (f32) hipLaunchKernelGGL((layer_norm_bwd_kernel<GL, CH, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((layer_norm_bwd_kernel<GL, CH, false>), grid, block, 0, st, p);
}
static void launch_norm(bool bwd, bool f32, const NormParams &p, hipStream_t st) {
  const NormShape s = norm_shape(p.n, bwd);
  const int key = s.gl * 16 + s.ch;
  switch (key) {
    case 8 * 16 + 1: return bwd ? launch_bwd<8, 1>(f32, p, st) : launch_fwd<8, 1>(f32, p, st);
    case 16 * 16 + 1: return bwd ? launch_bwd<16, 1>(f32, p, st) : launch_fwd<16, 1>(f32, p, st);
    case 32 * 16 + 1: return bwd ? launch_bwd<32, 1>(f32, p, st) : launch_fwd<32, 1>(f32, p, st);
    case 64 * 16 + 1: return bwd ? launch_bwd<64, 1>(f32, p, st) : launch_fwd<64, 1>(f32, p, st);
    case 64 * 16 + 2: return bwd ? launch_bwd<64, 2>(f32, p, st) : launch_fwd<64, 2>(f32, p, st);
    case 64 * 16 + 4: return launch_fwd<64, 4>(f32, p, st);
    case 64 * 16 + 8: return launch_fwd<64, 8>(f32, p, st);
    case 256 * 16 + 4: return launch_fwd<256, 4>(f32, p, st);
    case 256 * 16 + 8: return launch_fwd<256, 8>(f32, p, st);
    case 256 * 16 + 1: return launch_bwd<256, 1>(f32, p, st);
    case 256 * 16 + 2: return launch_bwd<256, 2>(f32, p, st);
    case 1024 * 16 + 1: return launch_bwd<1024, 1>(f32, p, st);
    default: return launch_bwd<1024, 2>(f32, p, st);
  }
}

static int check_norm(const char *who, int64_t rows, int64_t n, int dtype, int w_dtype) {
  DSA_REQUIRE(rows >= 0 && rows < (1ll << 31) && n > 0, "%s: bad sizes rows=%lld n=%lld", who, (long long)rows, (long long)n);
  DSA_REQUIRE((dtype == DSA_DTYPE_BF16 || dtype == DSA_DTYPE_F32) && (w_dtype == DSA_DTYPE_BF16 || w_dtype == DSA_DTYPE_F32),
              "%s: rows and weights are bf16 or f32, got dtypes %d, %d", who, dtype, w_dtype);
  if (n > kNormMost)
    return set_error(DSA_ERR_UNSUPPORTED, "%s: rows of %lld elements (at most %lld)", who, (long long)n, (long long)kNormMost);
  return DSA_OK;
}
static bool aligned_to(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace dsa

using namespace dsa;

extern "C" int dsa_layer_norm_fwd(const void *x, const void *weight, const void *bias, void *y, float *mean, float *rstd, int64_t rows,
                                  int64_t n, int64_t x_stride, float eps, int dtype, int w_dtype, void *stream) {
  const char *who = "dsa_layer_norm_fwd";
  const int rc = check_norm(who, rows, n, dtype, w_dtype);
  if (rc) return rc;
  DSA_REQUIRE(isfinite(eps) && eps >= 0.0f, "%s: eps must be finite and not negative, got %g", who, (double)eps);
  DSA_REQUIRE(x_stride >= 0, "%s: negative row stride", who);
  if (rows == 0) return DSA_OK;
  const int elt = dtype == DSA_DTYPE_F32 ? 4 : 2, welt = w_dtype == DSA_DTYPE_F32 ? 4 : 2;
  DSA_REQUIRE(x && y && (mean == nullptr) == (rstd == nullptr), "%s: null pointer (mean and rstd come together)", who);
  DSA_REQUIRE(aligned_to(x, elt) && aligned_to(y, elt) && aligned_to(weight, welt) && aligned_to(bias, welt) && aligned_to(mean, 4) && aligned_to(rstd, 4),
              "%s: misaligned pointer", who);
  NormParams p{};
  p.x = (const unsigned char *)x;
  p.weight = weight;
  p.bias = bias;
  p.y = (unsigned char *)y;
  p.mean = mean;
  p.rstd = rstd;
  p.rows = rows;
  p.x_stride = x_stride;
  p.n = (int)n;
  p.w_f32 = w_dtype == DSA_DTYPE_F32;
  p.eps = eps;
  p.inv_n = 1.0f / (float)n;
  launch_norm(false, dtype == DSA_DTYPE_F32, p, (hipStream_t)stream);
  return check_launch(who);
}

extern "C" size_t dsa_layer_norm_bwd_workspace_size(int64_t rows, int64_t n) {
  if (check_norm("dsa_layer_norm_bwd_workspace_size", rows, n, DSA_DTYPE_F32, DSA_DTYPE_F32)) return 0;
  return norm_bwd_plan(rows, n).bytes;
}

extern "C" int dsa_layer_norm_bwd(const void *dy, const void *x, const void *weight, const float *mean, const float *rstd, void *dx,
                                  void *dweight, void *dbias, void *workspace, size_t workspace_bytes, int64_t rows, int64_t n,
                                  int64_t dy_stride, int64_t x_stride, int dtype, int w_dtype, void *stream) {
  const char *who = "dsa_layer_norm_bwd";
  const int rc = check_norm(who, rows, n, dtype, w_dtype);
  if (rc) return rc;
  DSA_REQUIRE(x_stride >= 0 && dy_stride >= 0, "%s: negative row stride", who);
  const int elt = dtype == DSA_DTYPE_F32 ? 4 : 2, welt = w_dtype == DSA_DTYPE_F32 ? 4 : 2;
  DSA_REQUIRE(rows == 0 || (dy && x && mean && rstd), "%s: null pointer", who);
  DSA_REQUIRE(aligned_to(dy, elt) && aligned_to(x, elt) && aligned_to(dx, elt) && aligned_to(weight, welt) && aligned_to(dweight, welt) &&
                  aligned_to(dbias, welt) && aligned_to(mean, 4) && aligned_to(rstd, 4),
              "%s: misaligned pointer", who);
  NormParams p{};
  p.dy = (const unsigned char *)dy;
  p.x = (const unsigned char *)x;
  p.weight = weight;
  p.mean = const_cast<float *>(mean);
  p.rstd = const_cast<float *>(rstd);
  p.dx = (unsigned char *)dx;
  p.dweight = dweight;
  p.dbias = dbias;
  p.rows = rows;
  p.x_stride = x_stride;
  p.dy_stride = dy_stride;
  p.n = (int)n;
  p.w_f32 = w_dtype == DSA_DTYPE_F32;
  p.inv_n = 1.0f / (float)n;
  const NormBwdPlan k = norm_bwd_plan(rows, n);
  p.nwg = (int)k.nwg;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (sums && p.nwg > 1) {
    if (workspace == nullptr || workspace_bytes < k.bytes || !aligned_to(workspace, 4))
      return set_error(DSA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, k.bytes, workspace_bytes);
    p.part = (float *)workspace;
    if (k.runs) p.low = p.part + k.nwg * 2 * n;
  }
  if (rows > 0 && (sums || dx != nullptr)) {
    launch_norm(true, dtype == DSA_DTYPE_F32, p, (hipStream_t)stream);
    const int rc2 = check_launch(who);
    if (rc2) return rc2;
  }
  if (!sums || p.nwg == 1) return DSA_OK;
  hipLaunchKernelGGL(layer_norm_reduce_kernel, dim3((unsigned)((n + 63) / 64), 2), dim3(1024), 0, (hipStream_t)stream, p);
  return check_launch("dsa_layer_norm_bwd (reduce)");
}
