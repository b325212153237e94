// Rows into and out of the paged latent cache, and the plan of a serving step, on gfx950.
//
// latent_cache_append_kernel / latent_cache_gather_kernel: one thread per 8 channels of a
// row (16 bytes of bf16), both bound by the bytes they move.  MXFP4: the four neighbouring
// lanes of a 32-channel block share its largest magnitude; the scale is the power of two
// 2^(floor(log2 amax) - 2) (so the block's largest lands in [4, 8), of which what passes 6,
// the largest e2m1 value, saturates), the codes are rounded to nearest, ties to even.
//
// latent_plan_kernel: block table, slots, positions and lengths of a step, from the
// requests' lengths.  Every workgroup runs the same prefix sums over all requests (a few
// hundred integers) and writes what belongs to its own ones, so the plan is one launch.
//
// 16384 rows of 576 channels into MXFP4 pages 11 us, back 7.6 (26 MB each: 2.3, 3.4 TB/s,
// the launch among it); the plan of 16 requests 6.7 us, of 768 with 16384 tokens 15:
// latencies of the prefix sums, one after the other.
#include "latent_cache.hpp"

namespace dsa {

struct AppendParams {
  unsigned char *cache;
  const unsigned char *latent, *rope;
  int64_t latent_t, rope_t;  // row strides in bytes
  const int64_t *slots;
  int64_t T, num_slots;
};

template <int D_QK, int D_V, bool FP4>
__global__ void __launch_bounds__(256) latent_cache_append_kernel(const AppendParams p) {
  using Row = CacheRow<D_QK, D_V, FP4>;
  constexpr int CH = D_QK / 8, CV = D_V / 8;  // chunks of a row, of its latent part; both whole quads of lanes
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = id / CH;
  const int c = (int)(id - t * CH);
  if (t >= p.T) return;  // (whole quads)
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.num_slots) return;
  const i32x4 v = c < CV ? ld_global_16(p.latent + t * p.latent_t + c * 16) : ld_global_16(p.rope + t * p.rope_t + (c - CV) * 16);
  unsigned char *row = p.cache + slot * Row::BYTES;
  if (!FP4 || c >= CV) {
    *reinterpret_cast<i32x4 *>(row + (c < CV ? 0 : Row::OFF_ROPE - CV * 16) + c * 16) = v;
    return;
  }
  uint32_t top = 0;  // largest magnitude (bits: their order is the values')
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t u = (uint32_t)v[e];
    top = max(top, max((u << 16) & 0x7fff0000u, u & 0x7fff0000u));
  }
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  const bool bad = top >= 0x7f800000u;
  int ex = (int)(top >> 23) - 127 - 2;
  ex = ex < -125 ? -125 : ex;  // (at most 127 - 2)
  if (top == 0 || bad) ex = 0;
  const float inv = bad ? 0.0f : __uint_as_float((uint32_t)(127 - ex) << 23);
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = (uint32_t)v[e >> 1], h = (e & 1) ? u & 0xffff0000u : u << 16;
    const float a = bad ? 0.0f : __uint_as_float(h & 0x7fffffffu) * inv;
    // 0 0.5 1 1.5 2 3 4 6 are codes 0 .. 7: a tie goes to the even one
    const uint32_t code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
    codes |= (code | (h >> 31) << 3) << (4 * e);
  }
  *reinterpret_cast<uint32_t *>(row + c * 4) = codes;
  if ((c & 3) == 0) row[Row::OFF_EXP + (c >> 2)] = (unsigned char)(bad ? 255 : ex + 127);
}

template <int D_QK, int D_V, bool FP4>
__global__ void __launch_bounds__(256) latent_cache_gather_kernel(const unsigned char *cache, const int64_t *slots, uint16_t *out,
                                                                  int64_t T, int64_t num_slots) {
  using Row = CacheRow<D_QK, D_V, FP4>;
  constexpr int CH = D_QK / 8, CV = D_V / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = id / CH;
  const int c = (int)(id - t * CH);
  if (t >= T) return;
  const int64_t slot = slots[t];
  i32x4 v{0, 0, 0, 0};
  if (slot >= 0 && slot < num_slots) {
    const unsigned char *row = cache + slot * Row::BYTES;
    if (!FP4 || c >= CV) {
      v = ld_global_16(row + (c < CV ? 0 : Row::OFF_ROPE - CV * 16) + c * 16);
    } else {
      const uint32_t e = row[Row::OFF_EXP + (c >> 2)];
      v = e2m1x8_to_bf16(*reinterpret_cast<const uint32_t *>(row + c * 4), e8m0_scale(e));
      if (e == 255u) v = i32x4{0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0};
    }
  }
  *reinterpret_cast<i32x4 *>(out + t * D_QK + c * 8) = v;
}

template <int D_QK, int D_V, bool FP4>
static int append_as(const AppendParams &p, hipStream_t st) {
  const int64_t n = (p.T * (D_QK / 8) + 255) / 256;
  DSA_REQUIRE(n < (1ll << 24), "dsa_latent_cache_append: too many rows");  // (a grid's axis: fewer than 2^32 threads)
  hipLaunchKernelGGL((latent_cache_append_kernel<D_QK, D_V, FP4>), dim3((unsigned)n), dim3(256), 0, st, p);
  return check_launch("dsa_latent_cache_append");
}
int launch_cache_append(void *cache, const void *latent, int64_t latent_t, const void *rope, int64_t rope_t, const int64_t *slots,
                        int64_t T, int64_t num_slots, int64_t d_qk, bool fp4, hipStream_t st) {
  const AppendParams p{(unsigned char *)cache, (const unsigned char *)latent, (const unsigned char *)rope, latent_t, rope_t,
                       slots, T, num_slots};
  if (d_qk == 576) return fp4 ? append_as<576, 512, true>(p, st) : append_as<576, 512, false>(p, st);
  return fp4 ? append_as<128, 64, true>(p, st) : append_as<128, 64, false>(p, st);
}

template <int D_QK, int D_V, bool FP4>
static int gather_as(const void *cache, const int64_t *slots, void *out, int64_t T, int64_t num_slots, hipStream_t st) {
  const int64_t n = (T * (D_QK / 8) + 255) / 256;
  DSA_REQUIRE(n < (1ll << 24), "dsa_latent_cache_gather: too many rows");
  hipLaunchKernelGGL((latent_cache_gather_kernel<D_QK, D_V, FP4>), dim3((unsigned)n), dim3(256), 0, st,
                     (const unsigned char *)cache, slots, (uint16_t *)out, T, num_slots);
  return check_launch("dsa_latent_cache_gather");
}
int launch_cache_gather(const void *cache, const int64_t *slots, void *out, int64_t T, int64_t num_slots, int64_t d_qk, bool fp4,
                        hipStream_t st) {
  if (d_qk == 576)
    return fp4 ? gather_as<576, 512, true>(cache, slots, out, T, num_slots, st)
               : gather_as<576, 512, false>(cache, slots, out, T, num_slots, st);
  return fp4 ? gather_as<128, 64, true>(cache, slots, out, T, num_slots, st)
             : gather_as<128, 64, false>(cache, slots, out, T, num_slots, st);
}

// ---------------------------------------------------------------------------
// The plan of a serving step
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256, kPlanOwn = 64;  // requests of a workgroup, at most

struct PlanOwn {
  int64_t start;  // first token
  int ctx, n, held, got, before, back, granted, done;  // before: new blocks of earlier requests; back: blocks given back by them
};

// Blocks that a request holds: its context's, and those behind them up to the first negative entry of its table (tokens of
// an earlier step that were not kept).  The search doubles its stride, then halves it: one load where nothing is behind.
__device__ __forceinline__ int blocks_held(const int32_t *row, int of_context, int W) {
  int lo = of_context, hi = W;  // entries before lo are blocks; entry hi, if there is one, is none
  for (int step = 1; lo < hi; step *= 2) {
    const int at = step <= hi - lo ? lo + step - 1 : hi - 1;
    if (row[at] < 0) {
      hi = at;
      break;
    }
    lo = at + 1;
  }
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (row[mid] < 0) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// Inclusive prefix over the workgroup of two values per thread, and their totals.
__device__ __forceinline__ void scan2(int64_t &a, int64_t &b, int64_t (*tmp)[2], int64_t &ta, int64_t &tb) {
  const int lane = lane_id(), w = (int)(threadIdx.x >> 6);
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t x = __shfl_up(a, off, 64), y = __shfl_up(b, off, 64);
    if (lane >= off) {
      a += x;
      b += y;
    }
  }
  __syncthreads();
  if (lane == 63) {
    tmp[w][0] = a;
    tmp[w][1] = b;
  }
  __syncthreads();
  ta = tb = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i == w) {
      a += ta;
      b += tb;
    }
    ta += tmp[i][0];
    tb += tmp[i][1];
  }
}

__global__ void __launch_bounds__(kPlanThreads) latent_plan_kernel(const PlanParams p) {
  __shared__ int64_t tmp[kPlanThreads / 64][2];
  __shared__ PlanOwn own[kPlanOwn];
  __shared__ int used_lds;
  const int r0 = (int)blockIdx.x * p.per_wg, r1 = min(r0 + p.per_wg, p.R);
  const int64_t cap = (int64_t)p.W * p.block;
  const int have = min(max(p.free_count[0], 0), p.F);
  if (threadIdx.x == 0) used_lds = 0;
  int64_t tokens = 0, needed = 0, back = 0;  // of the requests before this chunk
  int used = 0;
  for (int c = 0; c < p.R; c += kPlanThreads) {
    const int r = c + (int)threadIdx.x;
    PlanOwn x{};
    int need = 0;
    int64_t a = 0, b = 0;
    if (r < p.R) {
      const int64_t ctx = p.context_lens[r];
      x.ctx = (int)(ctx < 0 ? 0 : (ctx < cap ? ctx : cap));
      const int asked = p.query_lens[r];
      x.done = asked < 0;
      x.n = asked > 0 ? asked : 0;
      x.held = blocks_held(p.table + (int64_t)r * p.W, (int)(((int64_t)x.ctx + p.block - 1) / p.block), p.W);
      a = x.n;
    }
    // tokens first: whether a request's fit decides what it needs
    int64_t ta, tb;
    b = x.done ? x.held : 0;
    scan2(a, b, tmp, ta, tb);
    const int64_t tok_end = tokens + a, back_end = back + b;
    const bool fits = r < p.R && !x.done && tok_end <= p.T && (int64_t)x.ctx + x.n <= cap;
    if (fits) need = max((int)(((int64_t)x.ctx + x.n + p.block - 1) / p.block) - x.held, 0);
    int64_t d = need, z = 0, td, tz;
    scan2(d, z, tmp, td, tz);
    const int64_t upto = needed + d;
    x.granted = fits && (need == 0 || upto <= have);
    x.got = x.granted ? need : 0;
    x.start = tok_end - x.n;
    x.before = (int)(upto - need);
    x.back = (int)(back_end - (x.done ? x.held : 0));
    if (x.granted) used = max(used, (int)min(upto, (int64_t)have) * (need > 0));
    if (r >= r0 && r < r1) own[r - r0] = x;
    tokens += ta;
    back += tb;
    needed += td;
  }
  __syncthreads();
  atomicMax(&used_lds, used);  // an integer maximum: its order does not matter
  __syncthreads();
  const int kept = have - used_lds;
  const int64_t left = kept + back < p.F ? kept + back : p.F;

  // lists and tokens that belong to no request, over all workgroups
  const int64_t gid = (int64_t)blockIdx.x * kPlanThreads + threadIdx.x, gsz = (int64_t)gridDim.x * kPlanThreads;
  for (int64_t i = gid; i < p.F; i += gsz)
    if (i < kept || i >= left) p.free_out[i] = i < kept ? p.free_blocks[i] : -1;
  for (int64_t i = (tokens < p.T ? tokens : p.T) + gid; i < p.T; i += gsz) {
    p.slots[i] = -1;
    p.positions[i] = -1;
  }
  if (gid == 0) {
    p.free_count_out[0] = (int)left;
    p.query_starts[p.R] = (int)(tokens < p.T ? tokens : p.T);
  }
  const int w = (int)(threadIdx.x >> 6), lane = lane_id();
  for (int r = r0 + (int)threadIdx.x; r < r1; r += kPlanThreads) {
    const PlanOwn &x = own[r - r0];
    p.query_starts[r] = (int)(x.start < p.T ? x.start : p.T);
    p.kv_lens[r] = x.granted ? x.ctx + x.n : 0;
    p.context_out[r] = x.done ? 0 : x.ctx + (x.granted ? x.n : 0);
    p.granted[r] = x.granted;
  }
  for (int r = r0 + w; r < r1; r += kPlanThreads / 64) {  // a wave per request
    const PlanOwn x = own[r - r0];
    const int32_t *in = p.table + (int64_t)r * p.W;
    int32_t *out = p.table_out + (int64_t)r * p.W;
    // block j of the request after this step
    auto block_at = [&](int j) {
      if (x.done || j >= x.held + x.got) return -1;
      return j < x.held ? in[j] : p.free_blocks[have - 1 - (x.before + j - x.held)];
    };
    for (int j = lane; j < p.W; j += 64) out[j] = block_at(j);
    if (x.done)
      for (int j = lane; j < x.held; j += 64) {
        const int64_t to = (int64_t)kept + x.back + j;
        if (to < p.F) p.free_out[to] = in[j];
      }
    for (int64_t i = lane; i < x.n && x.start + i < p.T; i += 64) {
      int64_t slot = -1;
      int pos = -1;
      if (x.granted) {
        pos = x.ctx + (int)i;
        const int j = pos / p.block, e = block_at(j);
        if (e >= 0) slot = (int64_t)e * p.block + (pos - j * p.block);
      }
      p.slots[x.start + i] = slot;
      p.positions[x.start + i] = pos;
    }
  }
}

int launch_latent_plan(PlanParams p, hipStream_t st) {
  // as many workgroups as fill the card, of at most kPlanOwn requests each
  int64_t wgs = p.R < 256 ? p.R : 256;
  if (wgs * kPlanOwn < p.R) wgs = (p.R + kPlanOwn - 1) / kPlanOwn;
  if (wgs < 1) wgs = 1;
  p.per_wg = (int)((p.R + wgs - 1) / wgs);
  hipLaunchKernelGGL(latent_plan_kernel, dim3((unsigned)wgs), dim3(kPlanThreads), 0, st, p);
  return check_launch("dsa_latent_plan_step");
}

}  // namespace dsa
