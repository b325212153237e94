// Index keys into and out of their paged cache, on gfx950: one thread per 8 channels (16
// bytes of bf16), bound by the bytes moved.  The four neighbouring lanes of a 32-channel
// block share its largest magnitude.  MXFP8: the scale is the least power of two under
// which that is at most 448, e4m3's largest value, so nothing saturates (but magnitudes
// past 1.75 2^127, as the exponent is held to 119); MXFP4: as the latent cache's.
// 65536 keys of 128 channels in MXFP4: append 7.0 us (3.1 TB/s, slots and rows one
// latency behind the other), gather 6.3; 64 keys 2.3 and 2.2, the launch.
#include "index_keys.hpp"

namespace dsa {

struct KeyCacheParams {
  unsigned char *cache;
  const unsigned char *k;
  uint16_t *out;
  const int64_t *slots;
  int64_t T, k_stride, num_slots, page_bytes;  // k_stride in bytes
  int block, block_shift;
};

__device__ __forceinline__ unsigned char *page_at(const KeyCacheParams &p, int64_t slot, int &off) {
  const int64_t page = p.block_shift >= 0 ? slot >> p.block_shift : slot / p.block;
  off = (int)(slot - page * p.block);
  return p.cache + page * p.page_bytes;
}

template <int D, int FMT>
__global__ void __launch_bounds__(256) index_key_append_kernel(const KeyCacheParams p) {
  using Row = KeyRow<D, FMT>;
  constexpr int CH = D / 8;  // threads of a key: whole quads
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, t = id / CH;
  const int c = (int)(id - t * CH);
  if (t >= p.T) return;
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.num_slots) return;
  const i32x4 v = ld_global_16(p.k + t * p.k_stride + c * 16);
  int off;
  unsigned char *page = page_at(p, slot, off), *row = page + (int64_t)off * Row::CODES;
  if constexpr (FMT == KEY_BF16) {
    *reinterpret_cast<i32x4 *>(row + c * 16) = v;
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
  int ex;
  if constexpr (FMT == KEY_MXFP8) {
    ex = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u);  // amax <= 1.75 * 2^8 * 2^ex
    ex = min(max(ex, kFp8LeastExp), kFp8MostExp);
  } else {
    ex = max((int)(top >> 23) - 127 - 2, -125);
  }
  if (top == 0 || bad) ex = 0;
  const float inv = bad ? 0.0f : __uint_as_float((uint32_t)(127 - ex) << 23);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = (uint32_t)v[e >> 1], h = (e & 1) ? u & 0xffff0000u : u << 16;
    x[e] = bad ? __uint_as_float(h & 0x80000000u) : __uint_as_float(h) * inv;
  }
  if constexpr (FMT == KEY_MXFP8) {
    i32x2 codes;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      int w = 0;
      auto held = [&](int i) { return __builtin_amdgcn_fmed3f(x[4 * e + i], -448.0f, 448.0f); };
      w = __builtin_amdgcn_cvt_pk_fp8_f32(held(0), held(1), w, false);
      codes[e] = __builtin_amdgcn_cvt_pk_fp8_f32(held(2), held(3), w, true);
    }
    *reinterpret_cast<i32x2 *>(row + c * 8) = codes;
  } else {
    uint32_t codes = 0;  // (the conversion rounds to nearest even and saturates)
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], 1.0f, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], 1.0f, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], 1.0f, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], 1.0f, 3);
    *reinterpret_cast<uint32_t *>(row + c * 4) = codes;
  }
  unsigned char *expo = page + (int64_t)p.block * Row::CODES + (int64_t)off * 4;
  if ((c & 3) == 0) {
    expo[c >> 2] = (unsigned char)(bad ? 255 : ex + 127);
    if (D < 128) expo[2 + (c >> 2)] = 0;
  }
}

template <int D, int FMT>
__global__ void __launch_bounds__(256) index_key_gather_kernel(const KeyCacheParams p) {
  using Row = KeyRow<D, FMT>;
  constexpr int CH = D / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, t = id / CH;
  const int c = (int)(id - t * CH);
  if (t >= p.T) return;
  const int64_t slot = p.slots[t];
  i32x4 v{0, 0, 0, 0};
  if (slot >= 0 && slot < p.num_slots) {
    int off;
    const unsigned char *page = page_at(p, slot, off), *row = page + (int64_t)off * Row::CODES;
    const uint32_t e = FMT == KEY_BF16 ? 0u : page[(int64_t)p.block * Row::CODES + (int64_t)off * 4 + (c >> 2)];
    if constexpr (FMT == KEY_BF16) {
      v = ld_global_16(row + c * 16);
    } else if constexpr (FMT == KEY_MXFP8) {
      const i32x2 x = ld_global_8(row + c * 8);
      v = key_values<FMT>(i32x4{x[0], x[1], 0, 0}, 0, e);
    } else {
      v = key_values<FMT>(i32x4{*reinterpret_cast<const int *>(row + c * 4), 0, 0, 0}, 0, e);
    }
  }
  *reinterpret_cast<i32x4 *>(p.out + t * D + c * 8) = v;
}

template <int D, int FMT>
static int launch_as(const char *who, bool append, const KeyCacheParams &p, hipStream_t st) {
  const int64_t n = (p.T * (D / 8) + 255) / 256;
  if (append) hipLaunchKernelGGL((index_key_append_kernel<D, FMT>), dim3((unsigned)n), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((index_key_gather_kernel<D, FMT>), dim3((unsigned)n), dim3(256), 0, st, p);
  return check_launch(who);
}
template <int D>
static int launch_of(const char *who, bool append, int fmt, const KeyCacheParams &p, hipStream_t st) {
  if (fmt == KEY_BF16) return launch_as<D, KEY_BF16>(who, append, p, st);
  return fmt == KEY_MXFP8 ? launch_as<D, KEY_MXFP8>(who, append, p, st) : launch_as<D, KEY_MXFP4>(who, append, p, st);
}

// A grid's threads along an axis stay below 2^32, its last workgroup's among them.
static bool countable(int64_t T, int64_t d) { return T >= 0 && T < (1ll << 28) && (T * (d / 8) + 255) / 256 < (1ll << 24); }

static int check_keys(const char *who, int64_t num_blocks, int64_t block, int64_t d, int dtype) {
  DSA_REQUIRE(num_blocks > 0 && num_blocks < (1ll << 31) && block > 0 && block <= 65536,
              "%s: num_blocks=%lld must be in [1, 2^31), block_size=%lld in [1, 65536]", who, (long long)num_blocks, (long long)block);
  DSA_REQUIRE(dtype == DSA_DTYPE_BF16 || dtype == DSA_DTYPE_MXFP8 || dtype == DSA_DTYPE_MXFP4,
              "%s: index keys are bf16, MXFP8 or MXFP4, got dtype %d", who, dtype);
  DSA_REQUIRE(dtype == DSA_DTYPE_BF16 || block % 4 == 0, "%s: pages of MX keys hold a multiple of 4, got block_size=%lld", who,
              (long long)block);
  if (d != 64 && d != 128)
    return set_error(DSA_ERR_UNSUPPORTED, "%s: no kernel for index keys of %lld channels (64, 128)", who, (long long)d);
  return DSA_OK;
}
static int key_format(int dtype) { return dtype == DSA_DTYPE_BF16 ? KEY_BF16 : dtype == DSA_DTYPE_MXFP8 ? KEY_MXFP8 : KEY_MXFP4; }

static int run_keys(const char *who, bool append, KeyCacheParams p, int64_t num_blocks, int64_t block, int64_t d, int dtype, hipStream_t st) {
  const int fmt = key_format(dtype);
  p.num_slots = num_blocks * block;
  p.page_bytes = block * key_row_bytes(d, fmt);
  p.block = (int)block;
  p.block_shift = shift_of(block);
  return d == 128 ? launch_of<128>(who, append, fmt, p, st) : launch_of<64>(who, append, fmt, p, st);
}

}  // namespace dsa

using namespace dsa;

extern "C" int64_t dsa_index_key_row_bytes(int64_t D, int dtype) {
  if (check_keys("dsa_index_key_row_bytes", 1, 4, D, dtype)) return 0;
  return key_row_bytes(D, key_format(dtype));
}

extern "C" int dsa_index_key_append(void *cache, const void *k, int64_t k_stride, const int64_t *slots, int64_t T, int64_t num_blocks,
                                    int64_t block_size, int64_t D, int dtype, void *stream) {
  const char *who = "dsa_index_key_append";
  const int rc = check_keys(who, num_blocks, block_size, D, dtype);
  if (rc) return rc;
  DSA_REQUIRE(countable(T, D), "%s: T=%lld must be in [0, 2^28), for 128 channels at most 2^28 - 16", who, (long long)T);
  if (T == 0) return DSA_OK;
  DSA_REQUIRE(cache && k && slots && aligned16(cache) && aligned16(k), "%s: null or misaligned pointer", who);
  DSA_REQUIRE(k_stride >= 0 && k_stride % 8 == 0, "%s: the row stride must be a non-negative multiple of 8 elements", who);
  KeyCacheParams p{};
  p.cache = (unsigned char *)cache;
  p.k = (const unsigned char *)k;
  p.slots = slots;
  p.T = T;
  p.k_stride = k_stride * 2;
  return run_keys(who, true, p, num_blocks, block_size, D, dtype, (hipStream_t)stream);
}

extern "C" int dsa_index_key_gather(const void *cache, const int64_t *slots, void *out, int64_t T, int64_t num_blocks, int64_t block_size,
                                    int64_t D, int dtype, void *stream) {
  const char *who = "dsa_index_key_gather";
  const int rc = check_keys(who, num_blocks, block_size, D, dtype);
  if (rc) return rc;
  DSA_REQUIRE(countable(T, D), "%s: T=%lld must be in [0, 2^28), for 128 channels at most 2^28 - 16", who, (long long)T);
  if (T == 0) return DSA_OK;
  DSA_REQUIRE(cache && slots && out && aligned16(cache) && aligned16(out), "%s: null or misaligned pointer", who);
  KeyCacheParams p{};
  p.cache = (unsigned char *)const_cast<void *>(cache);
  p.out = (uint16_t *)out;
  p.slots = slots;
  p.T = T;
  return run_keys(who, false, p, num_blocks, block_size, D, dtype, (hipStream_t)stream);
}

extern "C" int dsa_paged_index_scores(const void *q, const void *w, const void *cache, const int32_t *block_table,
                                      const int32_t *query_starts, const int32_t *kv_lens, float *scores, int32_t *windows, int64_t T,
                                      int64_t R, int64_t W, int64_t first, int64_t tokens, int64_t L, int64_t H, int64_t D,
                                      int64_t num_blocks, int64_t block_size, int dtype, int w_dtype, int use_relu, void *stream) {
  const char *who = "dsa_paged_index_scores";
  const int rc = check_keys(who, num_blocks, block_size, D, dtype);
  if (rc) return rc;
  DSA_REQUIRE(w_dtype == DSA_DTYPE_BF16 || w_dtype == DSA_DTYPE_F32, "%s: weights are bf16 or f32, got dtype %d", who, w_dtype);
  DSA_REQUIRE(T >= 0 && R >= 0 && W > 0 && H > 0 && L >= 0 && first >= 0 && tokens >= 0 && first + tokens <= T,
              "%s: bad sizes T=%lld R=%lld W=%lld H=%lld columns=%lld tokens %lld + %lld", who, (long long)T, (long long)R, (long long)W,
              (long long)H, (long long)L, (long long)first, (long long)tokens);
  DSA_REQUIRE(T < (1ll << 30) && R < (1 << 20) && W < (1ll << 31) && W * block_size < (1ll << 31) - 65536 && L <= W * block_size,
              "%s: sizes out of range (R < 2^20, T < 2^30, W * block_size below 2^31 - 65536, at most W * block_size columns)", who);
  if (H != 16 && H != 32 && H != 64)
    return set_error(DSA_ERR_UNSUPPORTED, "%s: no kernel for %lld index heads (16, 32, 64)", who, (long long)H);
  DSA_REQUIRE(query_starts != nullptr || T == R, "%s: without query_starts every request has one token: %lld tokens, %lld requests", who,
              (long long)T, (long long)R);
  if (tokens == 0 || (L == 0 && windows == nullptr)) return DSA_OK;
  DSA_REQUIRE(q && w && cache && (L == 0 || scores) && (R == 0 || (block_table && kv_lens)) && aligned16(q) && aligned16(cache),
              "%s: null or misaligned pointer", who);
  IndexScoreParams p{};
  p.q = (const unsigned char *)q;
  p.w = w;
  p.cache = (const unsigned char *)cache;
  p.table = block_table;
  p.req = Requests{query_starts, kv_lens, W * block_size, (int)T, (int)R};
  p.out = scores;
  p.windows = windows;
  p.first = (int)first;
  p.tokens = (int)tokens;
  p.W = (int)W;
  p.L = (int)L;
  p.block = (int)block_size;
  p.block_shift = shift_of(block_size);
  p.num_blocks = (int)num_blocks;
  p.page_bytes = block_size * key_row_bytes(D, key_format(dtype));
  p.w_f32 = w_dtype == DSA_DTYPE_F32;
  p.relu = use_relu != 0;
  return launch_index_scores(p, H, D, key_format(dtype), (hipStream_t)stream);
}
