// The paged cache of index keys (page format, conversions) and the requests of a paged call.
#pragma once

#include "dsa_common.hpp"
#include "latent_cache.hpp"

namespace dsa {

enum KeyFormat { KEY_BF16 = 0, KEY_MXFP8 = 1, KEY_MXFP4 = 2 };

// A page holds `block` keys of D channels.
//   bf16   their rows
//   mxfp8  their rows of D e4m3 codes, then four exponent bytes a key: byte b is that of channels 32 b .. 32 b + 31
//          (scale 2^(e - 127), 255: NaN), those past the last channel 0
//   mxfp4  the same of D / 2 bytes of e2m1 codes (channel 2 i in the low half of byte i)
// Exponents lie apart from the codes so that a page's codes are one run of whole 16-byte chunks.
template <int D, int FMT>
struct KeyRow {
  static constexpr int CODES = FMT == KEY_BF16 ? 2 * D : FMT == KEY_MXFP8 ? D : D / 2;  // bytes
  static constexpr int BYTES = CODES + (FMT == KEY_BF16 ? 0 : 4);                       // of a page, per key
  static constexpr int CPE = 16 * D / CODES;                                            // channels of a 16-byte chunk
};
inline int64_t key_row_bytes(int64_t d, int fmt) { return fmt == KEY_BF16 ? 2 * d : (fmt == KEY_MXFP8 ? d : d / 2) + 4; }

constexpr int kFp8LeastExp = -117, kFp8MostExp = 119;  // of an MXFP8 scale: every code then stands for a finite, normal bf16

// Eight e4m3 codes times 2^(e - 127) as bf16: exact, a code has four significant bits.
__device__ __forceinline__ i32x4 e4m3x8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  i32x4 r;
  r[0] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  r[1] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  r[2] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  r[3] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return r;
}
// Channels 8 u .. 8 u + 7 of a chunk of codes whose exponent byte is e.
template <int FMT>
__device__ __forceinline__ i32x4 key_values(i32x4 chunk, int u, uint32_t e) {
  if constexpr (FMT == KEY_BF16) {
    return chunk;
  } else {
    const float scale = e8m0_scale(e);
    const i32x4 v = FMT == KEY_MXFP8 ? e4m3x8_to_bf16((uint32_t)chunk[2 * u], (uint32_t)chunk[2 * u + 1], scale)
                                     : e2m1x8_to_bf16((uint32_t)chunk[u], scale);
    constexpr int nan2 = 0x7fc07fc0;
    return e == 255u ? i32x4{nan2, nan2, nan2, nan2} : v;
  }
}

// The requests of a call: tokens query_starts[r] .. query_starts[r + 1] of the batch (null: token r alone) are the last of
// request r's kv_lens[r] positions.
struct Requests {
  const int32_t *query_starts, *kv_lens;
  int64_t cap;  // W * block: lengths past it are cut
  int T, R;
  __device__ __forceinline__ int start(int r) const { return query_starts == nullptr ? r : min(max(query_starts[r], 0), T); }
  __device__ __forceinline__ int tokens(int r) const {
    if (query_starts == nullptr) return r < T ? 1 : 0;
    const int n = start(r + 1) - start(r);
    return n > 0 ? n : 0;
  }
  __device__ __forceinline__ int kv(int r) const {
    const int k = kv_lens[r];
    return k < 0 ? 0 : (k < cap ? k : (int)cap);
  }
  // The last request that begins at or before token t (the whole wave: 64 of them are looked at in a step).
  __device__ __forceinline__ int of(int t) const {
    if (query_starts == nullptr) return t < R ? t : R - 1;
    const int lane = lane_id();
    int lo = 0, n = R;
    while (n > 1) {
      const int step = (n + 63) / 64, at = lo + lane * step;
      const uint64_t before = __builtin_amdgcn_ballot_w64(lane * step < n && start(at < R ? at : 0) <= t);
      const int k = before == 0 ? 0 : 63 - (int)__builtin_clzll(before);
      n = n - k * step < step ? n - k * step : step;
      lo += k * step;
    }
    return lo;
  }
  // The same, lane by lane.
  __device__ __forceinline__ int of_lane(int t) const {
    if (query_starts == nullptr) return t < R ? t : R - 1;
    int lo = 0, hi = R - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (start(mid) <= t) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
  // Positions that token t of request r sees, -1 where it is not one of the request's.
  __device__ __forceinline__ int keys_of(int t, int r) const {
    const int at = start(r), n = tokens(r);
    return t >= at && t < at + n ? max(kv(r) - n + (t - at) + 1, 0) : -1;
  }
};

struct IndexScoreParams {
  const unsigned char *q;      // [T, H, D] bf16
  const void *w;               // [T, H] bf16 or f32
  const unsigned char *cache;  // [num_blocks] pages
  const int32_t *table;        // [R, W]
  Requests req;
  float *out;                  // [tokens, L] scores of tokens first ..
  int32_t *limits;             // [tokens] keys that a token sees (0: a token of no request), or null
  int64_t page_bytes;
  int first, tokens;           // tokens of the batch that are scored
  int W, L, block, block_shift, num_blocks;
  int chunk, tiles;            // keys of a workgroup; token tiles
  int w_f32, relu;
};
int launch_index_scores(IndexScoreParams p, int64_t H, int64_t D, int fmt, hipStream_t st);

}  // namespace dsa
