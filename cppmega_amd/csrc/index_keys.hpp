// The paged cache of index keys: page format, conversions, parameters of the scores over it.
#pragma once

#include "dsa_common.hpp"
#include "latent_cache.hpp"
#include "requests.hpp"

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

struct IndexScoreParams {
  const unsigned char *q;      // [T, H, D] bf16
  const void *w;               // [T, H] bf16 or f32
  const unsigned char *cache;  // [num_blocks] pages
  const int32_t *table;        // [R, W]
  Requests req;
  float *out;                  // [tokens, L] scores of tokens first ..
  int32_t *windows;            // [2, tokens] 0 and the columns that a token sees (0: of no request); null: every column is written
  int64_t page_bytes;
  int first, tokens;           // tokens of the batch that are scored
  int W, L, block, block_shift, num_blocks;
  int span;                    // keys whose pages lie in the window, whole blocks
  int w_f32, relu;
  int fill;                    // columns that no token of a request sees are written
  int whole_tiles;             // 64 keys from a multiple of 64 on lie on one page
};
int launch_index_scores(IndexScoreParams p, int64_t H, int64_t D, int fmt, hipStream_t st);

}  // namespace dsa
