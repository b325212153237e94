// The paged latent cache: row formats, and the conversions of its 4-bit form.
#pragma once

#include "dsa_common.hpp"

namespace dsa {

// A cache is pages of `block` rows.  Row formats:
//   bf16   d_qk channels (the latent's d_v, then the rope part)
//   mxfp4  d_v / 2 bytes of e2m1 codes (channel 2 i in the low half of byte i), the rope
//          part as bf16, d_v / 32 exponent bytes e (scale 2^(e - 127), 255: NaN), padded
//          to 16 bytes
template <int D_QK, int D_V, bool FP4>
struct CacheRow {
  static constexpr int ROPE = D_QK - D_V;
  static constexpr int OFF_ROPE = FP4 ? D_V / 2 : 2 * D_V, OFF_EXP = OFF_ROPE + 2 * ROPE;
  static constexpr int BYTES = FP4 ? (OFF_EXP + D_V / 32 + 15) / 16 * 16 : 2 * D_QK;
  static_assert(D_V % 32 == 0 && ROPE % 8 == 0, "whole blocks and 16-byte chunks");
};
inline int64_t cache_row_bytes(int64_t d_qk, int64_t d_v, bool fp4) {
  return fp4 ? (d_v / 2 + 2 * (d_qk - d_v) + d_v / 32 + 15) / 16 * 16 : 2 * d_qk;
}

// 2^(e - 127) of an exponent byte (255: NaN).
__device__ __forceinline__ float e8m0_scale(uint32_t e) {
  return __uint_as_float(e == 255u ? 0x7fc00000u : (e == 0u ? 0x00400000u : e << 23));
}

// Eight e2m1 codes (one dword, lowest half byte first) times 2^(e - 127) as bf16: exact, the
// products have two significant bits and, for the exponents that the append writes, are normal.
__device__ __forceinline__ i32x4 e2m1x8_to_bf16(uint32_t codes, float scale) {
  i32x4 r;
  r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return r;
}

struct PlanParams {
  const int32_t *context_lens, *query_lens, *table, *free_blocks, *free_count;
  int64_t *slots;
  int32_t *positions, *query_starts, *kv_lens, *context_out, *granted, *table_out, *free_out, *free_count_out;
  int64_t T;
  int R, W, F, block, per_wg;
};

int launch_cache_append(void *cache, const void *latent, int64_t latent_t, const void *rope, int64_t rope_t, const int64_t *slots,
                        int64_t T, int64_t num_slots, int64_t d_qk, bool fp4, hipStream_t st);
int launch_cache_gather(const void *cache, const int64_t *slots, void *out, int64_t T, int64_t num_slots, int64_t d_qk, bool fp4,
                        hipStream_t st);
int launch_latent_plan(PlanParams p, hipStream_t st);

}  // namespace dsa
