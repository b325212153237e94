// C entry points of dense latent attention: argument checks and parameter blocks.
#include <math.h>

#include "latent_mla.hpp"

namespace dsa {

// Tensors may be empty (no tokens): their pointers are then not looked at.
static bool given(const void *p, int64_t n) { return n == 0 || (p != nullptr && aligned16(p)); }

// Sizes, scale and windows that both forms and both directions share.
static int check_common(const char *who, int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t G, float sm_scale, int causal,
                        const int32_t *starts, const int32_t *ends) {
  DSA_REQUIRE(B >= 0 && S >= 0 && S_kv >= 0 && H > 0 && G > 0 && H % G == 0,
              "%s: bad sizes B=%lld S=%lld S_kv=%lld H=%lld G=%lld", who, (long long)B, (long long)S, (long long)S_kv,
              (long long)H, (long long)G);
  DSA_REQUIRE(H <= 4096 && S < (1ll << 30) && S_kv < (1ll << 30) && S * (H / G) < (1ll << 31) - 256 && B * G < (1ll << 24),
              "%s: sizes out of range (H <= 4096, S * H / G < 2^31 - 256, S_kv < 2^30, B * G < 2^24)", who);
  DSA_REQUIRE(isfinite(sm_scale) && sm_scale >= kLeastScale, "%s: sm_scale must be finite and at least 2^-100, got %g", who,
              (double)sm_scale);
  DSA_REQUIRE(causal == 0 || causal == 1, "%s: causal must be 0 or 1", who);
  DSA_REQUIRE((starts == nullptr) == (ends == nullptr), "%s: starts and ends come together", who);
  DSA_REQUIRE(starts == nullptr || !causal, "%s: row windows carry the mask: pass causal = 0 with them", who);
  return DSA_OK;
}

static LatentParams common_params(const void *q, const int32_t *starts, const int32_t *ends, int64_t B, int64_t S, int64_t S_kv,
                                  int64_t H, int64_t G, float sm_scale, int causal) {
  LatentParams p{};
  p.q = (const unsigned char *)q;
  p.starts = starts;
  p.ends = ends;
  p.B = B;
  p.S = S;
  p.S_kv = S_kv;
  p.H = H;
  p.G = G;
  p.hpg = (int)(H / G);
  p.rows = S * p.hpg;
  p.causal = causal;
  p.scale = sm_scale;
  p.sl2 = sm_scale * kLog2e;
  return p;
}

static void absorbed_kv(LatentParams &p, const void *kv, int64_t D) {
  p.k = (const unsigned char *)kv;
  p.k_g = D * 2;
  p.k_t = p.G * D * 2;
  p.k_b = p.S_kv * p.k_t;
}

static int expanded_kv(const char *who, LatentParams &p, const void *k_nope, const void *k_pe, const void *v,
                       const int64_t *st) {
  DSA_REQUIRE(st != nullptr, "%s: null strides", who);
  const int64_t n = p.B * p.S_kv;
  DSA_REQUIRE(given(k_nope, n) && given(k_pe, n) && given(v, n), "%s: k_nope, k_pe and v must be 16-byte aligned device pointers", who);
  for (int i = 0; i < 8; ++i)
    DSA_REQUIRE(st[i] >= 0 && st[i] % 8 == 0, "%s: strides must be non-negative multiples of 8 elements", who);
  DSA_REQUIRE(st[1] < (1ll << 23) && st[4] < (1ll << 23) && st[6] < (1ll << 23), "%s: token strides must be below 2^23 elements", who);
  p.k = (const unsigned char *)k_nope;
  p.kpe = (const unsigned char *)k_pe;
  p.v = (const unsigned char *)v;
  p.k_b = st[0] * 2;
  p.k_t = st[1] * 2;
  p.k_g = st[2] * 2;
  p.pe_b = st[3] * 2;
  p.pe_t = st[4] * 2;
  p.v_b = st[5] * 2;
  p.v_t = st[6] * 2;
  p.v_g = st[7] * 2;
  return DSA_OK;
}

static bool shape_served(int64_t d_qk, int64_t d_v, bool expanded) {
  if (expanded) return (d_qk == 192 && d_v == 128) || (d_qk == 128 && d_v == 64);
  return (d_qk == 128 && (d_v == 64 || d_v == 128)) || (d_qk == 192 && d_v == 128);
}
static int check_shape(const char *who, int64_t d_qk, int64_t d_v, bool expanded) {
  if (shape_served(d_qk, d_v, expanded)) return DSA_OK;
  return set_error(DSA_ERR_UNSUPPORTED, "%s: no kernel for d_qk=%lld d_v=%lld (%s)", who, (long long)d_qk, (long long)d_v,
                   expanded ? "64 of them k_pe; 192 / 128 or 128 / 64" : "128 / 64, 128 / 128 or 192 / 128; wider rows: the expanded form");
}

}  // namespace dsa

using namespace dsa;

extern "C" int dsa_latent_mla_fwd(const void *q, const void *kv, const int32_t *starts, const int32_t *ends, void *out,
                                  void *out_lo, float *lse2, int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t G, int64_t D_qk, int64_t D_v,
                                  float sm_scale, int causal, void *stream) {
  int rc = check_common("dsa_latent_mla_fwd", B, S, S_kv, H, G, sm_scale, causal, starts, ends);
  if (!rc) rc = check_shape("dsa_latent_mla_fwd", D_qk, D_v, false);
  if (rc) return rc;
  DSA_REQUIRE(G * D_qk < (1ll << 23), "dsa_latent_mla_fwd: G * D_qk must be below 2^23");
  if (B * S == 0) return DSA_OK;
  DSA_REQUIRE(given(q, 1) && given(kv, S_kv) && given(out, 1) && aligned16(out_lo) && lse2 != nullptr,
              "dsa_latent_mla_fwd: null or misaligned pointer");
  LatentParams p = common_params(q, starts, ends, B, S, S_kv, H, G, sm_scale, causal);
  absorbed_kv(p, kv, D_qk);
  p.out = (uint16_t *)out;
  p.out_lo = (uint16_t *)out_lo;
  p.lse = lse2;
  return launch_latent_fwd(p, D_qk, D_v, false, (hipStream_t)stream);
}

extern "C" int dsa_latent_mla_expanded_fwd(const void *q, const void *k_nope, const void *k_pe, const void *v, const int32_t *starts,
                                           const int32_t *ends, void *out, void *out_lo, float *lse2, int64_t B, int64_t S,
                                           int64_t S_kv, int64_t H, int64_t D_nope, int64_t D_pe, int64_t D_v, const int64_t *strides,
                                           float sm_scale, int causal, void *stream) {
  int rc = check_common("dsa_latent_mla_expanded_fwd", B, S, S_kv, H, H, sm_scale, causal, starts, ends);
  if (!rc) rc = check_shape("dsa_latent_mla_expanded_fwd", D_pe == 64 ? D_nope + D_pe : -1, D_v, true);
  if (rc) return rc;
  if (B * S == 0) return DSA_OK;
  DSA_REQUIRE(given(q, 1) && given(out, 1) && aligned16(out_lo) && lse2 != nullptr,
              "dsa_latent_mla_expanded_fwd: null or misaligned pointer");
  LatentParams p = common_params(q, starts, ends, B, S, S_kv, H, H, sm_scale, causal);
  rc = expanded_kv("dsa_latent_mla_expanded_fwd", p, k_nope, k_pe, v, strides);
  if (rc) return rc;
  p.out = (uint16_t *)out;
  p.out_lo = (uint16_t *)out_lo;
  p.lse = lse2;
  return launch_latent_fwd(p, D_nope + D_pe, D_v, true, (hipStream_t)stream);
}

extern "C" size_t dsa_latent_mla_bwd_workspace_size(int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t G, int64_t D_qk,
                                                    int64_t D_v, int expanded) {
  if (check_common("dsa_latent_mla_bwd_workspace_size", B, S, S_kv, H, G, 1.0f, 0, nullptr, nullptr)) return 0;
  if (check_shape("dsa_latent_mla_bwd_workspace_size", D_qk, D_v, expanded != 0)) return 0;
  return latent_bwd_workspace(common_params(nullptr, nullptr, nullptr, B, S, S_kv, H, G, 1.0f, 0), D_qk, D_v, expanded != 0);
}

static int backward(const char *who, LatentParams &p, const void *o, const void *o_lo, const void *dO, const float *lse2, void *dq, int64_t d_qk,
                    int64_t d_v, bool expanded, void *ws, size_t ws_bytes, void *stream) {
  const int64_t n = p.B * p.S;
  DSA_REQUIRE(given(p.q, n) && given(o, n) && aligned16(o_lo) && given(dO, n) && given(dq, n) && (n == 0 || lse2 != nullptr),
              "%s: null or misaligned pointer", who);
  const size_t need = latent_bwd_workspace(p, d_qk, d_v, expanded);
  if (need > 0 && (ws == nullptr || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u)))
    return set_error(DSA_ERR_WORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, got %zu", who, need, ws_bytes);
  p.o = (const unsigned char *)o;
  p.o_lo = (const unsigned char *)o_lo;
  p.dO = (const unsigned char *)dO;
  p.lse_in = lse2;
  p.dq = (uint16_t *)dq;
  return launch_latent_bwd(p, d_qk, d_v, expanded, (unsigned char *)ws, (hipStream_t)stream);
}

extern "C" int dsa_latent_mla_bwd(const void *q, const void *kv, const void *o, const void *o_lo, const void *dO, const float *lse2,
                                  const int32_t *starts, const int32_t *ends, void *dq, void *dkv, void *workspace,
                                  size_t workspace_bytes, int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t G, int64_t D_qk,
                                  int64_t D_v, float sm_scale, int causal, void *stream) {
  int rc = check_common("dsa_latent_mla_bwd", B, S, S_kv, H, G, sm_scale, causal, starts, ends);
  if (!rc) rc = check_shape("dsa_latent_mla_bwd", D_qk, D_v, false);
  if (rc) return rc;
  DSA_REQUIRE(G * D_qk < (1ll << 23), "dsa_latent_mla_bwd: G * D_qk must be below 2^23");
  if (B == 0) return DSA_OK;
  DSA_REQUIRE(given(kv, S_kv) && given(dkv, S_kv), "dsa_latent_mla_bwd: null or misaligned kv / dkv");
  LatentParams p = common_params(q, starts, ends, B, S, S_kv, H, G, sm_scale, causal);
  absorbed_kv(p, kv, D_qk);
  p.dk = (uint16_t *)dkv;
  return backward("dsa_latent_mla_bwd", p, o, o_lo, dO, lse2, dq, D_qk, D_v, false, workspace, workspace_bytes, stream);
}

extern "C" int dsa_latent_mla_expanded_bwd(const void *q, const void *k_nope, const void *k_pe, const void *v, const void *o,
                                           const void *o_lo, const void *dO, const float *lse2, const int32_t *starts, const int32_t *ends, void *dq,
                                           void *dk_nope, void *dk_pe, void *dv, void *workspace, size_t workspace_bytes,
                                           int64_t B, int64_t S, int64_t S_kv, int64_t H, int64_t D_nope, int64_t D_pe,
                                           int64_t D_v, const int64_t *strides, float sm_scale, int causal, void *stream) {
  const char *who = "dsa_latent_mla_expanded_bwd";
  int rc = check_common(who, B, S, S_kv, H, H, sm_scale, causal, starts, ends);
  if (!rc) rc = check_shape(who, D_pe == 64 ? D_nope + D_pe : -1, D_v, true);
  if (rc) return rc;
  if (B == 0) return DSA_OK;
  DSA_REQUIRE(given(dk_nope, S_kv) && given(dk_pe, S_kv) && given(dv, S_kv), "%s: null or misaligned gradient", who);
  LatentParams p = common_params(q, starts, ends, B, S, S_kv, H, H, sm_scale, causal);
  rc = expanded_kv(who, p, k_nope, k_pe, v, strides);
  if (rc) return rc;
  p.dk = (uint16_t *)dk_nope;
  p.dkpe = (uint16_t *)dk_pe;
  p.dv = (uint16_t *)dv;
  return backward(who, p, o, o_lo, dO, lse2, dq, D_nope + D_pe, D_v, true, workspace, workspace_bytes, stream);
}
