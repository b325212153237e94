// The indexer's scores of new tokens over a paged cache of index keys, on gfx950:
//   score[t, s] = sum_h w[t, h] relu(q[t, h] . k[s])   for the positions s that token t sees, -inf for the others.
//
// As in the dense indexer the rows of a 32x32x16 MFMA are (token, head) pairs and its columns 32 keys, and ReLU, weight
// and the sum over heads run on the accumulators.  MX keys are widened to bf16, exactly, in front of the product: the
// matrix instructions that take 8-bit codes keep fewer bits of their sums than 32 (a score was off by 1.5e-5 of the scores'
// size; this way 1e-7), and every key that is read serves 16 products at least.
//
// Two kernels.  Single tokens (index_rows_kernel): a workgroup has one token and a chunk of its keys, whose 32-key tiles
// its waves take in turn, straight from memory to operand registers (a lane's 16-byte piece of a key is two steps' operands
// in MXFP8 and four in MXFP4: the order of the channels in a product is free), two tiles ahead, without a barrier.
// Several tokens of a request (index_tiles_kernel): four waves with the (token, head) rows of 4 * 64 / H tokens share
// tiles of 64 keys in LDS, widened as they enter it.
#include "index_keys.hpp"
#include "wave_ops.hpp"

namespace dsa {

constexpr int kMostChunk = 2048;  // keys of a workgroup, at most: its pages lie in LDS

static __device__ const i32x4 kNoKey[16] = {};  // the row of a key that is not there

__device__ __forceinline__ i32x4 ld_16(const unsigned char *x) {
  return *reinterpret_cast<const __attribute__((address_space(1))) i32x4 *>(reinterpret_cast<uint64_t>(x));
}
__device__ __forceinline__ uint32_t ld_4(const unsigned char *x) {
  return *reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(reinterpret_cast<uint64_t>(x));
}
__device__ __forceinline__ int page_of(const IndexScoreParams &p, int key) {
  return p.block_shift >= 0 ? key >> p.block_shift : (int)((uint32_t)key / (uint32_t)p.block);
}
__device__ __forceinline__ float weight_at(const IndexScoreParams &p, int64_t i) {
  return p.w_f32 ? static_cast<const float *>(p.w)[i] : bf16_bits_to_f32(static_cast<const uint16_t *>(p.w)[i]);
}
// Row of accumulator register a in lane half g32.
__device__ __forceinline__ constexpr int score_row(int a, int g32) { return 8 * (a >> 2) + 4 * g32 + (a & 3); }

// Pages of keys [k0, kend) of request r into the window; whether all of them are there.
template <int NTHR>
__device__ __forceinline__ bool fill_window(const IndexScoreParams &p, int *window, int r, int k0, int kend) {
  const int pg0 = page_of(p, k0), n = page_of(p, kend - 1) - pg0 + 1;
  bool ok = true;
  for (int i = (int)threadIdx.x; i < n; i += NTHR) {
    int e = p.table[(int64_t)r * p.W + pg0 + i];
    if (e < 0 || e >= p.num_blocks) {
      e = -1;
      ok = false;
    }
    window[i] = e;
  }
  return __syncthreads_and(ok) != 0;
}
// A key's codes and exponents (kNoKey: past kend, or its page is not there).
struct KeyAt {
  const unsigned char *codes, *expo;
  bool there;
};
template <class Row>
__device__ __forceinline__ KeyAt key_at(const IndexScoreParams &p, const int *window, int pg0, int key, int kend) {
  const int pg = page_of(p, key), e = key < kend ? window[pg - pg0] : -1, off = key - pg * p.block;
  const unsigned char *page = p.cache + (int64_t)e * p.page_bytes, *none = reinterpret_cast<const unsigned char *>(kNoKey);
  KeyAt k;
  k.there = e >= 0;
  k.codes = k.there ? page + (int64_t)off * Row::CODES : none;
  k.expo = k.there ? page + (int64_t)p.block * Row::CODES + (int64_t)off * 4 : none;
  return k;
}
__device__ __forceinline__ void fill_none(float *row, int from, int to) {
  for (int i = from + (int)threadIdx.x; i < to; i += 256) row[i] = -INFINITY;
}

template <int H, int D, int FMT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) index_rows_kernel(const IndexScoreParams p) {
  using Row = KeyRow<D, FMT>;
  constexpr int MT = H > 32 ? H / 32 : 1, ROWS = H < 32 ? H / 2 : 16;  // row tiles; their accumulators with a head in them
  constexpr int NC = Row::CODES / 32, U = Row::CPE / 8;               // pieces of a key in a lane; their steps
  __shared__ int window[kMostChunk];
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const int tile = (int)blockIdx.x % p.tiles, k0 = (int)blockIdx.x / p.tiles * p.chunk, t = p.first + tile;
  int r = 0, lim = -1;  // keys of the token, -1: a token of no request
  if (p.req.R > 0) {
    r = __builtin_amdgcn_readfirstlane(p.req.of(t));
    const int at = p.req.start(r), n = p.req.tokens(r);
    if (t >= at && t < at + n) lim = max(p.req.kv(r) - n + (t - at) + 1, 0);
  }
  lim = __builtin_amdgcn_readfirstlane(lim);
  if (p.limits != nullptr && k0 == 0 && threadIdx.x == 0) p.limits[tile] = min(max(lim, 0), p.L);
  if (lim < 0) return;
  float *out = p.out + (int64_t)tile * p.L;
  const int k1 = min(k0 + p.chunk, p.L), kend = min(k1, lim);
  fill_none(out, max(k0, kend), k1);
  if (kend <= k0) return;

  // operand of step (c, u): channels CPE (2 c + g32) + 8 u ..
  i32x4 q[MT][NC * U];
  float wv[MT][ROWS];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int h = 32 * m + l32;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int u = 0; u < U; ++u)
        q[m][c * U + u] = h < H ? ld_global_16(p.q + (((int64_t)t * H + h) * D + Row::CPE * (2 * c + g32) + 8 * u) * 2) : i32x4{0, 0, 0, 0};
  }
  {
    const float wl = lane < H ? weight_at(p, (int64_t)t * H + lane) : 0.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int a = 0; a < ROWS; ++a) wv[m][a] = __shfl(wl, 32 * m + score_row(a, g32), 64);
  }
  const float least = p.relu ? 0.0f : -INFINITY;
  fill_window<256>(p, window, r, k0, kend);
  const int pg0 = page_of(p, k0);

  struct Piece {
    i32x4 codes[NC];
    uint32_t expo;
    bool there;
  };
  auto load = [&](Piece &x, int sub) {
    const KeyAt k = key_at<Row>(p, window, pg0, k0 + 32 * sub + l32, kend);
    x.there = k.there;
#pragma unroll
    for (int c = 0; c < NC; ++c) x.codes[c] = ld_16(k.codes + 16 * (2 * c + g32));
    x.expo = FMT == KEY_BF16 ? 0u : ld_4(k.expo);
  };
  auto score = [&](const Piece &x, int sub) {
    f32x16 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int a = 0; a < 16; ++a) acc[m][a] = 0.0f;
    const uint32_t mine = FMT == KEY_MXFP4 ? x.expo >> (8 * g32) : x.expo;  // byte of piece c: 2 c + g32, c
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint32_t e = (mine >> (FMT == KEY_MXFP4 ? 16 * c : 8 * c)) & 255u;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const i32x4 k = key_values<FMT>(x.codes[c], u, e);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(q[m][c * U + u]), as_bf16x8(k), acc[m], 0, 0, 0);
      }
    }
    float part = 0.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int a = 0; a < ROWS; ++a) part = fmaf(__builtin_elementwise_maximum(acc[m][a], least), wv[m][a], part);
    part = sum_halves(part);
    const int key = k0 + 32 * sub + l32;
    if (g32 == 0 && key < kend) out[key] = x.there ? part : -INFINITY;
  };
  const int nsub = (kend - k0 + 31) / 32;
  Piece a, b;  // (tiles past the last: kNoKey)
  load(a, w);
  load(b, w + 4);
  for (int sub = w; sub < nsub; sub += 8) {
    score(a, sub);
    load(a, sub + 8);
    if (sub + 4 < nsub) score(b, sub + 4);
    load(b, sub + 12);
  }
}

template <int H, int D, int FMT>
struct IndexTile {
  using Row = KeyRow<D, FMT>;
  static constexpr int TPW = 64 / H, TT = 4 * TPW;  // tokens of a wave, of a workgroup
  static constexpr int KT = 64, RB = 2 * D, CHUNKS = RB / 16;  // keys of a tile; bytes and 16-byte chunks of a widened row
  static constexpr int CPR = Row::CODES / 16, U = Row::CPE / 8;  // pieces of a key's codes; chunks of a piece
  static constexpr int N = KT * CPR, NL = (N + 255) / 256;       // pieces of a tile, of a thread
  // rows are RB apart on the 256 bytes of banks: chunks permuted so that 16 rows read at one chunk fall on distinct ones
  static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ ((row / (256 / RB)) & (CHUNKS - 1))) * 16); }
};

template <int H, int D, int FMT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) index_tiles_kernel(const IndexScoreParams p) {
  using C = IndexTile<H, D, FMT>;
  using Row = typename C::Row;
  constexpr int TPW = C::TPW, KS = D / 16;
  __shared__ __attribute__((aligned(16))) unsigned char K[2][C::KT * C::RB];
  __shared__ int window[kMostChunk];
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const int tile0 = (int)blockIdx.x % p.tiles * C::TT, k0 = (int)blockIdx.x / p.tiles * p.chunk, k1 = min(k0 + p.chunk, p.L);
  const int t0 = p.first + tile0, t1 = min(t0 + C::TT, p.first + p.tokens), my0 = t0 + w * TPW;  // the wave's first token

  i32x4 q[2][KS];
  float wv[2][16];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int row = 32 * m + l32;
    const bool ok = my0 + row / H < t1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      q[m][ks] = ok ? ld_global_16(p.q + (((int64_t)my0 * H + row) * D + 16 * ks + 8 * g32) * 2) : i32x4{0, 0, 0, 0};
  }
  {
    const float wl = my0 + lane / H < t1 ? weight_at(p, (int64_t)my0 * H + lane) : 0.0f;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int a = 0; a < 16; ++a) wv[m][a] = __shfl(wl, 32 * m + score_row(a, g32), 64);
  }
  const float least = p.relu ? 0.0f : -INFINITY;

  // the tile's tokens, request by request: [ta, tb) are of one
  for (int ta = t0; ta < t1;) {
    int r = 0, at = 0, n = 0;
    if (p.req.R > 0) {
      r = __builtin_amdgcn_readfirstlane(p.req.of(ta));
      at = __builtin_amdgcn_readfirstlane(p.req.start(r));
      n = __builtin_amdgcn_readfirstlane(p.req.tokens(r));
    }
    if (ta < at || ta >= at + n) {  // of no request
      if (p.limits != nullptr && k0 == 0 && threadIdx.x == 0) p.limits[ta - p.first] = 0;
      ++ta;
      continue;
    }
    const int tb = min(t1, at + n), kv = __builtin_amdgcn_readfirstlane(p.req.kv(r));
    auto keys_of = [&](int t) { return max(kv - n + (t - at) + 1, 0); };
    if (p.limits != nullptr && k0 == 0)
      for (int t = ta + (int)threadIdx.x; t < tb; t += 256) p.limits[t - p.first] = min(keys_of(t), p.L);
    const int kend = min(k1, keys_of(tb - 1));
    for (int t = ta; t < tb; ++t) fill_none(p.out + (int64_t)(t - p.first) * p.L, max(k0, kend), k1);
    if (kend > k0) {
      __syncthreads();  // the window's readers are done
      const bool all_there = fill_window<256>(p, window, r, k0, kend);
      const int pg0 = page_of(p, k0);
      const bool works = my0 < tb && my0 + TPW > ta;  // wave-uniform
      i32x4 raw[C::NL];
      uint32_t expo[C::NL];
      auto load = [&](int j) {
#pragma unroll
        for (int i = 0; i < C::NL; ++i) {
          const int x = (int)threadIdx.x + 256 * i;
          if (C::N % 256 != 0 && x >= C::N) break;
          const KeyAt k = key_at<Row>(p, window, pg0, k0 + C::KT * j + x / C::CPR, kend);
          raw[i] = ld_16(k.codes + 16 * (x % C::CPR));
          expo[i] = FMT == KEY_BF16 ? 0u : ld_4(k.expo);
        }
      };
      auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < C::NL; ++i) {
          const int x = (int)threadIdx.x + 256 * i, row = x / C::CPR, c = x % C::CPR;
          if (C::N % 256 != 0 && x >= C::N) break;
          const uint32_t e = (expo[i] >> (8 * (c * Row::CPE / 32))) & 255u;
#pragma unroll
          for (int u = 0; u < C::U; ++u) *reinterpret_cast<i32x4 *>(K[buf] + C::at(row, c * C::U + u)) = key_values<FMT>(raw[i], u, e);
        }
      };
      const int nt = (kend - k0 + C::KT - 1) / C::KT;
      load(0);
      for (int j = 0; j < nt; ++j) {
        store(j & 1);
        load(j + 1);  // (past the last: kNoKey)
        __syncthreads();  // tile j is whole; its buffer's readers of two tiles ago passed the barrier before
        if (!works) continue;
        float part[2][TPW];
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          f32x16 acc[2];
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int a = 0; a < 16; ++a) acc[m][a] = 0.0f;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const i32x4 k = *reinterpret_cast<const i32x4 *>(K[j & 1] + C::at(32 * sub + l32, 2 * ks + g32));
#pragma unroll
            for (int m = 0; m < 2; ++m)
              acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(q[m][ks]), as_bf16x8(k), acc[m], 0, 0, 0);
          }
#pragma unroll
          for (int tl = 0; tl < TPW; ++tl) part[sub][tl] = 0.0f;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int a = 0; a < 16; ++a) {
              const int tl = (32 * m + 8 * (a >> 2)) / H;
              part[sub][tl] = fmaf(__builtin_elementwise_maximum(acc[m][a], least), wv[m][a], part[sub][tl]);
            }
        }
        // two sums at a time: the low lanes get the first one's, the high lanes the second's
        auto put = [&](float x, float y, int t, int key) {
          const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
          float v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
          if (key >= keys_of(t) || (!all_there && key < kend && window[page_of(p, key) - pg0] < 0)) v = -INFINITY;
          if (t >= ta && t < tb && key < kend) p.out[(int64_t)(t - p.first) * p.L + key] = v;
        };
        const int key0 = k0 + C::KT * j;
        if constexpr (TPW == 1) {
          put(part[0][0], part[1][0], my0, key0 + lane);
        } else {
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int tl = 0; tl < TPW; tl += 2) put(part[sub][tl], part[sub][tl + 1], my0 + tl + g32, key0 + 32 * sub + l32);
        }
      }
      __syncthreads();  // the tiles' readers are done
    }
    ta = tb;
  }
}

template <int H, int D, int FMT>
static int launch_scores(IndexScoreParams p, hipStream_t st) {
  using C = IndexTile<H, D, FMT>;
  // single tokens: a request has fewer than two on average
  const bool rows = p.req.query_starts == nullptr || p.req.R == 0 || p.req.T < 2 * (int64_t)p.req.R;
  p.tiles = rows ? p.tokens : (p.tokens + C::TT - 1) / C::TT;
  // keys of a workgroup: as many as leave four workgroups for every compute unit
  p.chunk = kMostChunk;
  const auto chunks = [&] { return p.L > 0 ? ((int64_t)p.L + p.chunk - 1) / p.chunk : 1; };
  while (p.chunk > 128 && p.tiles * chunks() < 1024) p.chunk /= 2;
  const int64_t n = p.tiles * chunks();
  DSA_REQUIRE(n < (1ll << 31), "dsa_paged_index_scores: too many tokens for one call");
  if (rows) hipLaunchKernelGGL((index_rows_kernel<H, D, FMT>), dim3((unsigned)n), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((index_tiles_kernel<H, D, FMT>), dim3((unsigned)n), dim3(256), 0, st, p);
  return check_launch("dsa_paged_index_scores");
}
template <int H, int D>
static int launch_scores(const IndexScoreParams &p, int fmt, hipStream_t st) {
  if (fmt == KEY_BF16) return launch_scores<H, D, KEY_BF16>(p, st);
  return fmt == KEY_MXFP8 ? launch_scores<H, D, KEY_MXFP8>(p, st) : launch_scores<H, D, KEY_MXFP4>(p, st);
}
int launch_index_scores(IndexScoreParams p, int64_t H, int64_t D, int fmt, hipStream_t st) {
  if (D == 128) return H == 64 ? launch_scores<64, 128>(p, fmt, st) : H == 32 ? launch_scores<32, 128>(p, fmt, st) : launch_scores<16, 128>(p, fmt, st);
  return H == 64 ? launch_scores<64, 64>(p, fmt, st) : H == 32 ? launch_scores<32, 64>(p, fmt, st) : launch_scores<16, 64>(p, fmt, st);
}

}  // namespace dsa
