// The indexer's scores of new tokens over a paged cache of index keys, on gfx950:
//   score[t, s] = sum_h w[t, h] relu(q[t, h] . k[s])   for the positions s that token t sees, -inf for the others.
//
// As in the dense indexer the rows of a 32x32x16 MFMA are (token, head) pairs and its columns 32 keys, and ReLU, weight
// and the sum over heads run on the accumulators.  MX keys are widened to bf16, exactly, in front of the product: the
// matrix instructions that take 8-bit codes keep fewer bits of their sums than 32 (a score was off by 1.5e-5 of the scores'
// size; this way 1e-7), and every key that is read serves 16 products at least.
//
// Two kernels.  Single tokens, or the few of a request that fill 64 (token, head) rows (index_rows_kernel): a workgroup's waves
// take the 32-key tiles of a unit in turn, straight from memory to operand registers (a lane's 16-byte piece of a key is two
// steps' operands in MXFP8 and four in MXFP4: the order of the channels in a product is free), two tiles ahead, without a
// barrier.  Several tokens of a request (index_tiles_kernel): four waves with the (token, head) rows of 4 * 64 / H tokens share
// tiles of 64 keys in LDS, widened as they enter it.
//
// A unit is a token (or tile of tokens) with its request's keys in blocks of 128, and behind them the columns that no token
// of it sees, in blocks of -inf to write.  All units' blocks, one after the other, are split evenly over the workgroups
// that the card holds, on the device, from the lengths: the host knows none of them (64 single tokens 99 -> 67 us, prompts 127 ->
// 109).
//
// Single tokens are bound by the keys' bytes: 64 tokens over 301 .. 65536 MXFP8 keys, 64 heads of 128 channels, 65 us, 4.5 TB/s.
// Several tokens are bound by the MFMAs and the ReLU and weights beside them, which the SIMD overlaps in part: 5 prompts of 33
// .. 512 tokens on 1024 .. 16384 MXFP4 keys, 32 heads, 77 to 81 us, 730 TFLOP/s (of a CU's busy time MFMA 41 %, VALU 41 %); without the
// weights' work it would be 69, without the conversion and the keys' loads 63.  At 64 channels a tile is half the products between the
// same two barriers: 3 prompts of 100 .. 700 tokens on 1024 .. 8192 keys, 16 heads, 24 to 26 us in each type, 430 TFLOP/s.
// Most of index_tiles_kernel's forms of 128 channels spill 2 to 9 registers, read once a piece, none among a tile's products.
#include <type_traits>

#include "index_keys.hpp"
#include "wave_ops.hpp"

namespace dsa {

constexpr int kWindowPages = 2048;  // pages of a unit that a workgroup has in LDS
constexpr int kBlockKeys = 128;
constexpr int kMostSpan = 65536 - kBlockKeys;  // past a column, below 2^31 - 65536, it stays below 2^31

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
// -inf into columns [from, to) of a row.
__device__ __forceinline__ void fill_none(float *row, int from, int to) {
  int head = from + (int)((16u - (uint32_t)reinterpret_cast<uintptr_t>(row + from) % 16u) % 16u / 4u);  // 16-byte stores from here
  head = head < to ? head : to;
  const int wide = (to - head) / 4;
  if (from + (int)threadIdx.x < head) row[from + threadIdx.x] = -INFINITY;
  for (int i = (int)threadIdx.x; i < wide; i += 256)
    reinterpret_cast<f32x4 *>(row + head)[i] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (head + 4 * wide + (int)threadIdx.x < to) row[head + 4 * wide + threadIdx.x] = -INFINITY;
}

// The blocks of a request's units: its tokens that are scored by TT, each with nb blocks of keys and fb of columns to fill.
struct RequestUnits {
  int ta, n, nb, fb;  // first token, tokens
};
template <int TT>
struct ScoreUnits {
  static constexpr int FILL = TT == 1 ? 4096 : 16384 / TT;  // columns of a block to fill: about the time of a block of keys
  static __device__ __forceinline__ RequestUnits of(const IndexScoreParams &p, int r) {
    RequestUnits u;
    const int at = p.req.start(r), tb = min(at + p.req.tokens(r), p.first + p.tokens);
    u.ta = max(at, p.first);
    u.n = max(tb - u.ta, 0);
    const int keys = min(p.req.kv(r), p.L);
    u.nb = (keys + kBlockKeys - 1) / kBlockKeys;
    u.fb = p.fill ? max(p.L - u.nb * kBlockKeys + FILL - 1, 0) / FILL : 0;
    return u;
  }
  static __device__ __forceinline__ uint32_t blocks(const IndexScoreParams &p, int r) {
    const RequestUnits u = of(p, r);
    return (uint32_t)((u.n + TT - 1) / TT) * (uint32_t)(u.nb + u.fb);
  }
};
// The workgroup's range [at, end) of all blocks, and the request at `at`: 256 requests' first blocks stand in `begin`.
struct ScoreWalk {
  uint32_t at, end;
  int chunk, i;  // requests 256 chunk .., of which request i is at hand
};
struct ScoreLds {
  uint32_t tmp[4], begin[257];
};
template <int TT>
__device__ __forceinline__ void load_requests(const IndexScoreParams &p, ScoreLds &s, int chunk, uint32_t base) {
  const int r = 256 * chunk + (int)threadIdx.x;
  uint32_t total;
  const uint32_t mine = block_scan<256>(r < p.req.R ? ScoreUnits<TT>::blocks(p, r) : 0u, s.tmp, total);
  s.begin[threadIdx.x] = add_sat(base, mine);
  if (threadIdx.x == 0) s.begin[256] = add_sat(base, total);
  __syncthreads();
}
template <int TT>
__device__ __forceinline__ ScoreWalk start_walk(const IndexScoreParams &p, ScoreLds &s) {
  const int chunks = (p.req.R + 255) / 256;
  uint32_t total = 0;
  for (int c = 0; c < chunks; ++c) {
    load_requests<TT>(p, s, c, total);
    total = s.begin[256];
    __syncthreads();
  }
  const uint32_t per = total / gridDim.x + (total % gridDim.x != 0);
  ScoreWalk k;
  const uint64_t at = (uint64_t)blockIdx.x * per;
  k.at = at < total ? (uint32_t)at : total;
  k.end = per < total - k.at ? k.at + per : total;
  k.chunk = 0;
  k.i = 0;
  if (chunks > 1 && k.at < k.end) {
    uint32_t base = 0;
    for (int c = 0; c < chunks; ++c) {
      load_requests<TT>(p, s, c, base);
      base = s.begin[256];
      k.chunk = c;
      if (base > k.at) break;  // (uniform)
      __syncthreads();
    }
  }
  return k;
}
// The piece at k.at: request, its units' first block, the unit's tokens and its blocks [b0, b1); k.at moves past it.
struct ScorePiece {
  int r, ta, tb, nb, b0, b1;
};
template <int TT>
__device__ __forceinline__ ScorePiece next_piece(const IndexScoreParams &p, ScoreLds &s, ScoreWalk &k) {
  while (true) {
    if (k.i == 256) {  // (uniform, as are the loop's other values)
      const uint32_t base = s.begin[256];
      __syncthreads();
      load_requests<TT>(p, s, ++k.chunk, base);
      k.i = 0;
    }
    if (s.begin[k.i + 1] > k.at) break;
    ++k.i;
  }
  ScorePiece x;
  x.r = __builtin_amdgcn_readfirstlane(256 * k.chunk + k.i);
  const RequestUnits u = ScoreUnits<TT>::of(p, x.r);
  const uint32_t off = k.at - s.begin[k.i], ub = (uint32_t)(u.nb + u.fb), tile = off / ub, b0 = off - tile * ub;
  x.ta = __builtin_amdgcn_readfirstlane(u.ta + (int)tile * TT);
  x.tb = __builtin_amdgcn_readfirstlane(min(x.ta + TT, u.ta + u.n));
  x.nb = __builtin_amdgcn_readfirstlane(u.nb);
  x.b0 = __builtin_amdgcn_readfirstlane((int)b0);
  x.b1 = __builtin_amdgcn_readfirstlane((int)(ub - b0 < k.end - k.at ? ub : b0 + (k.end - k.at)));
  k.at += (uint32_t)(x.b1 - x.b0);
  return x;
}
// The piece's blocks to fill.
template <int TT>
__device__ __forceinline__ void fill_piece(const IndexScoreParams &p, const ScorePiece &x) {
  constexpr int FILL = ScoreUnits<TT>::FILL;
  if (x.b1 <= x.nb) return;
  const int keys = x.nb * kBlockKeys, from = keys + max(x.b0 - x.nb, 0) * FILL;
  const int64_t to = (int64_t)keys + (int64_t)(x.b1 - x.nb) * FILL;
  for (int t = x.ta; t < x.tb; ++t) fill_none(p.out + (int64_t)(t - p.first) * p.L, from, to < p.L ? (int)to : p.L);
}
__device__ __forceinline__ void write_windows(const IndexScoreParams &p) {
  if (p.windows == nullptr) return;
  for (int i = (int)blockIdx.x * 256 + (int)threadIdx.x; i < p.tokens; i += (int)gridDim.x * 256) {
    p.windows[i] = 0;
    p.windows[p.tokens + i] = p.req.R > 0 ? min(max(p.req.keys_of(p.first + i, p.req.of_lane(p.first + i)), 0), p.L) : 0;
  }
}

// NT tokens of a request at a time: one, or the 64 / H that fill two row tiles.
template <int H, int D, int FMT, int NT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) index_rows_kernel(const IndexScoreParams p) {
  using Row = KeyRow<D, FMT>;
  constexpr int RT = NT * H;                                              // rows
  constexpr int MT = RT > 32 ? RT / 32 : 1, ROWS = RT < 32 ? RT / 2 : 16;  // row tiles; their accumulators with a head in them
  constexpr int NC = Row::CODES / 32, U = Row::CPE / 8;                   // pieces of a key in a lane; their steps
  __shared__ int window[kWindowPages];
  __shared__ ScoreLds units;
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const float least = p.relu ? 0.0f : -INFINITY;
  write_windows(p);
  ScoreWalk walk = start_walk<NT>(p, units);
  while (walk.at < walk.end) {
    const ScorePiece x = next_piece<NT>(p, units, walk);
    fill_piece<NT>(p, x);
    if (x.b0 >= x.nb) continue;
    const int t = x.ta, kb1 = min(min(x.b1, x.nb) * kBlockKeys, p.L);
    const int most = __builtin_amdgcn_readfirstlane(p.req.keys_of(x.tb - 1, x.r));  // keys that the last token sees
    // the rows that the lane writes: of tokens 2 i + g32 (one token: its)
    constexpr int NP = NT > 1 ? NT / 2 : 1;
    float *out[NP];
    int sees[NP];  // (of a token that is not there: -1)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int tl = t + (NT > 1 ? 2 * i + g32 : 0);
      sees[i] = tl < x.tb ? max(most - (x.tb - 1 - tl), 0) : -1;
      out[i] = p.out + (int64_t)(tl - p.first) * p.L;
    }

    // operand of step (c, u): channels CPE (2 c + g32) + 8 u ..
    const int rows = (x.tb - t) * H;
    i32x4 q[MT][NC * U];
    float wv[MT][ROWS];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int h = 32 * m + l32;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = 0; u < U; ++u)
          q[m][c * U + u] = h < rows ? ld_global_16(p.q + (((int64_t)t * H + h) * D + Row::CPE * (2 * c + g32) + 8 * u) * 2) : i32x4{0, 0, 0, 0};
    }
    const float wl = lane < rows ? weight_at(p, (int64_t)t * H + lane) : 0.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int a = 0; a < ROWS; ++a) wv[m][a] = __shfl(wl, 32 * m + score_row(a, g32), 64);

    for (int k0 = x.b0 * kBlockKeys; k0 < kb1; k0 += p.span) {
      const int k1 = min(k0 + p.span, kb1), kend = min(k1, most);  // columns; keys that a token sees
      __syncthreads();  // the window's readers are done
      if (kend > k0) fill_window<256>(p, window, x.r, k0, kend);
      const int pg0 = page_of(p, k0);
      struct Piece {
        i32x4 codes[NC];
        uint32_t expo;
        bool there;
      };
      auto load = [&](Piece &y, int sub) {
        const KeyAt k = key_at<Row>(p, window, pg0, k0 + 32 * sub + l32, kend);
        y.there = k.there;
#pragma unroll
        for (int c = 0; c < NC; ++c) y.codes[c] = ld_16(k.codes + 16 * (2 * c + g32));
        y.expo = FMT == KEY_BF16 ? 0u : ld_4(k.expo);
      };
      auto score = [&](const Piece &y, int sub) {
        f32x16 acc[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int a = 0; a < 16; ++a) acc[m][a] = 0.0f;
        const uint32_t mine = FMT == KEY_MXFP4 ? y.expo >> (8 * g32) : y.expo;  // byte of piece c: 2 c + g32, c
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint32_t e = (mine >> (FMT == KEY_MXFP4 ? 16 * c : 8 * c)) & 255u;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const i32x4 k = key_values<FMT>(y.codes[c], u, e);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(q[m][c * U + u]), as_bf16x8(k), acc[m], 0, 0, 0);
          }
        }
        float part[NT];
#pragma unroll
        for (int tl = 0; tl < NT; ++tl) part[tl] = 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int a = 0; a < ROWS; ++a) {
            const int tl = (32 * m + 8 * (a >> 2)) / H;
            part[tl] = fmaf(__builtin_elementwise_maximum(acc[m][a], least), wv[m][a], part[tl]);
          }
        const int key = k0 + 32 * sub + l32;
        if constexpr (NT == 1) {
          part[0] = sum_halves(part[0]);
          if (g32 == 0 && key < k1) out[0][key] = y.there ? part[0] : -INFINITY;
        } else {
          // two sums at a time: the low lanes get the first one's, the high lanes the second's
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(part[2 * i]), __float_as_uint(part[2 * i + 1]), false, false);
            const float v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
            if (sees[i] >= 0 && key < k1) out[i][key] = y.there && key < sees[i] ? v : -INFINITY;
          }
        }
      };
      const int nsub = (k1 - k0 + 31) / 32;
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
  __shared__ int window[kWindowPages];
  __shared__ ScoreLds units;
  const int lane = lane_id(), w = wave_id(), g32 = lane >> 5, l32 = lane & 31;
  const float least = p.relu ? 0.0f : -INFINITY;
  write_windows(p);
  ScoreWalk walk = start_walk<C::TT>(p, units);
  while (walk.at < walk.end) {
    const ScorePiece x = next_piece<C::TT>(p, units, walk);
    fill_piece<C::TT>(p, x);
    if (x.b0 >= x.nb) continue;
    // Tiles that half of the waves would have: the other half takes the second 32 keys of every 64.
    const bool halves = x.tb - x.ta <= C::TT / 2;  // (uniform)
    const int my0 = x.ta + (halves ? w & 1 : w) * TPW;  // the wave's first token
    const int at = __builtin_amdgcn_readfirstlane(p.req.start(x.r)), n = __builtin_amdgcn_readfirstlane(p.req.tokens(x.r));
    const int kv = __builtin_amdgcn_readfirstlane(p.req.kv(x.r));
    auto keys_of = [&](int t) { return token_keys(kv, n, t - at); };
    const int kb1 = min(min(x.b1, x.nb) * kBlockKeys, p.L), most = keys_of(x.tb - 1);

    i32x4 q[2][KS];
    float wv[2][16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int row = 32 * m + l32;
      const bool ok = my0 + row / H < x.tb;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        q[m][ks] = ok ? ld_global_16(p.q + (((int64_t)my0 * H + row) * D + 16 * ks + 8 * g32) * 2) : i32x4{0, 0, 0, 0};
    }
    const float wl = my0 + lane / H < x.tb ? weight_at(p, (int64_t)my0 * H + lane) : 0.0f;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int a = 0; a < 16; ++a) wv[m][a] = __shfl(wl, 32 * m + score_row(a, g32), 64);
    const bool works = my0 < x.tb;  // wave-uniform

    for (int k0 = x.b0 * kBlockKeys; k0 < kb1; k0 += p.span) {
      const int k1 = min(k0 + p.span, kb1), kend = min(k1, most);  // columns; keys that a token sees
      __syncthreads();  // the readers of the window and the tiles are done
      const bool all_there = kend > k0 && fill_window<256>(p, window, x.r, k0, kend);
      const int pg0 = page_of(p, k0);
      i32x4 raw[C::NL];
      uint32_t expo[C::NL];
      auto load = [&](int j) {
        if (p.whole_tiles) {
          // The tile lies on one page, its codes and its exponents in a row each: one address a wave (2048 tokens over 8192 MXFP8
          // keys 254 -> 243 us).  Keys past kend are masked below, as are those of a page that is not there, for which page 0 stands.
          const int key = min(k0 + C::KT * j, kend - 1) & ~(C::KT - 1), pg = page_of(p, key), off = key - pg * p.block;
          const int e = max(__builtin_amdgcn_readfirstlane(window[pg - pg0]), 0);
          const unsigned char *page = p.cache + (int64_t)e * p.page_bytes;
          const unsigned char *codes = page + (int64_t)off * Row::CODES, *expos = page + (int64_t)p.block * Row::CODES + (int64_t)off * 4;
#pragma unroll
          for (int i = 0; i < C::NL; ++i) {
            const int y = (int)threadIdx.x + 256 * i;
            if (C::N % 256 != 0 && y >= C::N) break;
            raw[i] = ld_16(codes + (uint32_t)y * 16u);
            expo[i] = FMT == KEY_BF16 ? 0u : ld_4(expos + (uint32_t)(y / C::CPR) * 4u);
          }
          return;
        }
#pragma unroll
        for (int i = 0; i < C::NL; ++i) {
          const int y = (int)threadIdx.x + 256 * i;
          if (C::N % 256 != 0 && y >= C::N) break;
          const KeyAt k = key_at<Row>(p, window, pg0, k0 + C::KT * j + y / C::CPR, kend);
          raw[i] = ld_16(k.codes + 16 * (y % C::CPR));
          expo[i] = FMT == KEY_BF16 ? 0u : ld_4(k.expo);
        }
      };
      auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < C::NL; ++i) {
          const int y = (int)threadIdx.x + 256 * i, row = y / C::CPR, c = y % C::CPR;
          if (C::N % 256 != 0 && y >= C::N) break;
          const uint32_t e = (expo[i] >> (8 * (c * Row::CPE / 32))) & 255u;
#pragma unroll
          for (int u = 0; u < C::U; ++u) *reinterpret_cast<i32x4 *>(K[buf] + C::at(row, c * C::U + u)) = key_values<FMT>(raw[i], u, e);
        }
      };
      // the rows that the lane writes: of tokens 2 i + g32 (one token a wave: its)
      constexpr int NP = TPW > 1 ? TPW / 2 : 1;
      float *row[NP];
      int sees[NP];
      bool mine[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int t = my0 + (TPW > 1 ? 2 * i + g32 : 0);
        mine[i] = t < x.tb;
        sees[i] = keys_of(t);
        row[i] = p.out + (int64_t)(t - p.first) * p.L + k0;
      }
      const int least_keys = min(keys_of(my0), k1);
      const int nt = (k1 - k0 + C::KT - 1) / C::KT;
      if (kend <= k0) {  // columns of a block of keys that none of these tokens sees
        for (int t = x.ta; t < x.tb; ++t) fill_none(p.out + (int64_t)(t - p.first) * p.L, k0, k1);
        continue;
      }
      load(0);
      for (int j = 0; j < nt; ++j) {
        store(j & 1);
        load(j + 1);  // (past the last: kNoKey)
        __syncthreads();  // tile j is whole; its buffer's readers of two tiles ago passed the barrier before
        if (!works) continue;
        // Tiles of 32 rows by 32 keys, two or four; a tile's ReLU and weights beside the next one's products, in one stream,
        // since the SIMD overlaps the two within a wave far more than across waves.
        float part[2][TPW];
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int tl = 0; tl < TPW; ++tl) part[sub][tl] = 0.0f;
        f32x16 acc[2];
        i32x4 k[KS];
        auto weigh = [&](int sub, int m) {
#pragma unroll
          for (int a = 0; a < 16; ++a) {
            const int tl = (32 * m + 8 * (a >> 2)) / H;
            part[sub][tl] = fmaf(__builtin_elementwise_maximum(acc[m][a], least), wv[m][a], part[sub][tl]);
          }
        };
        auto tiles = [&](auto count, const unsigned char *keys) {  // of 32-key tiles from `keys` on
#pragma unroll
          for (int tile = 0; tile < decltype(count)::value; ++tile) {
            const int m = tile & 1;
            if (m == 0)
#pragma unroll
              for (int ks = 0; ks < KS; ++ks) k[ks] = *reinterpret_cast<const i32x4 *>(keys + C::at(16 * tile + l32, 2 * ks + g32));
#pragma unroll
            for (int a = 0; a < 16; ++a) acc[m][a] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
              acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(q[m][ks]), as_bf16x8(k[ks]), acc[m], 0, 0, 0);
            if (tile > 0) weigh((tile - 1) >> 1, (tile - 1) & 1);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
              __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);  // and what goes beside it
            }
          }
          weigh((decltype(count)::value - 1) >> 1, 1);
        };
        if (halves) tiles(std::integral_constant<int, 2>(), K[j & 1] + (w >> 1) * 32 * C::RB);
        else tiles(std::integral_constant<int, 4>(), K[j & 1]);
        // two sums at a time: the low lanes get the first one's, the high lanes the second's
        const int at_key = C::KT * j;
        const bool inside = all_there && k0 + at_key + C::KT <= least_keys;  // (wave-uniform) every key is seen by every token
        auto put = [&](float y, float z, int i, int off) {
          const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(z), false, false);
          float v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
          if (TPW == 1 && off == C::KT) return;
          off += at_key;
          if (!inside) {
            keep_branch();
            const int key = k0 + off;
            if (key >= sees[i] || (!all_there && key < kend && window[page_of(p, key) - pg0] < 0)) v = -INFINITY;
            if (key >= k1) return;
          }
          if (mine[i]) row[i][off] = v;
        };
        if constexpr (TPW == 1) {
          // (halves: both halves of the wave have the one sum's two parts, and the low lanes' result is stored)
          if (!halves) put(part[0][0], part[1][0], 0, lane);
          else put(part[0][0], part[0][0], 0, g32 == 0 ? 32 * (w >> 1) + l32 : C::KT);
        } else {
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            if (sub == 1 && halves) break;
#pragma unroll
            for (int i = 0; i < NP; ++i) put(part[sub][2 * i], part[sub][2 * i + 1], i, 32 * (halves ? w >> 1 : sub) + l32);
          }
        }
      }
    }
  }
}

template <int H, int D, int FMT>
static int launch_scores(IndexScoreParams p, hipStream_t st) {
  using C = IndexTile<H, D, FMT>;
  // Tokens of a unit, by those that a request has on average.  Replays of 32 requests, 8192 .. 32768 keys, us, tiles of tokens in LDS
  // and 64 rows from memory:
  //   16 heads  2 tokens MXFP8 42, 32, MXFP4 41, 28, bf16 42, 39; 4 tokens 43, 35; 43, 32; 44, 43; 6 tokens 47, 46; 48, 41; 47, 63
  //   32 heads  2 tokens MXFP8 41, 35, MXFP4 41, 32, bf16 40, 42; 4 tokens 48, 48; 48, 44; 45, 62; 6 tokens 58, 62; 57, 54; 55, 84
  //   64 heads  2 tokens MXFP8 48, 46, MXFP4 48, 41, bf16 52, 63; 3 tokens MXFP8 57, 60
  // and of 64 requests, 301 .. 65536 keys: 2 tokens, 32 heads MXFP8 110, 83, MXFP4 90, 58; 4 tokens, 16 heads MXFP4 98, 61.
  const int64_t T = p.req.T, R = p.req.R;
  const int nt = p.req.query_starts == nullptr || R == 0 || T < 2 * R ? 1 : T <= (FMT == KEY_MXFP4 ? 2 : 1) * C::TPW * R ? C::TPW : C::TT;  // tokens of a unit
  const bool rows = nt < C::TT;
  p.whole_tiles = p.block % C::KT == 0;
  // With windows nobody needs the columns that no token sees.  A top-k that reads whole rows finds those of a small call in the caches
  // all the same where they were written: 64 tokens of up to 8192 keys in 32768 columns, top-2048, us, written and not 39, 43; of
  // 65536 keys in 65536, top-256 97, 97, in 131072 101, 95; 1361 tokens of 16384 keys in 32768, top-2048 124, 113.
  p.fill = p.windows == nullptr || (int64_t)p.tokens * p.L <= (4 << 20);
  const int64_t span = (int64_t)(kWindowPages - 2) * p.block / kBlockKeys * kBlockKeys;
  p.span = (int)(span < kMostSpan ? span : kMostSpan);
  // blocks, at most: fewer than 2^31 of them, and workgroups that all run at once
  const int fill = nt == 1 ? ScoreUnits<1>::FILL : nt == C::TPW ? ScoreUnits<C::TPW>::FILL : ScoreUnits<C::TT>::FILL;
  const int64_t units = nt == 1 ? p.tokens : (int64_t)p.tokens / nt + (p.tokens < p.req.R ? p.tokens : p.req.R);
  const int64_t n = units * (((int64_t)p.L + kBlockKeys - 1) / kBlockKeys + ((int64_t)p.L + fill - 1) / fill);
  DSA_REQUIRE(n < (1ll << 31), "dsa_paged_index_scores: too many tokens for one call");
  const int64_t most = 256 * (nt * H < 64 ? 4 : 2);
  const dim3 grid((unsigned)(n < 1 ? 1 : n < most ? n : most));
  if (rows && nt == 1) hipLaunchKernelGGL((index_rows_kernel<H, D, FMT, 1>), grid, dim3(256), 0, st, p);
  else if (rows) hipLaunchKernelGGL((index_rows_kernel<H, D, FMT, C::TPW>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((index_tiles_kernel<H, D, FMT>), grid, dim3(256), 0, st, p);
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
