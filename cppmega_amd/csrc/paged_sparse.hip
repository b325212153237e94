// SparseMLA of new tokens over the paged latent cache, on gfx950: each token attends to the cached rows that its top-k
// names by their positions in its request.
//
// Rows of 128 channels: paged_sparse_narrow.hip.  Rows of 576: the kernels of paged latent attention, for which a token is a
// request of one token whose pages are single rows.  Their workgroups have whole tokens, equal pieces of one, or even ranges of
// all tokens' picks, 64 at a time, and paged_combine_kernel adds the pieces of a token that was cut; the picks' slots are formed as
// a workgroup fills its window of pages.
//
// 64 tokens, 128 heads, top-2048, bf16: 67 us, 540 TFLOP/s, in units of 32 rows.  Its four computing waves, one a SIMD, bound it: of a
// replay of 74 us the products alone take 64, the rows' loads alone 54 (by registers, two more steps in flight, the whole took 80).
// The rows come through the L2s, 600 MB at 9 TB/s; those are not the limit, as 500 tokens of 16 heads, 1.2 GB, get 12 of them (99 us:
// loads alone 86, products alone 82, which overlap in part).  1024 tokens, 128 heads: of 581 us the products 520, the loads 167.
// 96 tokens, 16 heads, MXFP4: 37 us and 4.4 for the joining; of a replay of 46 the products alone 41, loads and widening alone 34.
#include "latent_paged.hpp"
#include "paged_sparse.hpp"

namespace dsa {

// How a call with 576 channels is run: the rows of a unit.  A row that a unit reads serves all of its rows; fewer rows mean
// more units, of which fewer are cut, and their neighbours' reads of the same rows meet in an XCD's L2.  Replays of T tokens
// of as many requests (where marked *, of one), top-2048, us, fewer rows a unit and more:
//   bf16, 128 heads   of 32 and 64: T = 8* 34, 41; 32* 47, 48; 48 64, 73; 56 67, 79; of 64 and 128: 64 70, 80; 96 117, 120;
//                     192* 146, 155; 256* (no unit of 128 is cut) 174, 153; 400* 284, 275
//         64 heads    of 32 and 64: T = 2* 25, 34; 32* 37, 43; 64* 47, 48; 96 81, 77; 128 96, 91; of 64 and 128: 64* 48, 61
//         32 heads    of 32 and 64: T = 8* 27, 34; 64* 37, 44; 400* 112, 147
//         16 heads    of 16 (their waves share keys and channels) and 64: T = 8* 23, 32; 64* 31, 41; 400* 97, 150
//   MXFP4, 128 heads  of 32 and 64: T = 8* 36, 46; 32* 54, 53; 56 77, 83; 96* 115, 111; 256* 258, 213
//         64 heads    of 32 and 64: T = 16* 36, 45; 64* 54, 53; 128* 73, 76; 256* 135, 111
//         16 heads    of 16 and 32: T = 8* 26, 27; 96 49, 57; 400* 110, 122
struct SparseWidePlan {
  int wide, unit_rows, token_units, unit_blocks, nwg, min_blocks;
  int64_t per;  // blocks of a workgroup
};
// Ranges of whole units: nothing is cut, and nothing to join.
static bool all_whole(const SparseWidePlan &k) { return k.per % k.unit_blocks == 0; }
static bool nearly_all(int64_t units) { return units >= 192 && units <= 256; }
static SparseWidePlan sparse_wide_plan(int64_t T, int64_t topk, int64_t H, bool fp4) {
  SparseWidePlan r{};
  if (H <= 16) r.wide = 1;
  else if (H <= 32 || T * H <= 4096 || (H > 64 && nearly_all(T * ((H + 31) / 32)))) r.wide = 2;
  else r.wide = fp4 || H <= 64 || T * ((H + 127) / 128) < 256 ? 4 : 8;
  r.unit_rows = 16 * r.wide;
  r.token_units = (int)((H + r.unit_rows - 1) / r.unit_rows);
  r.unit_blocks = (int)((topk + paged_wide_keys() - 1) / paged_wide_keys());
  r.min_blocks = 256 / paged_wide_keys();  // picks that are worth a piece's beginning and end
  // Workgroups: a whole number of equal pieces of a unit each, so that none has the end of one unit and the beginning of the
  // next (112 tokens, 16 heads, bf16 64 us by even ranges of all blocks, 61 so; 96, 64 heads 77, 67; 224 units left whole 152,
  // 136), or, where that leaves much of the card idle, even ranges.
  const int64_t units = T * r.token_units;
  if (units <= 128 || nearly_all(units)) {
    const int most = 256 / (int)units, even = (r.unit_blocks + most - 1) / most, least = even > r.min_blocks ? even : r.min_blocks;
    const int per = r.unit_blocks - even <= 4 ? r.unit_blocks : least;  // (128 tokens, 32 heads, top-512 in two pieces 34, whole 28)
    const int pieces = (r.unit_blocks + per - 1) / per;
    r.per = per;
    r.unit_blocks = pieces * per;  // (blocks past the last pick hold none)
    r.nwg = (int)units * pieces;
  } else {
    // Units left whole, if that costs a workgroup no more than `most` blocks: a cut one has two beginnings and ends and is joined.
    // Even ranges and whole units, us, by the blocks that whole ones cost more (replays of one request's prompt):
    //   bf16, 16 rows   4: 257 tokens 37, 35; 420 59, 50;  7: 257 41, 41; 700 122, 112 (6);  10: 350 63, 58;  11: 257 46, 50
    //         32        4: 257 49, 43;  9: 257 56, 54;  10: 350 79, 68;  11: 257 58, 58;  15: 257 65, 68; 350 92, 89
    //         64        4: 257 57, 49;  8: 300 72, 72; 560 103, 104;  9: 257 70, 72;  10: 350 102, 99;  11: 257 75, 80; 420 175, 169
    //         128       4: 257 85, 72;  8: 300 111, 109; 560 167, 161;  9: 257 108, 109;  10: 350 161, 156;  11: 257 115, 124
    //   MXFP4, 16       4: 257 39, 38;  6: 560 65, 66;  7: 257 44, 46; 350 63, 58;  8: 300 49, 53; 700 169, 170;  9: 257 47, 52
    //         32        4: 257 50, 46;  7: 257 56, 56; 350 78, 70;  8: 300 60, 62; 700 198, 194;  9: 257 60, 63;  11: 257 63, 70
    //         64        4: 257 61, 59;  5: 350 86, 77;  6: 300 72, 77; 700 257, 256;  7: 257 72, 77; 350 104, 100;  9: 257 77, 88
    r.nwg = 256;
    const int64_t even = (units * r.unit_blocks + 255) / 256, whole = (units + 255) / 256 * r.unit_blocks;
    const int64_t most = !fp4 ? 10 : r.wide == 4 ? 5 : 7;
    r.per = whole - even <= most ? whole : even > r.min_blocks ? even : r.min_blocks;
  }
  r.min_blocks = (int)r.per;  // (what range_blocks has on the device)
  return r;
}

// Workgroups and blocks can be numbered.
bool paged_sparse_countable(int64_t T, int64_t topk, int64_t H, int64_t d_qk) {
  const int64_t units = T * ((H + 31) / 32);
  if (units >= (1ll << 26) || (d_qk == 128 && (units + 3) / 4 >= (1ll << 24))) return false;  // (four waves each, below 2^32 threads)
  bool ok = true;
  for (int fp4 = 0; d_qk == 576 && fp4 < 2; ++fp4) {
    const SparseWidePlan k = sparse_wide_plan(T, topk, H, fp4 != 0);
    ok = ok && T * k.token_units * (int64_t)k.unit_blocks < (1ll << 31);
  }
  return ok;
}

size_t paged_sparse_workspace(int64_t T, int64_t topk, int64_t H, int64_t d_qk, int64_t d_v) {
  if (d_qk == 128) return sparse_narrow_workspace(T, topk, H);
  size_t most = 0;  // of the two formats': the query does not know it
  for (int fp4 = 0; fp4 < 2; ++fp4) {
    const SparseWidePlan k = sparse_wide_plan(T, topk, H, fp4 != 0);
    const size_t n = all_whole(k) ? 0 : (size_t)k.nwg * 2 * (size_t)k.unit_rows * ((size_t)d_v + 2) * 4;
    most = n > most ? n : most;
  }
  return most;
}

int launch_paged_sparse(PagedParams p, const int32_t *indices, int64_t topk, int64_t d_qk, int64_t d_v, bool fp4, unsigned char *ws,
                        hipStream_t st) {
  const Picks picks{indices, p.table, p.req, p.W, (int)topk, p.block, p.block_shift, p.num_blocks};
  if (d_qk == 128) {
    SparseParams n{};
    n.q = p.q;
    n.cache = p.cache;
    n.picks = picks;
    n.out = p.out;
    n.lse = p.lse;
    n.H = p.H;
    n.sl2 = p.sl2;
    return launch_sparse_narrow(n, fp4, ws, st);
  }
  const SparseWidePlan k = sparse_wide_plan(p.T, topk, p.H, fp4);
  p.picks = picks;
  p.unit_rows = k.unit_rows;
  p.token_units = k.token_units;
  p.unit_blocks = k.unit_blocks;
  p.step_keys = paged_wide_keys();
  p.nwg = k.nwg;
  p.min_blocks = k.min_blocks;
  p.part_ml = (float *)ws;
  p.part_o = p.part_ml + (size_t)k.nwg * 2 * (size_t)k.unit_rows * 2;
  const int rc = launch_paged_wide(p, k.wide, fp4, true, st);
  if (rc || all_whole(k)) return rc;
  return launch_paged_combine(p, d_v, true, st);
}

}  // namespace dsa
