// serve_plan.cu -- host side of attention over caches: which kernel reads what, the workspace, and
// the sizes that the kernels' 32-bit counts hold.  No kernels here, so that it is tested alone.
#include <algorithm>
#include <cmath>

#include "fm_serve.cuh"

namespace fm {

// Up to so many rows an SM a merge block joins one row, its four warps a quarter of the pieces each:
// 512 rows of ~20 pieces, whole calls 42.2 -> 39.4 and 68.4 -> 64.5 us; 2048 rows 73.6 -> 77.6 us.
constexpr int64_t kMergeShared = 4;

CacheAttnPlan cache_attn_plan(int B, int L, int nh, int nkv, int d, int prefix_len, bool own, bool scored, int max_len,
                              int num_sms) {
  CacheAttnPlan p;
  const int64_t group = nh / nkv, rows_s = L * group, rows_p = B * rows_s;
  // Few rows to a key: attn_split_kernel, whose workers are warps, so that short pieces start and end
  // quickly (its row tiles past the first read the keys from L2 again).  More: attn_tc_kernel.
  // Whole calls, prefix by the one / by the other, 200 tokens of own cache: 32 rows (32
  // sequences of 16/16 heads, 4096 shared) 39 / 48 us, 64 rows (64 sequences) 61 / 70 us, 64 rows
  // (8 sequences of 32/4 heads, 16384 shared) 37 / 35 us, 128 rows (16 sequences, 8192) 32 / 33 us.
  p.tc_p = prefix_len > 0 && rows_p > kAttnSplitRows;
  // with slot weights the split kernel also leaves 4 bytes a row and slot: for one row tile only
  p.tc_s = own && rows_s > (scored ? kAttnRowTile : kAttnSplitRows);
  if (prefix_len > 0 && !p.tc_p) p.rt_p = static_cast<int>((rows_p + kAttnRowTile - 1) / kAttnRowTile);
  if (own && !p.tc_s) p.rt_s = static_cast<int>((rows_s + kAttnRowTile - 1) / kAttnRowTile);
  if (p.rt_p || p.rt_s) p.workers = num_sms * kAttnBlocksPerSm * kAttnWarps;
  auto add = [&](size_t bytes) {
    const size_t off = p.bytes;
    p.bytes = (p.bytes + bytes + 255) / 256 * 256;
    return off;
  };
  const size_t rows = p.workers ? (p.workers + static_cast<size_t>(nkv) * (p.rt_p + static_cast<size_t>(B) * p.rt_s)) * kAttnRowTile : 0;
  add(rows * d * sizeof(float));
  p.off_ml = add(rows * sizeof(float2));
  auto tc = [&](bool on, bool direct, int64_t nseq, int64_t item_rows, int& rps, int& workers, size_t& off_o, size_t& off_ml) {
    if (!on) return;
    rps = static_cast<int>((item_rows + kTcRows - 1) / kTcRows);
    workers = num_sms;
    const size_t n = (direct ? 2 * workers : workers + static_cast<size_t>(nseq) * rps * nkv) * kTcRows;
    off_o = add(n * d * sizeof(float));
    off_ml = add(n * sizeof(float2));
  };
  tc(p.tc_p, false, 1, rows_p, p.rps_p, p.workers_p, p.off_po, p.off_pml);
  tc(p.tc_s, prefix_len == 0, B, rows_s, p.rps_s, p.workers_s, p.off_so, p.off_sml);
  const int64_t all_rows = B * nkv * rows_s;
  p.merge_rows = all_rows <= kMergeShared * num_sms ? 1 : (rows_s + 15) / 16 * B * nkv < 8ll * num_sms ? 4 : 16;
  p.off_lse = add(scored ? sizeof(float) * B * L * nh : 0);
  const size_t key_items = static_cast<size_t>(B) * nkv * ((max_len + kTcKeys - 1) / kTcKeys);
  p.off_scores = add(scored && !p.tc_s ? sizeof(float) * B * nkv * rows_s * (static_cast<size_t>(max_len) + 3) / 4 * 4 : 0);
  p.off_w = add(scored && p.tc_s ? (num_sms + key_items) * kTcWeightParts * kTcKeys * sizeof(float) : 0);
  return p;
}

size_t cache_attn_bound(int B, int L, int nh, int nkv, int d, int max_len, int num_sms) {
  // every part at its largest: both kernels' pieces (which the number of keys does not change), the log sums,
  // the scores of one row tile, the slot weights' sums, and 4096 for the parts' alignment
  const size_t group = nh / nkv, rows_s = L * group, rows_p = B * rows_s;
  auto up = [](size_t n, size_t m) { return (n + m - 1) / m; };
  const size_t split = num_sms * kAttnBlocksPerSm * kAttnWarps +
                       nkv * (up(std::min<size_t>(rows_p, kAttnSplitRows), kAttnRowTile) +
                              B * up(std::min<size_t>(rows_s, kAttnSplitRows), kAttnRowTile));
  const size_t tc = 4 * num_sms + nkv * (up(rows_p, kTcRows) + B * up(rows_s, kTcRows));
  const size_t piece_rows = split * kAttnRowTile + tc * kTcRows;
  const size_t key_items = static_cast<size_t>(B) * nkv * up(max_len, kTcKeys);
  return piece_rows * (d * sizeof(float) + sizeof(float2)) + sizeof(float) * rows_p * nkv +
         sizeof(float) * B * nkv * std::min<size_t>(rows_s, kAttnRowTile) * (max_len + 3) +
         (num_sms + key_items) * kTcWeightParts * kTcKeys * sizeof(float) + 4096;
}

// Long caches of few heads: a cluster of four or two CTAs shares a head's slots, since one SM's passes take
// longer than what a cluster adds (barriers between the passes, ~4 us).  GPU time of one / two / four CTAs a
// head, 32 heads of 128, inputs out of cache; in place with one row to move, and cut to 2048 elsewhere:
//   10240 slots  17.3 / 21.3 / 19.9 us  and  40.2 / 42.3 / 41.3 us
//   12288        19.7 / 23.0 / 19.9          43.0 / 43.9 / 41.8
//   14336        22.7 / 24.5 / 21.2          46.0 / 45.4 / 42.2
//   16384        20.6 / 21.3 / 21.2          43.5 / 42.4 / 42.2
//   18432        23.2 / 23.1 / 22.7          46.4 / 44.0 / 43.8
//   24576        28.7 / 27.7 / 24.6          51.8 / 49.0 / 46.1
// (Eight CTAs of 16 heads of 65536: 57 where four take 38 and one 112.)  Only as many clusters as run at a
// time: SMs come in groups that clusters do not span, so that 33 of four fit 148 SMs, and 34 heads of 20480
// take 41 us in two rounds of them, 25 in clusters of two.
constexpr int kEvictFours = 14336, kEvictTwos = 18432;

int evict_ctas(int64_t heads, int max_len, const EvictClusters& c) {
  return max_len >= kEvictFours && heads <= c.fours ? 4 : max_len >= kEvictTwos && heads <= c.twos ? 2 : 1;
}

bool cache_attn_fits(const CacheAttnPlan& p, int B, int L, int nh, int nkv, int prefix_len, int max_len, bool scored) {
  // as many as a kernel's order has places when every length is max_len and nothing is hidden; in
  // doubles, which the products of the largest sizes cannot pass
  auto tiles = [](int len, int tile) { return std::ceil(static_cast<double>(len) / tile); };
  const double heads = static_cast<double>(B) * nkv, key_tiles = tiles(max_len, kTcKeys);
  const double split = static_cast<double>(nkv) * p.rt_p * tiles(prefix_len, kAttnTile) + heads * p.rt_s * tiles(max_len, kAttnTile);
  const double tc_p = static_cast<double>(nkv) * p.rps_p * (tiles(prefix_len, kTcKeys) + TcAttnArgs::kItemCost);
  const double tc_s = heads * p.rps_s * (key_tiles + TcAttnArgs::kItemCost);
  // the slot weights' tiles are whole tokens: a group of 65 heads has one of 128 rows to a token
  const double weights = scored && p.tc_s ? heads * key_tiles * (tiles(L, std::max(kTcKeys / (nh / nkv), 1)) + TcWeightArgs::kItemCost) : 0;
  return std::max(std::max(split, weights), std::max(tc_p, tc_s)) <= kMaxPlaces;
}

}  // namespace fm
