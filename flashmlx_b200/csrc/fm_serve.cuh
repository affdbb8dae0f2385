// fm_serve.cuh -- arguments of the serving kernels (serve.cu).
#pragma once

#include <algorithm>
#include <vector>

#include "fm_internal.cuh"

#define FM_HD __host__ __device__ __forceinline__

namespace fm {

// The serving kernels are launched with programmatic stream serialization: a kernel may begin
// while the one before it ends.  It touches nothing that an earlier kernel wrote before
// pdl_wait(), which returns when the kernel before it is complete, and says with pdl_trigger()
// that the next one may begin -- after its own wait, so that whatever came before a call's
// first kernel is complete when its second one begins.
#ifdef __CUDACC__
FM_DEV void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
FM_DEV void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... P, class... A>
cudaError_t launch_pdl_cluster(void (*kernel)(P...), int ctas, dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
  c.attrs = attr;
  c.numAttrs = ctas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

template <class... P, class... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
  return launch_pdl_cluster(kernel, 1, grid, block, smem, st, args...);
}
#endif

constexpr int kRopeMaxDim = 256;  // largest head size of the rotary kernels

struct RopeBase {
  const uint16_t* q;        // [T, q_ld]: nq heads of d
  uint16_t* q_out;          // [T, qo_ld]
  int64_t q_ld, qo_ld;
  const uint16_t* k;        // append: [T, kv_ld]: nkv heads of d, rotated into cache_k
  const uint16_t* v;        // append: copied into cache_v
  int64_t kv_ld;
  uint16_t* cache_k;        // [B, nkv, max_len, d]
  uint16_t* cache_v;
  const int32_t* positions; // [T]
  const int32_t* slots;     // [T] cache slot of token t of sequence t / L; < 0: not written
  int64_t T;
  int nq, nkv, d, rotary, L, max_len, traditional;
  int tpb;                  // tokens of a CTA
  float factor;             // on cos and sin
  uint32_t* err;
};

// with the full turns per position of each pair (the kernel's argument: half the heads' bytes where
// they fit, since the launch copies it)
template <int PAIRS>
struct RopeSet : RopeBase {
  double turns[PAIRS];
};
using RopeArgs = RopeSet<kRopeMaxDim / 2>;

// Attention over caches is split over keys.  A source of keys -- the shared prefix, or the
// sequences' own caches -- is read by one of two kernels:
//
//   attn_split_kernel (serve.cu), a worker a warp, for few query rows per key: items of 16 query
//     rows, tiles of 16 keys, mma.sync.  Bound by HBM.
//   attn_tc_kernel (attn_tc.cu), a worker a CTA, for many: items of 256 query rows (of the heads
//     that share a kv head, neighbouring tokens together), tiles of 128 keys, tcgen05.
//
// The kernels count these places in 32 bits (and a worker's range may reach past the last), so the
// host refuses calls that could have more than kMaxPlaces in one kernel (cache_attn_fits).
// Either way the tiles of all items, in order, are cut into one contiguous range per worker, so
// ragged lengths balance.  A worker's piece of an item leaves an unnormalised fp32 output,
// its maximum (log2 units) and its sum in slot worker + item -- both only grow along the
// order, so no two pieces share a slot -- and attn_merge_kernel joins an output row's pieces.
// (Where whole items go to the output at once, a worker leaves at most two pieces: slots
// 2 worker for the item that it goes on with, 2 worker + 1 for the one that it begins.)
constexpr double kMaxPlaces = 1 << 30;
constexpr int kAttnTile = 16;        // keys of a tile
constexpr int kAttnRowTile = 16;     // query rows of an item
constexpr int kAttnSplitRows = 64;   // up to so many query rows to a key the split kernel reads it
constexpr int kAttnMinTiles = 4;     // least tiles of a worker's range
constexpr int kAttnWarps = 4;        // workers of a CTA
constexpr int kAttnBlocksPerSm = 2;
constexpr int kAttnStages = 3;       // ring of K / V tiles of a worker
constexpr int attn_split_smem(int d) { return kAttnWarps * kAttnStages * 2 * kAttnTile * d * 2; }

constexpr int kTcKeys = 128;         // keys of a tile, rows of a TMEM tile
constexpr int kTcRows = 256;         // query rows of an item
constexpr int kTcWeightParts = 4;    // sums of a piece of slot weights

struct CacheAttnArgs {
  const uint16_t* q;        // [B * L, q_ld]: nh heads of d
  int64_t q_ld;
  const uint16_t* pk;       // [nkv, p_head / d, d] shared prefix
  const uint16_t* pv;
  int64_t p_head;           // elements from one prefix head to the next
  const uint16_t* ck;       // [B, nkv, max_len, d] the sequences' own caches
  const uint16_t* cv;
  const int32_t* lens;      // [B] or null: no own caches
  uint16_t* out;            // [B * L, nh * d]
  float* acc;               // [B, nkv, max_len] or null
  int B, L, nh, nkv, group, max_len;
  int split_prefix;         // prefix rows the split kernel reads (0: none, or the other kernel's)
  int split_own;            // 1: it reads the own caches
  int after_tc;             // attn_tc_kernel was launched before it: nothing of that is needed here
  float scale_log2;         // softmax scale * log2(e)
  int merge_rows;           // rows of a merge block: 1, 4 or 16
  int rt_p, rt_s;           // row tiles of the prefix items / of a sequence's items, per kv head
  int workers;
  float* part_o;            // [slots][16][d]
  float2* part_ml;          // [slots][16] (maximum in log2 units, sum)
  float* lse2;              // [B, nkv, L * group] or null
  float* scores;            // split, scored: [B, nkv, L * group][score_ld] scores in log2 units (-inf: hidden)
  int64_t score_ld;         // max_len rounded up to 4
  uint32_t* err;
};

// n / d for 0 <= n < 2^31 by a multiplication: with 2^s >= d and m = ceil(2^(31 + s) / d),
// m d - 2^(31 + s) < d <= 2^s, so n m / 2^(31 + s) passes n / d by less than 1 / d.
struct Divisor {
  uint32_t m, s;

  static Divisor of(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    return {static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d), 31 + s};
  }
  FM_HD int divide(int n) const { return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(n)) * m >> s); }
};

// One source of keys for attn_tc_kernel: nseq sequences of L query tokens.
struct TcAttnArgs {
  const uint16_t* q;        // [nseq * L, q_ld]
  int64_t q_ld;
  const uint16_t* v;        // [nseq, nkv, head_rows, d], as its map
  const int32_t* lens;      // [nseq], or null: const_len keys each
  int nseq, L, nh, nkv, group, max_len, const_len;
  int causal;               // token l sees the keys j <= len - L + l; 0: all
  int head_rows;            // rows of K / V from one (sequence, kv head) to the next
  int rps;                  // items per (sequence, kv head)
  Divisor by_rps, by_group;
  int workers;              // 0: this source is not read here
  int direct;               // the only source: an item that one worker has whole goes to out
  float scale_log2;         // >= 0
  uint32_t q_sign;          // 0x80008000: q is negated (a negative scale)
  float* part_o;            // [slots][256][d]
  float2* part_ml;
  uint16_t* out;
  float* lse2;
  uint32_t* err;

  static constexpr int kItemCost = 4;  // what an item costs beside its tiles, in tiles
  FM_HD int items() const { return nseq * rps; }
  // tiles of item flat = b * rps + rp: up to the last key that its last token sees
  FM_HD int tiles(int flat) const;
};

// The slot weights by slot_weight_tc_kernel (attn_tc.cu): an item is a kv head's 128 keys, its
// tiles the query rows that see any of them, tile_tokens whole tokens (at most 128 rows) at a
// time.
struct TcWeightArgs {
  const uint16_t* q;        // [B * L, q_ld]
  int64_t q_ld;
  const int32_t* lens;
  const float* lse2;        // [B, nkv, L * group]
  float* acc;               // [B, nkv, max_len]
  float* part;              // [workers + items][4][128] sums of every fourth tile of a piece
  int B, L, nh, nkv, group, max_len;
  int key_tiles;            // of max_len
  int tile_tokens;          // 128 / group
  int workers;
  float scale_log2;
  uint32_t* err;

  static constexpr int kItemCost = 2;
  FM_HD int items() const { return B * key_tiles; }
  FM_HD int first_tile(int key0, int len) const;  // of the rows that see key0
  FM_HD int tiles(int flat) const;
};

FM_HD int tc_len(const TcAttnArgs& a, int b) {
  const int n = a.lens ? a.lens[b] : a.const_len;
  return n < 0 || n > a.max_len ? 0 : n;  // reported by the merge
}

// the last key that every row of item `flat` sees, -1: none
FM_HD int tc_seen_by_all(const TcAttnArgs& a, int flat, int len) {
  return a.causal ? max(len - a.L + a.by_group.divide((flat - a.by_rps.divide(flat) * a.rps) * kTcRows), -1) : len - 1;
}

#ifdef __CUDACC__
// a bf16 pair with infinities and NaN (an exponent of ones) as zeros
FM_DEV uint32_t finite_or_zero(uint32_t w) {
  const uint32_t m = ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  return w & ~((m >> 15) * 0xffffu);
}

// those infinities and NaN of a bf16 pair added to a pair of fp32 sums
FM_DEV void add_not_finite(uint32_t w, float& lo, float& hi) {
  const uint32_t bad = w & ~finite_or_zero(w);
  if (bad & 0x7f80u) lo += __uint_as_float(bad << 16);
  if (bad & 0x7f800000u) hi += __uint_as_float(bad & 0xffff0000u);
}
#endif

FM_HD int TcAttnArgs::tiles(int flat) const {
  const int b = by_rps.divide(flat), rp = flat - b * rps;
  const int len = tc_len(*this, b);
  int seen = len;
  if (causal) seen = len - L + min(by_group.divide(rp * kTcRows + kTcRows - 1), L - 1) + 1;
  return seen <= 0 ? 0 : (seen + kTcKeys - 1) / kTcKeys;
}

FM_HD int TcWeightArgs::first_tile(int key0, int len) const {
  return max(key0 - (len - L), 0) / tile_tokens;  // token key0 - (len - L) is the first that sees key0
}

FM_HD int TcWeightArgs::tiles(int flat) const {
  const int b = flat / key_tiles, key0 = (flat - b * key_tiles) * kTcKeys;
  const int len = lens[b];
  if (len < 0 || len > max_len || key0 >= len) return 0;
  return (L + tile_tokens - 1) / tile_tokens - first_tile(key0, len);
}

// An item's start and end cost a worker about as much as kItemCost tiles, so the order has that
// many empty places before each item's tiles and ranges are cut by places.
template <class A>
FM_HD int tc_item_places(const A& a, int flat) {
  const int n = a.tiles(flat);
  return n ? n + A::kItemCost : 0;
}

// places of one kv head of items [0, n), summed by the whole warp (on the host, for tests of the cut, by
// one thread)
template <class A>
FM_HD int tc_places_before(const A& a, int n) {
  int s = 0;
#ifdef __CUDA_ARCH__
  for (int i = threadIdx.x & 31; i < n; i += 32) s += tc_item_places(a, i);
  return __reduce_add_sync(0xffffffffu, s);
#else
  for (int i = 0; i < n; ++i) s += tc_item_places(a, i);
  return s;
#endif
}

template <class A>
FM_HD int tc_places_per_worker(const A& a, int total) {
  return max(1, (total + a.workers - 1) / a.workers);
}

// The item (flat, kvh) that place `place` falls into, and which of its places; false past the
// end.  Whole warp.
template <class A>
FM_HD bool tc_locate(const A& a, int place, int& flat, int& kvh, int& at) {
#ifndef __CUDA_ARCH__
  int rest = place;
  for (flat = 0; flat < a.items(); ++flat) {
    const int places = tc_item_places(a, flat);
    if (rest < places * a.nkv) {
      kvh = rest / places;
      at = rest - kvh * places;
      return true;
    }
    rest -= places * a.nkv;
  }
  return false;
#else
  const int lane = threadIdx.x & 31;
  int rest = place;
  for (int base = 0; base < a.items(); base += 32) {
    const int i = base + lane;
    const int mine = i < a.items() ? tc_item_places(a, i) * a.nkv : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, incl > rest);
    if (past) {
      const int f = __ffs(past) - 1;
      rest -= __shfl_sync(0xffffffffu, incl - mine, f);
      const int places = __shfl_sync(0xffffffffu, mine, f) / a.nkv;
      flat = base + f;
      kvh = rest / places;
      at = rest - kvh * places;
      return true;
    }
    rest -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
#endif
}

// A worker's piece in hand: tiles [tile, tile + cnt) of item (flat, kvh); cnt 0 at the end.
struct TcPiece {
  int flat, kvh, tile, tiles, cnt;
  int left;  // places of the worker's range from the item's first (or the range's) on
};

// the piece of the range that begins at place `at` of item (flat, kvh)
template <class A>
FM_HD void tc_cut(const A&, TcPiece& p, int at) {
  const int end = at + p.left;  // in the item's places
  p.tile = max(at - A::kItemCost, 0);
  p.cnt = max(min(end - A::kItemCost, p.tiles) - p.tile, 0);
  p.left -= p.tiles + A::kItemCost - at;
}

// the next item's piece; ends with cnt 0
template <class A>
FM_HD void tc_next(const A& a, TcPiece& p) {
  p.cnt = 0;
  while (p.left > 0 && p.cnt == 0) {
    if (++p.kvh == a.nkv) {
      p.kvh = 0;
      do {
        if (++p.flat >= a.items()) return;
        p.tiles = a.tiles(p.flat);
      } while (p.tiles == 0);
    }
    tc_cut(a, p, 0);
  }
}

template <class A>
FM_HD void tc_first(const A& a, int worker, int per, TcPiece& p) {  // whole warp
  int at;
  p.left = per;
  p.cnt = 0;
  if (!tc_locate(a, worker * per, p.flat, p.kvh, at)) return;
  p.tiles = a.tiles(p.flat);
  tc_cut(a, p, at);
  if (p.cnt == 0) tc_next(a, p);
}

// the slot of a worker's piece
FM_HD int64_t tc_slot(const TcAttnArgs& a, int worker, const TcPiece& p) {
  return a.direct ? 2 * static_cast<int64_t>(worker) + (p.tile == 0) : worker + static_cast<int64_t>(p.flat) * a.nkv + p.kvh;
}
FM_HD int64_t tc_slot(const TcWeightArgs& a, int worker, const TcPiece& p) {
  return worker + static_cast<int64_t>(p.flat) * a.nkv + p.kvh;
}

// Which kernel reads what, and the workspace.
struct CacheAttnPlan {
  bool tc_p = false, tc_s = false;  // the prefix / the own caches by attn_tc_kernel
  int rt_p = 0, rt_s = 0, rps_p = 0, rps_s = 0, merge_rows = 16;
  int workers = 0, workers_p = 0, workers_s = 0;
  size_t off_ml = 0, off_po = 0, off_pml = 0, off_so = 0, off_sml = 0, off_lse = 0, off_w = 0, off_scores = 0, bytes = 0;
};
CacheAttnPlan cache_attn_plan(int B, int L, int nh, int nkv, int d, int prefix_len, bool own, bool scored, int max_len,
                              int num_sms);

// At least what any call of up to B sequences of L tokens over such caches and any prefix needs.
size_t cache_attn_bound(int B, int L, int nh, int nkv, int d, int max_len, int num_sms);

// One handle's serving calls share a workspace, so a call on another stream than the calls before it
// waits for them.  Streams are followed, not calls: `busy` says that calls were made on the bound
// stream, `behind` holds the streams whose calls the bound one has yet to wait for.  What a capture
// records runs later, and its replays are the caller's to order: a stream waits only for streams of its
// own capture (whose branches a replay would run side by side), and one that is being captured stays
// `behind`.  Cuda has the two stream calls, so that tests can do without a device.
class StreamOrder {
 public:
  // the handle is bound to `now` instead of `before`
  void rebind(cudaStream_t before, cudaStream_t now) {
    if (before == now) return;
    if (busy_ && std::find(behind_.begin(), behind_.end(), before) == behind_.end()) behind_.push_back(before);
    busy_ = false;
  }

  // a call on the bound stream
  void mark() { busy_ = true; }

  // what stream `now`, the bound one, does next waits for the calls on the others
  template <class Cuda>
  cudaError_t join(cudaStream_t now, Cuda&& cuda) {
    if (behind_.empty()) return cudaSuccess;
    uint64_t mine = 0, its = 0;
    cudaError_t e = cuda.capture(now, &mine);
    for (size_t i = 0; i < behind_.size() && e == cudaSuccess;) {
      const cudaStream_t s = behind_[i];
      if (s != now) e = cuda.capture(s, &its);
      if (e == cudaSuccess && s != now && its == mine) e = cuda.wait(now, s);
      if (s == now || (e == cudaSuccess && its == 0 && mine == 0)) behind_.erase(behind_.begin() + i);
      else ++i;
    }
    return e;
  }

  // the bound stream was synchronized after join()
  void settle() { busy_ = false; }

 private:
  std::vector<cudaStream_t> behind_;
  bool busy_ = false;
};

// Whether every count of the plan's kernels fits their 32 bits (group at most kTcKeys when scored).
bool cache_attn_fits(const CacheAttnPlan& p, int B, int L, int nh, int nkv, int prefix_len, int max_len, bool scored);

struct EvictArgs {
  const uint16_t* cache_k;  // [B, nkv, max_len, d]
  const uint16_t* cache_v;
  const float* acc;         // [B, nkv, max_len]
  const int32_t* positions; // [B, nkv, max_len] or null: a slot's position is its index
  const int32_t* lens;      // [B]
  uint16_t* out_k;          // [B, nkv, out_max_len, d]; cache_k when in place
  uint16_t* out_v;
  float* out_acc;
  int32_t* out_positions;   // or null
  int32_t* out_lens;        // [B]
  int B, nkv, d, max_len, out_max_len, budget, sinks, recent;
  int in_place;
  int ctas;                 // of the cluster that selects in a head
  int words;                // 32-slot words of a CTA, at most
  int keys_in_smem;
  int fused;                // the select kernel makes the moves
  int32_t* list;            // [B * nkv][2][budget] destinations, sources
  int32_t* counts;          // [B * nkv][2] rows to move, slots that stay
  uint32_t* err;
};

cudaError_t launch_rope(RopeArgs& a, int num_sms, cudaStream_t st);
// How many clusters of two and of four CTAs of the selecting kernel run at a time.
struct EvictClusters {
  int twos = 0, fours = 0;
};
int evict_ctas(int64_t heads, int max_len, const EvictClusters& c);  // CTAs that share a head
cudaError_t serve_init(EvictClusters* c);
// p, s: the prefix / own caches by attn_tc_kernel where their workers are set, with its maps
struct TcMapsKV {
  CUtensorMap k, v;
  CUtensorMap q;  // the slot weights' query tiles: [tokens][heads][d], box {64, group, tile_tokens}
};
cudaError_t launch_cache_attn(const CacheAttnArgs& a, const TcAttnArgs& p, const TcMapsKV& mp, const TcAttnArgs& s,
                              const TcMapsKV& ms, const TcWeightArgs& w, int d, cudaStream_t st);
cudaError_t attn_tc_init();
cudaError_t launch_attn_tc(const TcAttnArgs& a, int d, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t st);
cudaError_t launch_slot_weight_tc(const TcWeightArgs& a, int d, const CUtensorMap& k, const CUtensorMap& q, cudaStream_t st);
cudaError_t launch_evict(EvictArgs a, bool lens_apart, const EvictClusters& clusters, int num_sms, cudaStream_t st);

}  // namespace fm
