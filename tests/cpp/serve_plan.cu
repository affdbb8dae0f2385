// The host side of attention over caches (csrc/serve_plan.cu) for tests/test_serve.py: reads one
// command a line, answers one line.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <map>
#include <random>
#include <set>
#include <utility>
#include <vector>

#include "fm_serve.cuh"

namespace {

cudaStream_t stream(int i) { return reinterpret_cast<cudaStream_t>(static_cast<intptr_t>(i)); }

// the calls that StreamOrder makes, written down
struct Calls {
  std::map<cudaStream_t, uint64_t> captured;
  int fails = 0;  // the n-th next wait fails
  cudaError_t capture(cudaStream_t s, uint64_t* id) {
    *id = captured.count(s) ? captured[s] : 0;
    return cudaSuccess;
  }
  cudaError_t wait(cudaStream_t now, cudaStream_t s) {
    if (fails && --fails == 0) return cudaErrorInvalidResourceHandle;
    std::printf(" %d<%d", static_cast<int>(reinterpret_cast<intptr_t>(now)), static_cast<int>(reinterpret_cast<intptr_t>(s)));
    return cudaSuccess;
  }
};

// order <n>, n steps: b<stream> bind, c call (join, mark), s sync (join, settle), +<stream> a capture begins,
// *<stream> the stream joins the last one, -<stream> it is captured no longer, f<n> the n-th next wait
// fails; answers the waits of the calls
bool order() {
  int n, now = 0, captures = 0;
  fm::StreamOrder o;
  Calls cuda;
  if (std::scanf("%d", &n) != 1) return false;
  for (int i = 0; i < n; ++i) {
    char what[16];
    if (std::scanf("%15s", what) != 1) return false;
    int to = 0;
    std::sscanf(what + 1, "%d", &to);
    if (what[0] == 'b') {
      o.rebind(stream(now), stream(to));
      now = to;
    } else if (what[0] == 'c' || what[0] == 's') {
      std::printf(" |");
      if (o.join(stream(now), cuda) != cudaSuccess) std::printf(" error");
      else if (what[0] == 'c') o.mark();
      else o.settle();
    } else if (what[0] == '+') {
      cuda.captured[stream(to)] = ++captures;
    } else if (what[0] == '*') {
      cuda.captured[stream(to)] = captures;
    } else if (what[0] == '-') {
      cuda.captured.erase(stream(to));
    } else {
      cuda.fails = to;
    }
  }
  std::printf("\n");
  return true;
}

// A piece as a worker of the cut makes it.
struct Made {
  int worker, tile, cnt;
  int64_t slot;
};

#define EXPECT(ok)                                                    \
  if (!(ok)) {                                                        \
    std::printf("line %d: %s (case %d)\n", __LINE__, #ok, the_case); \
    return false;                                                     \
  }
int the_case = 0;

// The workers' pieces of a tcgen05 kernel's order: every tile once, the pieces of an item with the workers
// and in the slots in which the kernels that join them look, every slot once and within `slots`.
// direct: an item that one worker has whole takes no slot.
template <class A>
bool cut(const A& a, int64_t slots, bool direct) {
  const int per = fm::tc_places_per_worker(a, fm::tc_places_before(a, a.items()) * a.nkv);
  std::map<std::pair<int, int>, std::vector<Made>> items;
  std::set<int64_t> used;
  for (int w = 0; w < a.workers; ++w) {
    fm::TcPiece p;
    for (fm::tc_first(a, w, per, p); p.cnt > 0; fm::tc_next(a, p)) {
      EXPECT(p.flat >= 0 && p.flat < a.items() && p.kvh >= 0 && p.kvh < a.nkv && p.tiles == a.tiles(p.flat))
      EXPECT(p.tile >= 0 && p.tile + p.cnt <= p.tiles)
      const int64_t slot = fm::tc_slot(a, w, p);
      if (!direct || p.cnt < p.tiles) {
        EXPECT(slot >= 0 && slot < slots)
        EXPECT(used.insert(slot).second)
      }
      items[{p.flat, p.kvh}].push_back({w, p.tile, p.cnt, slot});
    }
  }
  std::map<std::pair<int, int>, int> joined;  // by the blocks of attn_merge_cut_kernel
  for (int w = 0; direct && w < a.workers - 1; ++w) {
    int flat, kvh, at;
    const int place = (w + 1) * per;
    if (!fm::tc_locate(a, place, flat, kvh, at)) continue;
    const int first = place - at + A::kItemCost;
    if (first >= place || first / per != w) continue;
    ++joined[{flat, kvh}];
  }
  for (int flat = 0; flat < a.items(); ++flat) {
    const int tiles = a.tiles(flat);
    for (int kvh = 0; kvh < a.nkv; ++kvh) {
      const auto& made = items[{flat, kvh}];
      if (tiles == 0) {
        EXPECT(made.empty())
        continue;
      }
      const int first = fm::tc_places_before(a, flat) * a.nkv + kvh * (tiles + A::kItemCost) + A::kItemCost;
      const int w0 = first / per, w1 = (first + tiles - 1) / per;
      EXPECT(static_cast<int>(made.size()) == w1 - w0 + 1)
      int next = 0;
      for (int i = 0; i <= w1 - w0; ++i) {
        EXPECT(made[i].worker == w0 + i && made[i].tile == next)
        next += made[i].cnt;
        const int64_t want = !direct ? w0 + i + static_cast<int64_t>(flat) * a.nkv + kvh : 2 * static_cast<int64_t>(w0 + i) + (i == 0);
        EXPECT(made[i].slot == want)
      }
      EXPECT(next == tiles)
      if (direct) EXPECT((joined[{flat, kvh}]) == (w1 > w0 ? 1 : 0))
    }
  }
  return true;
}

// The split kernel's: items of tiles in order, cut into ranges of `per`; a piece's slot is the worker's
// number plus the item's.
bool cut_split(const fm::CacheAttnPlan& p, const std::vector<int>& lens, int nkv, int prefix, int64_t slots) {
  std::vector<std::pair<int64_t, int>> items;  // number, tiles
  for (int i = 0; i < nkv * p.rt_p; ++i) items.push_back({i, (prefix + fm::kAttnTile - 1) / fm::kAttnTile});
  for (size_t b = 0; b < lens.size(); ++b)
    for (int i = 0; i < nkv * p.rt_s; ++i)
      items.push_back({nkv * p.rt_p + static_cast<int64_t>(b) * nkv * p.rt_s + i, (lens[b] + fm::kAttnTile - 1) / fm::kAttnTile});
  int64_t total = 0, first = 0;
  for (const auto& i : items) total += i.second;
  const int64_t per = std::max<int64_t>(fm::kAttnMinTiles, (total + p.workers - 1) / p.workers);
  std::set<int64_t> used;
  for (const auto& i : items) {
    if (i.second == 0) continue;
    for (int64_t w = first / per; w <= (first + i.second - 1) / per; ++w) {
      EXPECT(w < p.workers && w + i.first < slots && used.insert(w + i.first).second)
    }
    first += i.second;
  }
  return true;
}

// cut <seed> <cases>: random calls, their lengths ragged, some 0 or out of range
bool cuts() {
  int seed, cases;
  if (std::scanf("%d %d", &seed, &cases) != 2) return false;
  std::mt19937 rng(seed);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  auto logpick = [&](int hi) { return std::min(hi, pick(0, 1) ? pick(1, hi) : pick(1, 1 << pick(0, 10))); };
  for (the_case = 0; the_case < cases; ++the_case) {
    const int nkv = pick(1, 5), group = pick(0, 3) ? pick(1, 9) : pick(10, 128), nh = nkv * group, d = pick(0, 1) ? 64 : 128;
    const int B = logpick(40), L = pick(0, 2) ? logpick(700) : 1, max_len = logpick(5000), sms = pick(0, 2) ? pick(2, 200) : 148;
    const bool scored = pick(0, 1);
    const int prefix = scored || pick(0, 2) == 0 ? 0 : logpick(20000);
    std::vector<int32_t> lens(B);
    std::vector<int> held(B);
    const int kind = pick(0, 3);
    for (int b = 0; b < B; ++b) {
      lens[b] = kind == 0 ? max_len : kind == 1 ? pick(0, max_len) : pick(0, 4) ? logpick(max_len) : pick(-2, 0) + (pick(0, 1) ? max_len + 2 : 0);
      held[b] = lens[b] < 0 || lens[b] > max_len ? 0 : lens[b];
    }
    const fm::CacheAttnPlan p = fm::cache_attn_plan(B, L, nh, nkv, d, prefix, true, scored, max_len, sms);
    const size_t piece = (static_cast<size_t>(d) * 4 + 8), rows = fm::kTcRows;
    if (p.workers) {
      const int64_t slots = p.workers + static_cast<int64_t>(nkv) * (p.rt_p + static_cast<int64_t>(B) * p.rt_s);
      EXPECT(p.bytes >= slots * fm::kAttnRowTile * piece)
      if (!cut_split(p, held, nkv, prefix, slots)) return false;
    }
    for (int i = 0; i < 2; ++i) {
      if (!(i ? p.tc_s : p.tc_p)) continue;
      fm::TcAttnArgs a = {};
      a.lens = i ? lens.data() : nullptr;
      a.nseq = i ? B : 1;
      a.L = i ? L : B * L;
      a.nh = nh;
      a.nkv = nkv;
      a.group = group;
      a.max_len = i ? max_len : prefix;
      a.const_len = prefix;
      a.causal = i;
      a.rps = i ? p.rps_s : p.rps_p;
      a.by_rps = fm::Divisor::of(a.rps);
      a.by_group = fm::Divisor::of(group);
      a.workers = i ? p.workers_s : p.workers_p;
      a.direct = i && prefix == 0;
      const int64_t slots = a.direct ? 2 * a.workers : a.workers + static_cast<int64_t>(a.nseq) * a.rps * nkv;
      EXPECT((i ? p.off_so + slots * rows * d * 4 <= p.off_sml : p.off_po + slots * rows * d * 4 <= p.off_pml))
      EXPECT(p.bytes >= (i ? p.off_sml : p.off_pml) + slots * rows * 8)
      if (!cut(a, slots, a.direct)) return false;
    }
    if (scored && p.tc_s) {
      fm::TcWeightArgs w = {};
      w.lens = lens.data();
      w.B = B;
      w.L = L;
      w.nh = nh;
      w.nkv = nkv;
      w.group = group;
      w.max_len = max_len;
      w.key_tiles = (max_len + fm::kTcKeys - 1) / fm::kTcKeys;
      w.workers = sms;
      w.tile_tokens = fm::kTcKeys / group;
      const int64_t slots = sms + static_cast<int64_t>(B) * nkv * w.key_tiles;
      EXPECT(p.bytes >= p.off_w + slots * fm::kTcWeightParts * fm::kTcKeys * 4)
      if (!cut(w, slots, false)) return false;
    }
    EXPECT(fm::cache_attn_bound(B, L, nh, nkv, d, max_len, sms) >= p.bytes)
  }
  std::printf("ok\n");
  return true;
}

// divide <cases>: Divisor against the division, at its borders too
bool divides() {
  int cases;
  if (std::scanf("%d", &cases) != 1) return false;
  std::mt19937 rng(cases);
  for (int i = 0; i < cases; ++i) {
    const int d = 1 + static_cast<int>((rng() & 0x7fffffff) >> (rng() % 31));
    if (d < 1) continue;
    const fm::Divisor by = fm::Divisor::of(d);
    const int top = 0x7fffffff / d * d;
    for (const int64_t n : {int64_t(0), int64_t(d) - 1, int64_t(d), int64_t(top) - 1, int64_t(top), int64_t(0x7fffffff),
                            int64_t(rng() & 0x7fffffff)})
      if (n >= 0 && n <= 0x7fffffff && by.divide(static_cast<int>(n)) != static_cast<int>(n) / d) {
        std::printf("%lld / %d\n", static_cast<long long>(n), d);
        return false;
      }
  }
  std::printf("ok\n");
  return true;
}

}  // namespace

int main() {
  char what[32];
  while (std::scanf("%31s", what) == 1) {
    if (!std::strcmp(what, "fits")) {
      int B, L, nh, nkv, d, prefix, own, scored, max_len;
      if (std::scanf("%d %d %d %d %d %d %d %d %d", &B, &L, &nh, &nkv, &d, &prefix, &own, &scored, &max_len) != 9) return 1;
      const fm::CacheAttnPlan p = fm::cache_attn_plan(B, L, nh, nkv, d, prefix, own != 0, scored != 0, max_len, 148);
      std::printf("%d\n", fm::cache_attn_fits(p, B, L, nh, nkv, prefix, max_len, scored != 0));
    } else if (!std::strcmp(what, "evict")) {
      int heads, max_len;
      fm::EvictClusters c;
      if (std::scanf("%d %d %d %d", &heads, &max_len, &c.twos, &c.fours) != 4) return 1;
      std::printf("%d\n", fm::evict_ctas(heads, max_len, c));
    } else if (!std::strcmp(what, "order")) {
      if (!order()) return 1;
    } else if (!std::strcmp(what, "cut")) {
      if (!cuts()) return 1;
    } else if (!std::strcmp(what, "divide")) {
      if (!divides()) return 1;
    } else {
      return 1;
    }
  }
  return 0;
}
