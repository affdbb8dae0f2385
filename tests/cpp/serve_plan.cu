// The host side of attention over caches (csrc/serve_plan.cu) for tests/test_serve.py: reads one
// command a line, answers one line.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <set>

#include "fm_serve.cuh"

namespace {

cudaStream_t stream(int i) { return reinterpret_cast<cudaStream_t>(static_cast<intptr_t>(i)); }

// the calls that StreamOrder makes, written down
struct Calls {
  std::set<cudaStream_t> captured;
  int fails = 0;  // the n-th next wait fails
  cudaError_t capturing(cudaStream_t s, bool* yes) {
    *yes = captured.count(s) > 0;
    return cudaSuccess;
  }
  cudaError_t wait(cudaStream_t now, cudaStream_t s) {
    if (fails && --fails == 0) return cudaErrorInvalidResourceHandle;
    std::printf(" %d<%d", static_cast<int>(reinterpret_cast<intptr_t>(now)), static_cast<int>(reinterpret_cast<intptr_t>(s)));
    return cudaSuccess;
  }
};

// order <n>, n steps: b<stream> bind, c call (join, mark), s sync (join, settle), +<stream> / -<stream> a
// capture begins / ends, f<n> the n-th next wait fails; answers the waits of the calls
bool order() {
  int n, now = 0;
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
      cuda.captured.insert(stream(to));
    } else if (what[0] == '-') {
      cuda.captured.erase(stream(to));
    } else {
      cuda.fails = to;
    }
  }
  std::printf("\n");
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
    } else if (!std::strcmp(what, "order")) {
      if (!order()) return 1;
    } else {
      return 1;
    }
  }
  return 0;
}
