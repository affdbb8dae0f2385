// The host side of attention over caches (csrc/serve_plan.cu) for tests/test_serve.py: reads one
// command a line, answers one line.
#include <cstdio>
#include <cstring>

#include "fm_serve.cuh"

int main() {
  char what[32];
  while (std::scanf("%31s", what) == 1) {
    if (!std::strcmp(what, "fits")) {
      int B, L, nh, nkv, d, prefix, own, scored, max_len;
      if (std::scanf("%d %d %d %d %d %d %d %d %d", &B, &L, &nh, &nkv, &d, &prefix, &own, &scored, &max_len) != 9) return 1;
      const fm::CacheAttnPlan p = fm::cache_attn_plan(B, L, nh, nkv, d, prefix, own != 0, scored != 0, max_len, 148);
      std::printf("%d\n", fm::cache_attn_fits(p, B, L, nh, nkv, prefix, max_len, scored != 0));
    } else {
      return 1;
    }
  }
  return 0;
}
