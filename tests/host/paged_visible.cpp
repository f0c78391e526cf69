// Host check of what a single-token query sees of a paged cache (cache_visible in lucid_kernels_b200/csrc/attn_geometry.h):
// every position of the cache that the rule shows, once and in order, and no other, for lengths up to and far beyond the cache.
#include <cstdio>
#include <cstdlib>
#include "attn_geometry.h"

using namespace lucid;

int main() {
  srand(1);
  auto r = [](int lo, int hi) { return lo + rand() % (hi - lo + 1); };
  int n = 0;
  for (int round = 0; round < 20000; ++round) {
    const int cap = r(1, 300);
    const int windows[] = {0, 1, r(2, 40), r(1, 700), kNoWindow}, firsts[] = {0, 1, r(2, 12), r(0, 600), 1 << 30};
    const int lens[] = {0, -5, r(1, cap), cap, cap + 1, cap + r(0, 50), r(1, 1200), 0x7fffffff, 0x7fffffff - r(0, 1000)};
    const int W = windows[r(0, 4)], S = firsts[r(0, 4)], len = lens[r(0, 8)];
    const Visible v = cache_visible(W, S, len, cap);
    int at = 0;
    for (int p = 0; p < cap; ++p) {
      const bool sees = p < len && (W >= kNoWindow || (long long)p > (long long)len - 1 - W || p < S);
      if (!sees) continue;
      if (at >= v.n || v.pos(at) != p) {
        printf("cap %d W %d S %d len %d: position %d is missing\n", cap, W, S, len, p);
        return 1;
      }
      ++at;
    }
    if (at != v.n) {
      printf("cap %d W %d S %d len %d: %d positions, %d expected\n", cap, W, S, len, v.n, at);
      return 1;
    }
    ++n;
  }
  printf("ok %d\n", n);
  return 0;
}
