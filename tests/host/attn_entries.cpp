// Host check of how the forward's roles number the entries of an item (lucid_kernels_b200/csrc/attn_geometry.h): the entries
// that are one tile's own are its list in order, and every entry of a union is somebody's; the entries of a split list, dealt
// out in turns, are the two halves' tiles, every tile of the list once.
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "attn_geometry.h"

using namespace lucid;

static int check(const AttnShape& a, int len) {
  FwdItem it;
  for (int n = 0; fwd_item(a, false, n, it); ++n) {
    const PairTiles pt = pair_tiles(a, it, len);
    std::vector<int> owners(pt.n, 0);
    for (int k = 0; k < 2; ++k) {
      const KeyTiles own = pt.list(k);
      const OwnEntries e = own_entries(own, pt.lo, pt.sink);
      int at = 0;
      for (int u = 0; u < pt.n; ++u) {
        if (!e.has(u)) continue;
        if (at >= own.n || own.tile(at) != pt.tile(u)) return 1;
        if ((at == 0 && e.first) != (own.sink && own.tile(at) == 0 && at == 0)) return 2;
        ++owners[u];
        ++at;
      }
      if (at != own.n) return 3;
    }
    for (int v : owners)
      if (v == 0) return 4;
  }
  for (int n = 0; fwd_item(a, true, n, it); ++n) {
    const PairTiles pt = pair_tiles(a, it, len);
    const KeyTiles t = key_tiles(a, it.block(0), len);
    if (pt.n != t.n || pt.x.n != t.n) return 5;       // (an item's number of entries)
    for (int parts = 1; parts <= 8; parts *= 2) {
      std::vector<int> seen(a.nkb, 0);
      int entries = 0;
      for (int part = 0; part < parts; ++part) {
        const KeyTiles run = part_list(t, part, parts), x = half_list(run, 0), y = half_list(run, 1);
        int at[2] = {0, 0};
        for (int u = 0; u < run.n; ++u, ++entries) {
          const KeyTiles& half = u & 1 ? y : x;
          if (at[u & 1] >= half.n || split_entry(x, y, u) != half.tile(at[u & 1])) return 6;
          ++at[u & 1];
          const int j = split_entry(x, y, u);
          if (j < 0 || j >= a.nkb || seen[j]++) return 7;
        }
        if (at[0] != x.n || at[1] != y.n) return 8;
      }
      if (entries != t.n) return 9;
      for (int e = 0; e < t.n; ++e)
        if (!seen[t.tile(e)]) return 10;
    }
  }
  return 0;
}

int main() {
  srand(2);
  auto r = [](int lo, int hi) { return lo + rand() % (hi - lo + 1); };
  const int edge[] = {1, 127, 128, 129, 256, 257, 511, 640, 1500};
  int n = 0;
  for (int round = 0; round < 6000; ++round) {
    AttnShape a;
    a.B = 1;
    a.Nk = r(0, 1) ? edge[r(0, 8)] : r(1, 4000);
    a.Nq = r(0, 1) ? a.Nk : r(1, a.Nk);
    a.Hkv = 1;
    a.G = r(1, 3);
    a.Hq = a.G;
    a.off = a.Nk - a.Nq;
    const int w = r(0, 4);
    a.W = w == 0 ? kNoWindow : w == 1 ? r(0, 2) : w == 2 ? 128 * r(1, 6) : r(1, 900);
    if (a.W >= a.Nk) a.W = kNoWindow;
    const int firsts[] = {0, 1, 4, 64, 128};
    a.S = a.W == kNoWindow ? 0 : firsts[r(0, 4)];
    a.nqb = (a.Nq + 127) / 128;
    a.nkb = (a.Nk + 127) / 128;
    const int len = r(0, 2) ? a.Nk : r(0, a.Nk), rc = check(a, len);
    if (rc) {
      printf("case %d: check %d Nq=%d Nk=%d G=%d W=%d S=%d len=%d\n", round, rc, a.Nq, a.Nk, a.G, a.W, a.S, len);
      return 1;
    }
    ++n;
  }
  printf("ok %d\n", n);
  return 0;
}
