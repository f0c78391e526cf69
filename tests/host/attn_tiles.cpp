// Host check of the windowed attention's tile lists (lucid_kernels_b200/csrc/attn_geometry.h): for random shapes,
// windows, visible first keys and lengths, the tiles that the forward, the dQ and the dK/dV kernels visit, with the masks
// they apply, cover every visible (query, key) pair of every head exactly once and no other pair; the two tiles of a
// forward item each see their own list, in order, through the union's `active`.
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "attn_geometry.h"

using namespace lucid;

static bool sees(const AttnShape& a, int i, int j, int len) {
  const long long p = (long long)i + a.off;
  return j <= p && (a.W >= kNoWindow || j > p - a.W || j < a.S) && j < len && p < len;
}

static int check(const AttnShape& a, const std::vector<int>& lens) {
  // by queries: dQ's lists
  for (int b = 0; b < a.B; ++b) {
    const int len = lens[b];
    std::vector<int> seen((size_t)a.Nq * a.Nk, 0);
    for (int blk = 0; blk < a.nqb; ++blk) {
      const KeyTiles t = key_tiles(a, blk, len);
      int before = -1;
      for (int u = 0; u < t.n; ++u) {
        const int j0 = t.tile(u) << 7;
        if (t.tile(u) <= before || j0 >= a.Nk || j0 < 0) return 1;
        before = t.tile(u);
        const bool masked = tile_masked(a, t, t.tile(u), len);
        for (int i = blk * 128; i < blk * 128 + 128 && i < a.Nq && i + a.off < len; ++i) {
          const RowMask m = row_mask(a, i + a.off, j0, len);
          for (int e = 0; e < 128; ++e) {
            if (((m.word(e & ~31) >> (e & 31)) & 1) != (m.sees(e) ? 1u : 0u)) return 16;
            if (masked && !m.sees(e)) continue;
            if (tile_narrow(a, t, t.tile(u)) && (!masked || e >= kNarrow)) return 17;
            if (j0 + e >= a.Nk) return 2;
            ++seen[(size_t)i * a.Nk + j0 + e];
          }
        }
      }
    }
    for (int i = 0; i < a.Nq; ++i) {
      int keys = 0;
      for (int j = 0; j < a.Nk; ++j) {
        if (seen[(size_t)i * a.Nk + j] != (sees(a, i, j, len) ? 1 : 0)) return 3;
        keys += seen[(size_t)i * a.Nk + j];
      }
      if (i + a.off < len && sees_one(a, i + a.off) != (keys == 1)) return 24;
      // a block that holds such a row shows it at one of its ends, and only in masked pairs of tiles
      const int p0 = (i & ~127) + a.off;
      if (i + a.off < len && keys == 1 && !sees_one(a, p0) && !sees_one(a, p0 + 127)) return 25;
    }
  }
  // forward items: every (b, head, block) once, its own list in order
  std::vector<int> tiles((size_t)a.B * a.Hq * a.nqb, 0);
  FwdItem it;
  int n = 0;
  for (; fwd_item(a, false, n, it); ++n) {
    if (it.b < 0 || it.b >= a.B || it.hk != it.h(0) / a.G || it.hk != it.h(1) / a.G) return 4;
    const PairTiles pt = pair_tiles(a, it, lens[it.b]);
    for (int k = 0; k < 2; ++k) {
      if (it.block(k) < a.nqb) ++tiles[((size_t)it.b * a.Hq + it.h(k)) * a.nqb + it.block(k)];
      const KeyTiles t = key_tiles(a, it.block(k), lens[it.b]), own = pt.list(k);
      if (own.n != t.n) return 5;
      int at = 0;
      for (int u = 0; u < pt.n; ++u) {
        if (!pt.active(t, u)) continue;
        if (at >= t.n || t.tile(at) != pt.tile(u)) return 6;
        ++at;
      }
      if (at != t.n) return 7;
    }
  }
  if (n != fwd_items(a, false)) return 8;
  // split items: every (b, head, block) once, the halves one after the other make the list, tile 0's first
  std::vector<int> halves((size_t)a.B * a.Hq * a.nqb, 0);
  for (n = 0; fwd_item(a, true, n, it); ++n) {
    if (it.hk != it.h(0) / a.G || it.h(0) != it.h(1) || it.block(0) != it.block(1)) return 19;
    ++halves[((size_t)it.b * a.Hq + it.h(0)) * a.nqb + it.block(0)];
    const KeyTiles t = key_tiles(a, it.block(0), lens[it.b]), x = half_list(t, 0), y = half_list(t, 1);
    if (x.n + y.n != t.n || x.n < y.n || x.n > y.n + 1) return 20;
    for (int e = 0; e < t.n; ++e)
      if ((e < x.n ? x.tile(e) : y.tile(e - x.n)) != t.tile(e)) return 21;
    // runs for a cluster's CTAs: one after the other they make the list too
    if (t.n > longest_list(a)) return 27;
    for (int parts = 1; parts <= 8; parts *= 2) {
      int at = 0;
      for (int k = 0; k < parts; ++k) {
        const KeyTiles run = part_list(t, k, parts);
        const KeyTiles r0 = half_list(run, 0), r1 = half_list(run, 1);
        if (run.n < 0 || run.n > t.n / parts + 1 || run.p_lo != t.p_lo || run.p_hi != t.p_hi || r0.n + r1.n != run.n) return 28;
        for (int e = 0; e < run.n; ++e, ++at)
          if (run.tile(e) != t.tile(at) || (e < r0.n ? r0.tile(e) : r1.tile(e - r0.n)) != t.tile(at)) return 29;
        if (run.sink && !(t.sink && at == run.n)) return 30;
      }
      if (at != t.n) return 31;
    }
  }
  if (n != fwd_items(a, true)) return 22;
  for (int v : halves)
    if (v != 1) return 23;
  for (int x : tiles)
    if (x != 1) return 9;
  // by keys: dK/dV's items
  const int chunks = sink_chunks(a);
  std::vector<std::vector<int>> got(a.B * a.Hkv, std::vector<int>((size_t)a.Nq * a.Nk, 0));
  KvItem kv;
  int m = 0;
  for (; kv_item(a, chunks, m, kv); ++m) {
    const int len = lens[kv.b];
    const QueryBlocks q = item_blocks(a, kv, len);
    if (kv.b < 0 || kv.b >= a.B || kv.hk < 0 || kv.hk >= a.Hkv || kv.tile >= a.nkb) return 10;
    for (int blk = q.first; blk <= q.last; ++blk) {
      if (blk < 0 || blk >= a.nqb) return 11;
      const int p0 = blk * 128 + a.off, j0 = kv.tile * 128;
      const bool masked = block_masked(a, j0, p0, len);
      if (!masked && (sees_one(a, p0) || sees_one(a, p0 + 127))) return 26;
      for (int j = j0; j < j0 + 128 && j < a.Nk; ++j) {
        const ColMask c = col_mask(a, j, p0, len);
        for (int e = 0; e < 128; ++e) {
          if (((c.word(e & ~31) >> (e & 31)) & 1) != (c.sees(e) ? 1u : 0u)) return 18;
          if (masked && !c.sees(e)) continue;
          if (blk * 128 + e >= a.Nq) return 12;
          if (kv.chunk >= 0 && j >= a.S) return 13;     // a chunk holds first keys only
          ++got[kv.b * a.Hkv + kv.hk][(size_t)(blk * 128 + e) * a.Nk + j];
        }
      }
    }
  }
  if (m != kv_items(a)) return 14;
  for (int b = 0; b < a.B; ++b)
    for (int h = 0; h < a.Hkv; ++h)
      for (int i = 0; i < a.Nq; ++i)
        for (int j = 0; j < a.Nk; ++j)
          if (got[b * a.Hkv + h][(size_t)i * a.Nk + j] != (sees(a, i, j, lens[b]) ? 1 : 0)) return 15;
  return 0;
}

int main() {
  srand(1);
  auto r = [](int lo, int hi) { return lo + rand() % (hi - lo + 1); };
  const int edge[] = {1, 2, 127, 128, 129, 255, 256, 257, 300, 511, 640};
  int n = 0;
  for (int round = 0; round < 1500; ++round) {
    AttnShape a;
    a.B = r(1, 2);
    a.Nk = r(0, 2) ? edge[r(0, 10)] : r(1, round % 20 ? 700 : 2600);
    a.Nq = r(0, 1) ? a.Nk : r(1, a.Nk);
    a.Hkv = r(1, 2);
    a.G = r(1, 4);
    a.Hq = a.Hkv * a.G;
    a.off = a.Nk - a.Nq;
    const int w = r(0, 5);
    a.W = w == 0 ? kNoWindow : w == 1 ? r(0, 2) : w == 2 ? 128 * r(1, 3) : r(1, 400);
    if (a.W >= a.Nk) a.W = kNoWindow;
    const int firsts[] = {0, 0, 1, 4, 5, 64, 127, 128};
    a.S = a.W == kNoWindow ? 0 : firsts[r(0, 7)];
    a.nqb = (a.Nq + 127) / 128;
    a.nkb = (a.Nk + 127) / 128;
    std::vector<int> lens;
    for (int b = 0; b < a.B; ++b) lens.push_back(r(0, 1) ? a.Nk : r(0, a.Nk));
    const int rc = check(a, lens);
    if (rc) {
      printf("case %d: check %d B=%d Nq=%d Nk=%d Hkv=%d G=%d W=%d S=%d len=%d\n", round, rc, a.B, a.Nq, a.Nk, a.Hkv, a.G, a.W,
             a.S, lens[0]);
      return 1;
    }
    ++n;
  }
  printf("ok %d\n", n);
  return 0;
}
