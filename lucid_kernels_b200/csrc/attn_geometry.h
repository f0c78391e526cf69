// Which tiles the windowed attention kernels visit, and in which order.  Plain integer arithmetic, usable from host
// code as well: every role of a kernel derives the same lists from it, so it is checked on the CPU.
//
// Query i of Nq sits at position p = i + off with off = Nk - Nq >= 0 (the queries are the last Nq positions).  In a
// sequence of n valid positions it sees key j when  j <= p,  (j > p - W  or  j < S),  j < n  and  p < n.
#pragma once
#include "schedule.h"

namespace lucid {

constexpr int kNoWindow = 1 << 30;   // W of full causality
constexpr int kMaxSinks = 128;       // S <= 128: visible first keys all lie in key tile 0

LUCID_HD int imax(int a, int b) { return a > b ? a : b; }

struct AttnShape {
  int B, Nq, Nk, Hq, Hkv;
  int G;      // query heads per key head
  int off;    // Nk - Nq
  int W, S;
  int nqb, nkb;   // 128-row blocks of queries and keys
};

// Rows of a block in `rest` (what the rounding of the result took off): whole blocks, but no more rows than there are queries -
// a few queries of many heads would otherwise keep up to 128 times what they need.
LUCID_HD int rest_rows(const AttnShape& a) { return imin(a.Nq, 128); }

// Key tiles of one block of 128 queries: an optional first tile 0 that holds only visible first keys, then lo .. hi.
struct KeyTiles {
  int n;         // how many, 0 = no query of the block sees anything
  int sink;      // 1: tile 0 comes first although the window does not reach it
  int lo;
  int p_lo, p_hi;   // positions of the block's first and last valid query
  LUCID_HD int tile(int u) const { return u < sink ? 0 : lo + u - sink; }
};

LUCID_HD KeyTiles key_tiles(const AttnShape& a, int block, int len) {
  KeyTiles t;
  const int i0 = block * 128;
  const int last = imin(imin(i0 + 127, a.Nq - 1), len - 1 - a.off);   // last valid query of the block
  t.p_lo = i0 + a.off;
  t.p_hi = last + a.off;
  t.n = 0;
  t.sink = 0;
  t.lo = 0;
  if (last < i0) return t;
  const int lo_key = a.W >= kNoWindow ? 0 : imax(0, t.p_lo - a.W + 1);
  const bool near = a.W > 0;                        // W == 0: no key of the window, only first keys
  t.lo = lo_key >> 7;
  const int hi = t.p_hi >> 7;
  t.sink = (a.S > 0 && (!near || t.lo > 0)) ? 1 : 0;
  t.n = t.sink + (near ? hi - t.lo + 1 : 0);
  return t;
}

// Does any (query, key) pair of the tile have to be masked?
LUCID_HD bool tile_masked(const AttnShape& a, const KeyTiles& t, int tile, int len) {
  const int j0 = tile << 7;
  return j0 + 127 > t.p_lo || (a.W < kNoWindow && j0 <= t.p_hi - a.W) || j0 + 127 >= len;
}

// Does the query at position p see exactly one key?  Its weight is 1 whatever the scores are: no gradient reaches q or k.
LUCID_HD bool sees_one(const AttnShape& a, int p) {
  const int near = a.W >= kNoWindow ? p + 1 : imin(a.W, p + 1);
  const int first = a.W >= kNoWindow ? 0 : imin(a.S, p + 1 - near);
  return near + first == 1;
}

// A tile visited for its visible first keys alone, few enough for a product of kNarrow keys.
constexpr int kNarrow = 32;
LUCID_HD bool tile_narrow(const AttnShape& a, const KeyTiles& t, int tile) { return t.sink && tile == 0 && a.S <= kNarrow; }

// Columns of a key tile (first key j0) that the query at position p sees: e <= hi and (e >= lo or e < first).
struct RowMask {
  int hi, lo, first;
  LUCID_HD bool sees(int e) const { return e <= hi && (e >= lo || e < first); }
  // bit e: column base + e, e < 32
  LUCID_HD unsigned word(int base) const {
    return below(hi + 1 - base) & (~below(lo - base) | below(first - base));
  }
  LUCID_HD static unsigned below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }   // bits 0 .. n-1
};
LUCID_HD RowMask row_mask(const AttnShape& a, int p, int j0, int len) {
  return RowMask{imin(p, len - 1) - j0, p - a.W + 1 - j0, a.S - j0};
}

// Transposed: does any pair of key tile j0 and the 128 queries from position p0 on have to be masked, and which columns
// (queries) lo .. hi see key j.
LUCID_HD bool block_masked(const AttnShape& a, int j0, int p0, int len) {
  return p0 < j0 + 127 || p0 + 127 >= len || j0 + 127 >= len || (a.W < kNoWindow && p0 + 127 > j0 + a.W - 1);
}
struct ColMask {
  int lo, hi;
  LUCID_HD bool sees(int e) const { return e >= lo && e <= hi; }
  LUCID_HD unsigned word(int base) const { return RowMask::below(hi + 1 - base) & ~RowMask::below(lo - base); }
};
LUCID_HD ColMask col_mask(const AttnShape& a, int j, int p0, int len) {
  ColMask m;
  m.lo = j - p0;
  m.hi = len - 1 - p0;
  if (a.W < kNoWindow && j >= a.S) m.hi = imin(m.hi, j + a.W - 1 - p0);
  if (j >= len) m.hi = -1;
  return m;
}

// Forward work item: two tiles of 128 queries that read the same keys.  With an even number of query heads per key
// head they are two heads of one block of rows (same keys exactly), otherwise two neighbouring blocks of one head.
LUCID_HD bool pair_heads(const AttnShape& a) { return (a.G & 1) == 0; }
LUCID_HD int fwd_items(const AttnShape& a, bool split) {
  if (split) return a.B * a.Hq * a.nqb;
  return pair_heads(a) ? a.B * (a.Hq / 2) * a.nqb : a.B * a.Hq * ((a.nqb + 1) / 2);
}
// The item that CTA `cta` of `grid` takes in its round `r`: back and forth, so that the CTAs that got the longest items of
// one round get the shortest of the next (the items are sorted by length).
LUCID_HD int snake_item(int r, int cta, int grid) { return r * grid + ((r & 1) ? grid - 1 - cta : cta); }
struct FwdItem {
  int b, hk;
  int h0, h1, block0, block1;    // block >= nqb: no such tile
  LUCID_HD int h(int k) const { return k ? h1 : h0; }
  LUCID_HD int block(int k) const { return k ? block1 : block0; }
};
LUCID_HD bool fwd_item(const AttnShape& a, bool split, int idx, FwdItem& it) {
  if (idx >= fwd_items(a, split)) return false;
  // blocks from the last to the first (under full causality the last ones take longest), heads side by side
  if (split) {
    const int per = a.B * a.Hq, r = idx % per;
    it.b = r / a.Hq;
    it.h0 = it.h1 = r % a.Hq;
    it.block0 = it.block1 = a.nqb - 1 - idx / per;
  } else if (pair_heads(a)) {
    const int per = a.B * (a.Hq / 2);
    const int blk = a.nqb - 1 - idx / per, r = idx % per;
    it.b = r / (a.Hq / 2);
    it.h0 = 2 * (r % (a.Hq / 2));
    it.h1 = it.h0 + 1;
    it.block0 = it.block1 = blk;
  } else {
    const int per = a.B * a.Hq, nb = (a.nqb + 1) / 2;
    const int bp = nb - 1 - idx / per, r = idx % per;
    it.b = r / a.Hq;
    it.h0 = it.h1 = r % a.Hq;
    it.block0 = 2 * bp;
    it.block1 = 2 * bp + 1;
  }
  it.hk = it.h0 / a.G;
  return true;
}
// With fewer such pairs than SMs the item is ONE tile of queries, and its list is split: the first half goes to tile 0, the
// rest to tile 1, entries of the two in turn; their results are joined at the end.
LUCID_HD KeyTiles half_list(const KeyTiles& t, int k) {
  KeyTiles h = t;
  const int n0 = (t.n + 1) / 2;
  h.n = k ? t.n - n0 : n0;
  if (k) {
    h.sink = 0;
    h.lo = t.n > 0 ? t.tile(n0) : 0;
  } else if (h.n == 0) {
    h.sink = 0;
  }
  return h;
}
// And with fewer still the list is first dealt out in `parts` runs, one per CTA of a cluster.
LUCID_HD KeyTiles part_list(const KeyTiles& t, int k, int parts) {
  KeyTiles h = t;
  const int from = (int)((long long)t.n * k / parts), to = (int)((long long)t.n * (k + 1) / parts);
  h.n = to - from;
  if (h.n == 0 || from > 0) h.sink = 0;
  if (h.n > 0 && from > 0) h.lo = t.tile(from);
  return h;
}
// The most key tiles a block of queries visits.
LUCID_HD int longest_list(const AttnShape& a) {
  const int near = a.W >= kNoWindow ? a.nkb : imin(a.nkb, (a.W + 253) / 128 + 1);
  return near + (a.S > 0 ? 1 : 0);
}
// Entry u of such a run goes to tile u & 1, as the next of its half.
LUCID_HD int split_entry(const KeyTiles& half0, const KeyTiles& half1, int u) { return (u & 1 ? half1 : half0).tile(u >> 1); }

// The entries of a union of two lists that are one list's own: entry 0 for the visible first keys, and from .. to-1.
struct OwnEntries {
  int first, from, to;
  LUCID_HD bool has(int u) const { return (u == 0 && first) || (u >= from && u < to); }
};
LUCID_HD OwnEntries own_entries(const KeyTiles& own, int union_lo, int union_sink) {
  OwnEntries e;
  const int near = own.n - own.sink;
  e.first = own.n > 0 && own.sink;
  e.from = near > 0 ? own.lo - union_lo + union_sink : 0;
  e.to = e.from + (near > 0 ? near : 0);
  return e;
}

// The union of the two tiles' lists, in increasing order; `active` says which of the two visits an entry.
struct PairTiles {
  KeyTiles x, y;
  int n, sink, lo;
  LUCID_HD KeyTiles list(int k) const { return k ? y : x; }
  LUCID_HD int tile(int u) const { return u < sink ? 0 : lo + u - sink; }
  LUCID_HD bool active(const KeyTiles& t, int u) const { return own_entries(t, lo, sink).has(u); }
};
LUCID_HD PairTiles pair_tiles(const AttnShape& a, const FwdItem& it, int len) {
  PairTiles p;
  const KeyTiles x = p.x = key_tiles(a, it.block0, len);
  const KeyTiles y = p.y = key_tiles(a, it.block1, len);
  // runs of window tiles: both non-empty, or one of them (x comes first: its rows are the lower ones)
  const int nx = x.n - x.sink, ny = y.n - y.sink;
  int hi;
  if (nx > 0 && ny > 0) {
    p.lo = imin(x.lo, y.lo);
    hi = imax(x.lo + nx, y.lo + ny) - 1;
  } else if (nx > 0) {
    p.lo = x.lo;
    hi = x.lo + nx - 1;
  } else {
    p.lo = y.lo;
    hi = y.lo + ny - 1;
  }
  const bool any = nx > 0 || ny > 0;
  // one list's first tile 0 may be the other list's window tile 0
  p.sink = ((x.n > 0 && x.sink) || (y.n > 0 && y.sink)) && !(any && p.lo == 0) ? 1 : 0;
  p.n = p.sink + (any ? hi - p.lo + 1 : 0);
  return p;
}

// Query blocks whose rows may see a key of key tile `tile` through the window (first .. last; none: first > last).
struct QueryBlocks {
  int first, last;
};
LUCID_HD QueryBlocks query_blocks(const AttnShape& a, int tile, int len) {
  QueryBlocks q;
  const int j0 = tile << 7, j1 = imin(j0 + 127, len - 1);
  const int i_max = imin(a.Nq, len - a.off) - 1;         // last valid query
  q.first = imax(0, j0 - a.off) >> 7;
  q.last = -1;
  if (j0 >= len || i_max < 0 || a.W == 0) {
    q.first = 0;
    return q;
  }
  const int i_hi = a.W >= kNoWindow ? i_max : imin(i_max, j1 + a.W - 1 - a.off);
  if (i_hi < imax(0, j0 - a.off)) {
    q.first = 0;
    return q;
  }
  q.last = i_hi >> 7;
  return q;
}
// Query blocks that see key tile 0 only through the visible first keys: those behind the window's, up to the last
// valid query.
LUCID_HD QueryBlocks sink_blocks(const AttnShape& a, int len) {
  const QueryBlocks w = query_blocks(a, 0, len);
  QueryBlocks q;
  const int i_max = imin(a.Nq, len - a.off) - 1;
  q.first = w.last + 1;
  q.last = (a.S > 0 && i_max >= 0 && len > 0) ? i_max >> 7 : -1;
  return q;
}

// dK/dV work items.  Every key tile of a (batch, key head) is one item.  The query blocks that see key tile 0 only
// through the visible first keys would make its item as long as the sequence: they are dealt out in chunks of
// `chunk` blocks as items of their own, whose sums meet in fp32 and are added in a fixed order.
LUCID_HD int sink_chunk_blocks(const AttnShape& a) { return a.W >= kNoWindow ? 1 : imax(8, a.W / 128 + 2); }
LUCID_HD int sink_chunks(const AttnShape& a) {           // per (batch, key head), from the longest possible sequence
  if (a.S == 0) return 0;
  const QueryBlocks q = sink_blocks(a, a.Nk);
  const int n = q.last - q.first + 1, c = sink_chunk_blocks(a);
  return n > 0 ? (n + c - 1) / c : 0;
}
struct KvItem {
  int b, hk, tile;
  int chunk;             // -1: the tile's own item; else the chunk of its first-key blocks
};
LUCID_HD int kv_items(const AttnShape& a) { return a.B * a.Hkv * (a.nkb + sink_chunks(a)); }
LUCID_HD bool kv_item(const AttnShape& a, int chunks, int idx, KvItem& it) {
  const int per = a.B * a.Hkv;
  if (idx >= per * (a.nkb + chunks)) return false;
  const int s = idx / per, r = idx % per;
  it.b = r / a.Hkv;
  it.hk = r % a.Hkv;
  it.chunk = s < chunks ? s : -1;
  it.tile = s < chunks ? 0 : s - chunks;
  return true;
}
// the blocks of an item; for chunks counted from the longest possible sequence, so that they do not depend on `len`
LUCID_HD QueryBlocks item_blocks(const AttnShape& a, const KvItem& it, int len) {
  if (it.chunk < 0) return query_blocks(a, it.tile, len);
  const QueryBlocks all = sink_blocks(a, len);
  QueryBlocks q;
  const int c = sink_chunk_blocks(a);
  const int base = sink_blocks(a, a.Nk).first;
  q.first = it.chunk == 0 ? all.first : imax(all.first, base + it.chunk * c);
  q.last = imin(all.last, base + it.chunk * c + c - 1);
  return q;
}

// Single-token attention over a paged cache of `cap` positions: what the query at position len - 1 sees, positions 0 ..
// first-1 and lo .. lo+near-1, counted through as 0 .. n-1.  A length beyond the cache (reported where the newest position is
// looked up) moves the window like any other; the positions that do not exist are left out, not replaced by earlier ones.
struct Visible {
  int n, first, lo;
  LUCID_HD int pos(int v) const { return v < first ? v : lo + v - first; }
};
LUCID_HD Visible cache_visible(int W, int S, int len, int cap) {
  Visible v;
  if (len < 0) len = 0;
  v.lo = W < kNoWindow && W < len ? len - W : 0;
  v.first = imin(imin(S, v.lo), cap);
  v.n = v.first + imax(0, imin(len, cap) - v.lo);
  return v;
}

}  // namespace lucid
