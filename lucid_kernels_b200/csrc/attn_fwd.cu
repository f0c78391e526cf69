// Sliding-window attention with visible first keys, forward, on sm_100a.
//
//   s_ij = scale q_i . k_j over the visible j (attn_geometry.h),  O_i = sum_j exp(s_ij - lse_i) v_j
//
// One pass over the keys with a running maximum m and sum l per row; O is kept in tensor memory relative to a
// reference maximum that is only moved when the running one has outgrown it by 2^8 (exact in the end: O and l share
// the reference, and 2^8, for fp16 2^12 (kTopWeight), is inside the limits of fp32 sums and 16-bit weights).
//
// A CTA works on two tiles of 128 queries that read the same keys (two heads of a key head, or two neighbouring
// blocks), so a key/value tile brought into shared memory feeds four products.  Per tile of queries: S (fp32, 128
// columns of TMEM; the 16-bit weights P overwrite it) and O (128 columns): 512 columns in all.  While the tensor pipe
// runs one tile's P V and next S, the other tile's warps form exponentials.
//
// Warp roles (512 threads): warp 0 producer; warps 1 and 2 issue the products of one tile each, P V and the next S, taking
// turns: the two tiles' scores become ready half a period apart and their exponentials do not compete (issuers that do not
// take turns interleave their products, and both groups run in phase), while one issuer's waits and the queue's drain are
// covered by the other's products (65536 tokens, 8/4 heads, window 1024: 320 us where one warp for both tiles took 348); warp 3
// owns TMEM; warps 4-7 write finished results beside the next item's first
// tiles; warps 8-11 and 12-15 are the softmax groups of the two tiles, one row per thread.  P is handed over in two
// halves, so that P V starts while the second half's exponentials are formed.  Persistent CTAs, items dealt out back and forth, the
// longest first; the steps of consecutive items follow one another without a pause.
#include <type_traits>
#include "attn.h"

namespace lucid {

static __device__ Control g_attn_fwd_ctl;

constexpr int kFwRing = 4, kFwSlots = 4;

// An item as its roles need it, worked out by one thread: its divisions and lists would be in every role's way
struct FwdSlot {
  int n;                  // entries of the union, -1: no more items
  int b, hk, len, sink, lo;
  struct Tile {
    int h, block;
    KeyTiles list;        // its own entries
    OwnEntries own;       // which of the union's they are (not split)
  } t[2];
  __device__ __forceinline__ int tile(int u, bool split) const {
    if (!split) return u < sink ? 0 : lo + u - sink;
    return split_entry(t[0].list, t[1].list, u);
  }
};
struct AttnFwdSmem {
  alignas(1024) uint8_t q[2][kTileBytes];
  alignas(1024) uint8_t ring[kFwRing][kTileBytes];   // K(0), V(0), K(1), V(1), ... of the union of the two tiles' lists
  alignas(1024) uint8_t stage[kTileBytes];            // a tile's result: per warp two panels of 32 rows x 64 columns
  alignas(8) uint64_t full[kFwRing];
  uint64_t empty[kFwRing], q_full[2], q_free[2], s_full[2], p_half[2], p_ready[2], turn[2], o_full[2], o_free[2], l_full[2], l_free[2];
  uint64_t slot_full[kFwSlots], slot_free[kFwSlots];
  FwdSlot slot[kFwSlots];
  alignas(16) float2 l[2][kBlock];       // a finished row's sum and the reference of its exponents (kTrain: and its lse in base 2)
  uint32_t tmem_base;
  int abort_flag;
};

static_assert(sizeof(AttnFwdSmem) <= 232448, "shared memory of a CTA");

enum AttnFwdBar : int { AF_FULL = 401, AF_EMPTY, AF_Q_FULL, AF_Q_FREE, AF_S_FULL, AF_P_HALF, AF_P_READY, AF_TURN, AF_O_FULL, AF_O_FREE, AF_L_FULL, AF_L_FREE, AF_SLOT_FULL, AF_SLOT_FREE };

constexpr int kFwThreads = 512;
constexpr int kFwS = 0, kFwO = 256;      // + 128 * tile
constexpr int kFwRegsService = 80, kFwRegsSoftmax = 176;    // 256 * 80 + 256 * 176 = 512 * 128, the launch's total
constexpr float kFwSlack = 8.f;          // log2 of how far the maximum may outgrow the reference

// A part's O in the ring: rows of 128 fp32, 16-byte pieces permuted by the row (threads of a warp write equal pieces of 32 rows)
__device__ __forceinline__ uint32_t join_off(int row, int piece) { return row * 512 + ((piece ^ (row & 31)) << 4); }

// This CTA's share of a tile's rows, joined from the parts of all CTAs of the cluster.  One warp per row, four columns per lane;
// 8 warps call it.
template <bool kBf16>
__device__ __forceinline__ void join_rows(AttnFwdSmem& s, const AttnFwdArgs& args, int warp, int lane) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  const AttnShape& A = args.a;
  const int parts = args.parts, part = blockIdx.x % parts, per = kBlock / parts;
  FwdItem it;
  if (!fwd_item(A, true, blockIdx.x / parts, it)) return;
  const int len = attn_length(A, args.lengths, it.b);
  const uint32_t sums = smem_u32(s.ring[2]), tile = smem_u32(s.ring[0]);
  elem_t* out = reinterpret_cast<elem_t*>(args.out) + it.b * args.out_strides.b + it.h0 * args.out_strides.h + 4 * lane;
  for (int y = warp; y < per; y += 8) {
    const int r = part * per + y, i = it.block0 * kBlock + r;
    if (i >= A.Nq) break;
    float l[8], ref[8], top = -INFINITY;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      l[p] = 0.f;
      ref[p] = -INFINITY;
      if (p < parts) ld_cluster2(mapa_u32(sums + 8 * r, p), l[p], ref[p]);
      top = fmaxf(top, ref[p]);
    }
    float sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      if (l[p] == 0.f) continue;            // (no weight: nothing was written there; a NaN sum goes on)
      const float f = top == -INFINITY ? 1.f : ex2_approx(ref[p] - top);
      float o[4];
      ld_cluster4(mapa_u32(tile + join_off(r, lane), p), o);
      sum += f * l[p];
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += f * o[e];
    }
    const bool some = i + A.off < len && sum != 0.f;
    const float inv = some ? 1.f / sum : 0.f;
    uint2 w = make_uint2(0u, 0u);
    if (some) w = make_uint2(pack2<kBf16>(a[0] * inv, a[1] * inv), pack2<kBf16>(a[2] * inv, a[3] * inv));
    *reinterpret_cast<uint2*>(out + (long long)i * args.out_strides.n) = w;
  }
}

// The result is normalised by the sum of the weights as they are rounded, so that it is a mean of values even where one
// weight is nearly all (the mixed-precision adds cost nothing measurable; unpacking the halves first took 8 % longer).
// kTrain: lse is wanted, for a backward to come.  lse comes from the sum of the weights themselves, and what the rounding of the result
// takes off is kept (if `rest` is given): delta = dO . O is subtracted from a nearly equal dO . v_j where a row is peaked.
// kJoin: a cluster of `parts` CTAs owns one tile of queries, each CTA a run of its keys; they leave O (fp32, unnormalised),
// sums and references in the ring, which is free by then, and each joins a share of the rows from all CTAs' shared memory.
template <bool kBf16, bool kTrain, bool kJoin>
__global__ void __launch_bounds__(kFwThreads, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const AttnFwdArgs args) {
  // (no room to round the base up: the kernel has no static shared memory, and the window starts on 1 KiB)
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  AttnFwdSmem& s = *reinterpret_cast<AttnFwdSmem*>(smem_raw);
  const AttnShape& A = args.a;
  Control* ctl = &g_attn_fwd_ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned long long limit = args.wait_ns;
  volatile int* cta_abort = &s.abort_flag;

  if (smem_u32(smem_raw) & 1023) {       // (operand tiles would be misread)
    if (tid == 0) report_error(ctl, kErrAborted, -1, -1, blockIdx.x, 0);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < kFwRing; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 2);
    }
    for (int i = 0; i < kFwSlots; ++i) {
      mbar_init(&s.slot_full[i], 1);
      mbar_init(&s.slot_free[i], 15);      // producer, two issuers, four epilogue and eight softmax warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_free[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.turn[i], 1);
      mbar_init(&s.p_half[i], 128);
      mbar_init(&s.p_ready[i], 128);
      mbar_init(&s.o_full[i], 1);
      mbar_init(&s.o_free[i], 128);
      mbar_init(&s.l_full[i], 128);
      mbar_init(&s.l_free[i], 128);
    }
    s.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 3) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s.tmem_base;
  const bool split = args.split != 0;
  // The items of this CTA, one after another: `next` waits for the slot, `done` hands it back (per warp; whoever reads it
  // later keeps copies).
  uint32_t slots = 0;
  auto next = [&](bool one_thread = false) -> const FwdSlot* {
    uint64_t* bar = &s.slot_full[slots % kFwSlots];
    const uint32_t parity = (slots / kFwSlots) & 1;
    if (!(one_thread ? wait_lane(bar, parity, cta_abort, limit, AF_SLOT_FULL) : wait_lean(bar, parity, cta_abort, limit, AF_SLOT_FULL)))
      return nullptr;
    const FwdSlot* slot = &s.slot[slots % kFwSlots];
    return slot->n < 0 ? nullptr : slot;
  };
  auto done = [&](bool one_thread) {
    if (!one_thread) __syncwarp();
    if (one_thread || lane == 0) mbar_arrive(&s.slot_free[slots % kFwSlots]);
    ++slots;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFwRegsService));
    if (warp == 0) {
      // =========================== producer (one lane) ===========================
      if (lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        uint32_t stage = 0, phase = 0;
        uint32_t nq[2] = {0, 0};      // Q tiles loaded
        bool alive = true;
        while (alive) {
          const FwdSlot* it = next(true);
          if (!it) break;
          const int b = it->b, hk = it->hk;
          auto load = [&](const CUtensorMap* tm, int tile) -> bool {
            if (!wait_lane(&s.empty[stage], phase ^ 1, cta_abort, limit, AF_EMPTY)) return false;
            mbar_expect_tx(&s.full[stage], kTileBytes);
            tma_load_4d(s.ring[stage], tm, &s.full[stage], 0, tile * kBlock, hk, b);
            tma_load_4d(s.ring[stage] + kHalfBytes, tm, &s.full[stage], 64, tile * kBlock, hk, b);
            if (++stage == kFwRing) {
              stage = 0;
              phase ^= 1;
            }
            return true;
          };
          for (int t = 0; t < 2; ++t) {
            if (it->t[t].list.n == 0) continue;
            if (!wait_lane(&s.q_free[t], (nq[t] & 1) ^ 1, cta_abort, limit, AF_Q_FREE)) {
              alive = false;
              break;
            }
            ++nq[t];
            mbar_expect_tx(&s.q_full[t], kTileBytes);
            tma_load_4d(s.q[t], &tm_q, &s.q_full[t], 0, it->t[t].block * kBlock, it->t[t].h, b);
            tma_load_4d(s.q[t] + kHalfBytes, &tm_q, &s.q_full[t], 64, it->t[t].block * kBlock, it->t[t].h, b);
          }
          for (int u = 0, n = it->n; u < n && alive; ++u) {
            const int j = it->tile(u, split);
            alive = load(&tm_k, j) && load(&tm_v, j);
          }
          done(true);
        }
      }
    } else if (warp == 3) {
      // =========================== the items (one lane) ===========================
      if (lane == 0) {
        FwdItem it;
        for (int rnd = 0;; ++rnd) {
          const int k = rnd % kFwSlots;
          if (!wait_lane(&s.slot_free[k], ((rnd / kFwSlots) & 1) ^ 1, cta_abort, limit, AF_SLOT_FREE)) break;
          FwdSlot& x = s.slot[k];
          const bool more = kJoin ? rnd == 0 && fwd_item(A, true, blockIdx.x / args.parts, it)
                                  : fwd_item(A, split, snake_item(rnd, blockIdx.x, gridDim.x), it);
          if (more) {
            x.len = attn_length(A, args.lengths, it.b);
            const PairTiles pt = pair_tiles(A, it, x.len);
            const KeyTiles run = kJoin ? part_list(pt.x, blockIdx.x % args.parts, args.parts) : pt.x;
            x.n = kJoin ? run.n : pt.n;
            x.b = it.b;
            x.hk = it.hk;
            x.sink = pt.sink;
            x.lo = pt.lo;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const KeyTiles kt = split ? half_list(run, t) : pt.list(t);
              FwdSlot::Tile& y = x.t[t];
              y.h = it.h(t);
              y.block = it.block(t);
              y.list = kt;
              y.own = own_entries(kt, pt.lo, pt.sink);
            }
          } else {
            x.n = -1;
          }
          mbar_arrive(&s.slot_full[k]);
          if (!more) break;
        }
      }
    } else if (warp < 3) {
      // =========================== issuer of one tile's products ===========================
      // A step per entry of the items' unions, one after another, and one at the end: P V of this tile's previous entry (it
      // may be the last of the item before), then S of this entry, in turns with the other tile's issuer.  One thread has
      // the role to itself (votes of the whole warp at each wait took 2.5 % longer in the 64k prefill).
      if (elect_one()) {
        const int t = warp - 1;
        constexpr int fmt = kBf16 ? 1 : 0;
        constexpr uint32_t idesc_s = umma_idesc(fmt, 0, 0, 128, 128);          // Q K^T: both K-major
        constexpr uint32_t idesc_sn = umma_idesc(fmt, 0, 0, 128, kNarrow);     // the first kNarrow keys only
        constexpr uint32_t idesc_o = umma_idesc(fmt, 0, 1, 128, 128);          // P V: P from TMEM, V rows = k
        const uint64_t dq = umma_smem_desc(smem_u32(s.q[t]), 16, 1024);
        const uint64_t d_k0 = umma_smem_desc(smem_u32(s.ring[0]), 16, 1024);
        const uint64_t d_v0 = umma_smem_desc(smem_u32(s.ring[0]), kHalfBytes, 1024);
        const uint32_t s_tmem = tmem + kFwS + 128 * t, o_tmem = tmem + kFwO + 128 * t;
        uint32_t st = 0, phase = 0;             // ring stage and phase of this entry's K; its V is in the stage behind it
        uint32_t v_st = 0, v_phase = 0;         // V of the entry before
        uint32_t nq = 0, no = 0, np = 0, turns = 0;   // items begun and results begun (with tiles); weights consumed; turns taken
        bool before = false;                    // is there an entry before
        bool pend = false, pend_first = false, pend_last = false, pend_narrow = false;   // its weights are this tile's
        auto step = [&](bool more, bool act, bool first, bool last, bool narrow) -> bool {
          if (before && !wait_lane(&s.full[v_st], v_phase, cta_abort, limit, AF_FULL)) return false;
          if (more && !wait_lane(&s.full[st], phase, cta_abort, limit, AF_FULL)) return false;
          if (act && first && !wait_lane(&s.q_full[t], nq++ & 1, cta_abort, limit, AF_Q_FULL)) return false;
          if (pend) {
            if (!wait_lane(&s.p_half[t], np & 1, cta_abort, limit, AF_P_HALF)) return false;
            // the epilogue of this tile's previous item has read O
            if (pend_first && !wait_lane(&s.o_free[t], (no++ & 1) ^ 1, cta_abort, limit, AF_O_FREE)) return false;
          }
          const uint64_t dv = d_v0 + v_st * (kTileBytes >> 4), dk = d_k0 + st * (kTileBytes >> 4);
          if (!wait_lane(&s.turn[t], (turns++ & 1) ^ (t ^ 1), cta_abort, limit, AF_TURN)) return false;
          tc_fence_after_sync();
          if (pend) {
            const uint32_t add = pend_first ? 0u : 1u;
            if (pend_narrow) {
#pragma unroll
              for (int k = 0; k < kNarrow / 16; ++k) umma_ts(o_tmem, s_tmem + 8 * k, dv + k * (2048 >> 4), idesc_o, k ? 1u : add);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) umma_ts(o_tmem, s_tmem + 8 * k, dv + k * (2048 >> 4), idesc_o, k ? 1u : add);
            }
            if (!wait_lane(&s.p_ready[t], np++ & 1, cta_abort, limit, AF_P_READY)) return false;
            if (!pend_narrow) {
              tc_fence_after_sync();
#pragma unroll
              for (int k = 4; k < 8; ++k) umma_ts(o_tmem, s_tmem + 8 * k, dv + k * (2048 >> 4), idesc_o, 1u);
            }
            if (pend_last) umma_commit(&s.o_full[t]);
          }
          if (act) {
            const uint32_t idesc = narrow ? idesc_sn : idesc_s;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
              umma_ss(s_tmem, dq + off, dk + off, idesc, k ? 1u : 0u);
            }
          }
          mbar_arrive(&s.turn[t ^ 1]);
          if (act) umma_commit(&s.s_full[t]);
          // the stages go back when both issuers' products that read them are complete (an issuer without products on
          // them only says that it is past them)
          if (before) umma_commit(&s.empty[v_st]);
          if (more) umma_commit(&s.empty[st]);
          if (act && last) umma_commit(&s.q_free[t]);
          pend = act;
          pend_first = first;
          pend_last = last;
          pend_narrow = narrow;
          before = true;
          v_st = st + 1;
          v_phase = phase;
          if (v_st == kFwRing) {
            v_st = 0;
            v_phase ^= 1;
          }
          st = v_st + 1;
          phase = v_phase;
          if (st == kFwRing) {
            st = 0;
            phase ^= 1;
          }
          return true;
        };
        bool alive = true;
        while (alive) {
          const FwdSlot* it = next(true);
          if (!it) break;
          const int n = it->n, count = it->t[t].list.n;
          const OwnEntries own = it->t[t].own;
          done(true);
          const bool narrow0 = own.first && A.S <= kNarrow;       // (tile_narrow)
          int at = 0;
          for (int u = 0; u < n && alive; ++u) {
            const bool act = split ? (u & 1) == t : own.has(u);
            alive = step(true, act, at == 0, at == count - 1, narrow0 && u == 0);
            if (act) ++at;
          }
        }
        if (alive && before) step(false, false, false, false, false);
      }
    }
  } else if (warp < 8) {
    // =========================== epilogue of both tiles ===========================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFwRegsService));
    typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
    const int row = ((warp & 3) << 5) + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // Through two staging panels of the warp's own, 32 rows x 64 columns each: a thread has a row, but its own stores would
    // touch 32 lines per instruction; read back in rows, one instruction writes four lines.  O is handed back as soon as it
    // stands in the panels: the next item's first P V waits for it.
    uint8_t* panel = s.stage + (warp & 3) * 8192;
    uint32_t no0 = 0, no1 = 0;
    bool alive = true;
    while (alive) {
      const FwdSlot* it = next();
      if (!it) break;
      const int len = it->len, b = it->b;
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const int block = it->t[t].block, h = it->t[t].h;
        if (block >= A.nqb || (split && t)) continue;
        const bool has = it->t[t].list.n > 0;
        const int i = block * kBlock + row;
        float l = 0.f, ref = 0.f;
        // split: the other half's sum and reference, and the factors that bring both halves to a common reference
        const bool two = split && it->t[1].list.n > 0;
        float f0 = 1.f, f1 = 0.f;
        if (two) {
          if (!wait_lean(&s.l_full[1], no1 & 1, cta_abort, limit, AF_L_FULL)) { alive = false; break; }
          const float2 x = s.l[1][row];
          mbar_arrive(&s.l_free[1]);
          if (!wait_lean(&s.o_full[1], no1 & 1, cta_abort, limit, AF_O_FULL)) { alive = false; break; }
          ++no1;
          l = x.x;
          ref = x.y;
        }
        if (has) {
          const uint32_t n = t ? no1++ : no0++;
          if (!wait_lean(&s.l_full[t], n & 1, cta_abort, limit, AF_L_FULL)) { alive = false; break; }
          const float2 x = s.l[t][row];
          mbar_arrive(&s.l_free[t]);
          if (two) {
            const float both = fmaxf(x.y, ref), z = both == -INFINITY ? 0.f : both;
            f0 = ex2_approx(x.y - z);
            f1 = ex2_approx(ref - z);
            l = x.x * f0 + l * f1;
            ref = both;
          } else {
            l = x.x;
            ref = x.y;
          }
          if (!wait_lean(&s.o_full[t], n & 1, cta_abort, limit, AF_O_FULL)) { alive = false; break; }
          tc_fence_after_sync();
        }
        const bool some = i + A.off < len && l != 0.f;     // (a NaN sum is written as it is)
        const float inv = some ? 1.f / l : 0.f;
        elem_t* out = reinterpret_cast<elem_t*>(args.out) + b * args.out_strides.b + h * args.out_strides.h + (lane & 7) * 8;
        const int r0 = block * kBlock + (warp & 3) * 32 + (lane >> 3);
        const uint32_t o_tmem = tmem + lanes + kFwO + 128 * t;
        const int rest_step = rest_rows(A) * 8;
        const bool keep = kTrain && args.rest && row < rest_rows(A);
        elem_t* rest = keep ? reinterpret_cast<elem_t*>(args.rest) + (((long long)b * A.Hq + h) * A.nqb + block) * 16 * rest_step + row * 8 : nullptr;
        if (has) {
          uint32_t oa[16], ob[16];
          auto put = [&](const uint32_t (&o)[16], int c) {        // columns 16c .. 16c+15
            if constexpr (kJoin) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint4*>(s.ring[0] + join_off(row, 4 * c + e)) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
              return;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint4 w = make_uint4(0, 0, 0, 0);
              if (some) {
                w.x = pack2<kBf16>(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
                w.y = pack2<kBf16>(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
                w.z = pack2<kBf16>(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
                w.w = pack2<kBf16>(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
              }
              *reinterpret_cast<uint4*>(panel + (c >> 2) * 4096 + sw128_off(lane, 2 * (c & 3) + e)) = w;
              if (kTrain && keep) {
                const uint32_t hi[4] = {w.x, w.y, w.z, w.w};
                uint32_t lo[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const float2 h2 = unpack2<kBf16>(hi[y]);
                  lo[y] = some ? pack2<kBf16>(__uint_as_float(o[8 * e + 2 * y]) * inv - h2.x, __uint_as_float(o[8 * e + 2 * y + 1]) * inv - h2.y) : 0u;
                }
                *reinterpret_cast<uint4*>(rest + (2 * c + e) * rest_step) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            }
          };
          if (two) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              tmem_ld16(o_tmem + 16 * c, oa);
              tmem_ld16(o_tmem + 128 + 16 * c, ob);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) oa[e] = __float_as_uint(__uint_as_float(oa[e]) * f0 + __uint_as_float(ob[e]) * f1);
              put(oa, c);
            }
            tc_fence_before_sync();
            mbar_arrive(&s.o_free[0]);
            mbar_arrive(&s.o_free[1]);
          } else {
          tmem_ld16(o_tmem, oa);
          tmem_wait_ld();
#pragma unroll 1
          for (int c = 0; c < 8; c += 2) {
            tmem_ld16(o_tmem + 16 * (c + 1), ob);
            put(oa, c);
            tmem_wait_ld();
            if (c < 6) tmem_ld16(o_tmem + 16 * (c + 2), oa);
            else {
              // (all of O is in registers)
              tc_fence_before_sync();
              mbar_arrive(&s.o_free[t]);
            }
            put(ob, c + 1);
            if (c < 6) tmem_wait_ld();
          }
          }
        }
        if (kTrain && keep && !has) {
#pragma unroll 1
          for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(rest + c * rest_step) = make_uint4(0, 0, 0, 0);
        }
        if constexpr (kJoin) {
          reinterpret_cast<float2*>(s.ring[2])[row] = has ? make_float2(l, ref) : make_float2(0.f, -INFINITY);
          continue;
        }
        __syncwarp();
#pragma unroll 1
        for (int y = 0; y < 8; ++y) {
          const uint4 w0 = *reinterpret_cast<const uint4*>(panel + sw128_off(4 * y + (lane >> 3), lane & 7));
          const uint4 w1 = *reinterpret_cast<const uint4*>(panel + 4096 + sw128_off(4 * y + (lane >> 3), lane & 7));
          const uint4 zero = make_uint4(0, 0, 0, 0);
          if (r0 + 4 * y < A.Nq) {
            elem_t* at = out + (long long)(r0 + 4 * y) * args.out_strides.n;
            *reinterpret_cast<uint4*>(at) = has ? w0 : zero;
            *reinterpret_cast<uint4*>(at + 64) = has ? w1 : zero;
          }
        }
        __syncwarp();
        if (kTrain && i < A.Nq) args.lse[((long long)b * A.Hq + h) * A.Nq + i] = some ? ref * 0.6931471805599453f : -INFINITY;
      }
      done(false);
    }
  } else {
    // =========================== softmax of one tile ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFwRegsSoftmax));
    const int t = (warp - 8) >> 2;
    const int row = ((warp & 3) << 5) + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + kFwS + 128 * t, o_tmem = tmem + lanes + kFwO + 128 * t;
    const float sl2 = args.scale_log2;
    const unsigned long long sl22 = f32x2(sl2, sl2);
    uint32_t ns = 0, nl = 0, r = 0;
    bool alive = true;
    while (alive) {
      const FwdSlot* it = next();
      if (!it) break;
      const int len = it->len, u_sink = it->sink, u_lo = it->lo, u_n = it->n;
      const KeyTiles kt = it->t[t].list;
      const int p = it->t[t].block * kBlock + row + A.off;
      done(false);
      float ref = -INFINITY, l16 = 0.f;                // l16: the sum of the weights as they are rounded
      [[maybe_unused]] float l = 0.f;
      for (int x = 0; x < kt.n; ++x, ++ns) {
        const int tile = kt.tile(x), j0 = tile << 7;
        if (!wait_lean(&s.s_full[t], ns & 1, cta_abort, limit, AF_S_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        const bool masked = tile_masked(A, kt, tile, len);
        const RowMask mask = row_mask(A, p, j0, len);
        if (masked) {
          if (j0 + 127 >= len && len < A.Nk) {
            // rows behind the sequence hold anything, and 0 * NaN is not 0: the value tile's become zero
            const uint32_t use = r + 2 * (split ? 2 * x + t : tile == 0 && u_sink ? 0 : tile - u_lo + u_sink) + 1;
            if (!wait_lean(&s.full[use % kFwRing], (use / kFwRing) & 1, cta_abort, limit, AF_FULL)) {
              alive = false;
              break;
            }
            if (j0 + row >= len) zero_tile_row(s.ring[use % kFwRing], row);
            __syncwarp();
            fence_proxy_async_smem();
          }
        }
        // the tile's first 32 * kChunks columns (the rest is not visible, and P is not read there)
        auto weights = [&](auto chunks, auto some_masked) {
          constexpr int kChunks = decltype(chunks)::value;
          constexpr bool kMasked = decltype(some_masked)::value;
          uint32_t v[kChunks][32];
#pragma unroll
          for (int c = 0; c < kChunks; ++c) tmem_ld32(s_tmem + 32 * c, v[c]);
          tmem_wait_ld();
          // most chunks of a masked tile are whole or empty for all rows of a warp
          bool empty[kChunks];
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            empty[c] = false;
            if constexpr (kMasked) {
              const uint32_t w = mask.word(32 * c);
              empty[c] = __all_sync(0xffffffffu, w == 0u);
              if (!empty[c] && !__all_sync(0xffffffffu, w == ~0u)) {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[c][e] = (w & (1u << e)) ? v[c][e] : 0xff800000u;
              }
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            if (kMasked && empty[c]) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(v[c][e]));
          }
          const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
          const float top = m - kTopWeight<kBf16>;
          const bool grow = top > ref + kFwSlack;
          if (x == 0) {
            ref = top;
          } else if (__any_sync(0xffffffffu, grow)) {
            // S(u) is complete, and with it every product issued before it: O holds all earlier tiles
            const float next = fmaxf(ref, top);
            const float f = next == -INFINITY ? 1.f : ex2_approx(ref - next);
            ref = next;
            l16 *= f;
            if constexpr (kTrain) l *= f;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(o_tmem + 16 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(o_tmem + 16 * c, o);
            }
          }
          // (a part of the exponentials as a polynomial on the FMA pipe, one pair in 2, 3 or 4, took 2 to 12 % longer in all)
          const float neg = ref == -INFINITY ? 0.f : -ref;
          const unsigned long long neg2 = f32x2(neg, neg);
          [[maybe_unused]] unsigned long long sum = 0, sum2 = 0;     // two zeros each
          float rounded0 = 0.f, rounded1 = 0.f;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t pk[16];
            if (kMasked && empty[c]) {
#pragma unroll
              for (int e = 0; e < 16; ++e) pk[e] = 0u;
            } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const unsigned long long y =
                  f32x2_fma(f32x2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), sl22, neg2);
              float2 w = f32x2_unpack(y);
              w.x = ex2_approx(w.x);
              w.y = ex2_approx(w.y);
              if constexpr (kTrain) {
                if (e & 1) sum2 = f32x2_add(sum2, f32x2(w.x, w.y));
                else sum = f32x2_add(sum, f32x2(w.x, w.y));
              }
              pk[e] = pack2<kBf16>(w.x, w.y);
              add_halves<kBf16>(rounded0, rounded1, pk[e]);
            }
            }
            tmem_st16(s_tmem + 16 * c, pk);
            if (c == 1 && kChunks > 2) {
              tmem_wait_st();
              tc_fence_before_sync();
              mbar_arrive(&s.p_half[t]);
            }
          }
          tmem_wait_st();
          tc_fence_before_sync();
          if (kChunks <= 2) mbar_arrive(&s.p_half[t]);
          mbar_arrive(&s.p_ready[t]);
          l16 += rounded0 + rounded1;
          if constexpr (kTrain) {
            const float2 both = f32x2_unpack(f32x2_add(sum, sum2));
            l += both.x + both.y;
          }
        };
        if (!masked) weights(std::integral_constant<int, 4>{}, std::false_type{});
        else if (tile_narrow(A, kt, tile)) weights(std::integral_constant<int, kNarrow / 32>{}, std::true_type{});
        else weights(std::integral_constant<int, 4>{}, std::true_type{});
      }
      if (!alive) break;
      r += 2 * u_n;

      if (kt.n > 0) {
        if (!wait_lean(&s.l_free[t], (nl++ & 1) ^ 1, cta_abort, limit, AF_L_FREE)) break;
        if constexpr (kTrain) s.l[t][row] = make_float2(l16, ref + log2f(l));
        else s.l[t][row] = make_float2(l16, ref);
        mbar_arrive(&s.l_full[t]);
      }
    }
  }

  if (s.abort_flag) {
    // a role gave up: leave the copies and products in flight time to land before the CTA's memory goes
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before_sync();
  if constexpr (kJoin) {
    __syncwarp();
    cluster_sync_all();               // (also after an abort: every role comes here)
    if (warp >= 8) join_rows<kBf16>(s, args, warp - 8, lane);
    __syncwarp();
    cluster_sync_all();               // nobody leaves while its memory is being read
  } else {
    __syncthreads();
  }
  // (reported once every role is here: this thread's own role may have ended long before another's wait ran out)
  if (tid == 0 && s.abort_flag) report_error(ctl, kErrBarrierTimeout, -1, -1, blockIdx.x, s.abort_flag);
  if (warp == 3) tmem_dealloc(tmem, 512);
}

template <bool kBf16>
static cudaError_t join_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, int items, int parts, cudaStream_t stream) {
  const int bytes = (int)sizeof(AttnFwdSmem);
  static SmemOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(attn_fwd_kernel<kBf16, false, true>), bytes);
  if (e != cudaSuccess) return e;
  cfg->gridDim = dim3(items * parts);
  cfg->blockDim = dim3(kFwThreads);
  cfg->dynamicSmemBytes = bytes;
  cfg->stream = stream;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = parts;
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 1;
  return cudaSuccess;
}

// How many clusters of `parts` CTAs the device holds at once (its groups of SMs are not multiples of 8); asked once.
template <bool kBf16>
static int clusters_at_once(int parts) {
  static std::atomic<int> known[64][4];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::atomic<int>& k = known[dev][parts >= 8 ? 3 : parts >= 4 ? 2 : 1];
  if ((n = k.load(std::memory_order_relaxed)) > 0) return n - 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  if (join_config<kBf16>(&cfg, attr, 1, parts, nullptr) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, attn_fwd_kernel<kBf16, false, true>, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  k.store(n + 1, std::memory_order_relaxed);
  return n;
}

// Sharing a list costs a cluster launch and the join, some 4 us, and saves up to (1 - 1/parts) of the list's steps: as many CTAs
// as there is room for, two tiles each or more, from 8 tiles on - for two CTAs, which save least, from 12 on.  One query on 65536
// keys, 8 heads: 594 us alone, 85 us in eights; 256 queries on 2048 keys: 26 and 17 us in eights; 1024 queries on 4096 keys: 44 and
// 32 us in twos; 4 tiles: 12.9 and 16 us in twos (alone it is); 1000 queries, 8 tiles: 17.7 and 18.5 us in twos.
int fwd_parts(const AttnShape& a, bool bf16, int sms) {
  const int items = fwd_items(a, true), list = longest_list(a);
  if (list < 8) return 1;
  int parts = 1;
  while (parts < 8 && items * parts * 2 <= sms && list >= parts * 4 &&
         items <= (bf16 ? clusters_at_once<true>(parts * 2) : clusters_at_once<false>(parts * 2)))
    parts *= 2;
  return parts == 2 && list < 12 ? 1 : parts;
}

template <bool kBf16>
static cudaError_t launch_typed(const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const AttnFwdArgs& args,
                                int sms, cudaStream_t stream) {
  const int items = fwd_items(args.a, args.split != 0), grid = items < sms ? items : sms;
  const int bytes = (int)sizeof(AttnFwdSmem);
  if (args.parts > 1) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const cudaError_t e = join_config<kBf16>(&cfg, attr, items, args.parts, stream);
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, attn_fwd_kernel<kBf16, false, true>, tm_q, tm_k, tm_v, args);
  }
  const bool train = args.lse != nullptr;
  auto kernel = train ? attn_fwd_kernel<kBf16, true, false> : attn_fwd_kernel<kBf16, false, false>;
  static SmemOnce once[2];
  const cudaError_t e = once[train].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kFwThreads, bytes, stream>>>(tm_q, tm_k, tm_v, args);
  return cudaGetLastError();
}

cudaError_t launch_attn_fwd(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                            const AttnFwdArgs& args, int sms, cudaStream_t stream) {
  return bf16 ? launch_typed<true>(tm_q, tm_k, tm_v, args, sms, stream) : launch_typed<false>(tm_q, tm_k, tm_v, args, sms, stream);
}

cudaError_t attn_fwd_status(cudaStream_t stream, int out[8]) { return take_status(&g_attn_fwd_ctl, stream, out); }

}  // namespace lucid
