// Sliding-window attention with visible first keys, forward, on sm_100a.
//
//   s_ij = scale q_i . k_j over the visible j (attn_geometry.h),  O_i = sum_j exp(s_ij - lse_i) v_j
//
// One pass over the keys with a running maximum m and sum l per row; O is kept in tensor memory relative to a
// reference maximum that is only moved when the running one has outgrown it by 2^8 (exact in the end: O and l share
// the reference, and 2^8 is far from the limits of fp32 sums and 16-bit weights).
//
// A CTA works on two tiles of 128 queries that read the same keys (two heads of a key head, or two neighbouring
// blocks), so a key/value tile brought into shared memory feeds four products.  Per tile of queries: S (fp32, 128
// columns of TMEM; the 16-bit weights P overwrite it) and O (128 columns): 512 columns in all.  While the tensor pipe
// runs one tile's P V and next S, the other tile's warps form exponentials.
//
// Warp roles (384 threads): warp 0 producer; warps 1 and 2 issue the products of one tile each, P V and the next S, taking
// turns: the two tiles' scores become ready half a period apart and their exponentials do not compete (issuers that do not
// take turns interleave their products, and both groups run in phase), while one issuer's waits and the queue's drain are
// covered by the other's products (one warp for both tiles took 2320 cycles per tile, 1460 of them for 16 products); warp 3
// owns TMEM; warps 4-7 and 8-11 are the softmax groups of the two tiles, one row per thread.  P is handed over in two
// halves, so that P V starts while the second half's exponentials are formed.  Persistent CTAs, items dealt out round
// robin, the longest first; results leave through a staging panel per tile and TMA (a thread's own row stores touch 32 lines
// per instruction and took as long as one and a half tiles).
#include <type_traits>
#include "attn.h"

namespace lucid {

static __device__ Control g_attn_fwd_ctl;

constexpr int kFwRing = 4;
struct AttnFwdSmem {
  alignas(1024) uint8_t q[2][kTileBytes];
  alignas(1024) uint8_t ring[kFwRing][kTileBytes];   // K(0), V(0), K(1), V(1), ... of the union of the two tiles' lists
  alignas(1024) uint8_t stage[2][kHalfBytes];         // 128 rows x 64 columns of a tile's result
  alignas(8) uint64_t full[kFwRing];
  uint64_t empty[kFwRing], q_full[2], q_free[2], s_full[2], p_half[2], p_ready[2], turn[2], meet[2], o_full[2], o_free[2];
  uint32_t tmem_base;
  int abort_flag;
};

enum AttnFwdBar : int { AF_FULL = 401, AF_EMPTY, AF_Q_FULL, AF_Q_FREE, AF_S_FULL, AF_P_HALF, AF_P_READY, AF_TURN, AF_MEET, AF_O_FULL, AF_O_FREE };

constexpr int kFwThreads = 384;
constexpr int kFwS = 0, kFwO = 256;      // + 128 * tile
constexpr int kFwRegsService = 88, kFwRegsSoftmax = 208;    // 128 * 88 + 256 * 208 = 384 * 168, the launch's total
constexpr float kFwSlack = 8.f;          // log2 of how far the maximum may outgrow the reference

template <bool kBf16>
__global__ void __launch_bounds__(kFwThreads, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_out,
                const AttnFwdArgs args) {
  extern __shared__ uint8_t smem_raw[];
  AttnFwdSmem& s = *reinterpret_cast<AttnFwdSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const AttnShape& A = args.a;
  Control* ctl = &g_attn_fwd_ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned long long limit = args.wait_ns;
  volatile int* cta_abort = &s.abort_flag;

  if (tid == 0) {
    for (int i = 0; i < kFwRing; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_free[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.turn[i], 1);
      mbar_init(&s.meet[i], 128);
      mbar_init(&s.p_half[i], 128);
      mbar_init(&s.p_ready[i], 128);
      mbar_init(&s.o_full[i], 1);
      mbar_init(&s.o_free[i], 128);
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
  auto length_of = [&](int b) -> int { return attn_length(A, args.lengths, b); };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFwRegsService));
    if (warp == 0) {
      // =========================== producer (one lane) ===========================
      if (lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        uint32_t r = 0, stage = 0, phase = 0;
        uint32_t nq[2] = {0, 0};      // Q tiles loaded
        bool alive = true;
        FwdItem it;
        for (int rnd = 0, idx; alive && fwd_item(A, idx = snake_item(rnd, blockIdx.x, gridDim.x), it); ++rnd) {
          const PairTiles pt = pair_tiles(A, it, length_of(it.b));
          auto load = [&](const CUtensorMap* tm, int tile) -> bool {
            if (!wait_lean(&s.empty[stage], phase ^ 1, cta_abort, limit, AF_EMPTY)) return false;
            mbar_expect_tx(&s.full[stage], kTileBytes);
            tma_load_4d(s.ring[stage], tm, &s.full[stage], 0, tile * kBlock, it.hk, it.b);
            tma_load_4d(s.ring[stage] + kHalfBytes, tm, &s.full[stage], 64, tile * kBlock, it.hk, it.b);
            ++r;
            if (++stage == kFwRing) {
              stage = 0;
              phase ^= 1;
            }
            return true;
          };
          for (int t = 0; t < 2 && alive; ++t) {
            if (pt.list(t).n == 0) continue;
            if (!wait_lean(&s.q_free[t], (nq[t] & 1) ^ 1, cta_abort, limit, AF_Q_FREE)) {
              alive = false;
              break;
            }
            ++nq[t];
            mbar_expect_tx(&s.q_full[t], kTileBytes);
            tma_load_4d(s.q[t], &tm_q, &s.q_full[t], 0, it.block(t) * kBlock, it.h(t), it.b);
            tma_load_4d(s.q[t] + kHalfBytes, &tm_q, &s.q_full[t], 64, it.block(t) * kBlock, it.h(t), it.b);
          }
          for (int u = 0; u < pt.n && alive; ++u) {
            const int j = pt.tile(u);
            alive = load(&tm_k, j) && load(&tm_v, j);
          }
        }
      }
    } else if (warp < 3) {
      // =========================== issuer of one tile's products ===========================
      // Step u of the union: P V of the tile's previous entry and S of entry u, in turns with the other tile's issuer
      const int t = warp - 1;
      constexpr int fmt = kBf16 ? 1 : 0;
      constexpr uint32_t idesc_s = umma_idesc(fmt, 0, 0, 128, 128);          // Q K^T: both K-major
      constexpr uint32_t idesc_sn = umma_idesc(fmt, 0, 0, 128, kNarrow);     // the first kNarrow keys only
      constexpr uint32_t idesc_o = umma_idesc(fmt, 0, 1, 128, 128);          // P V: P from TMEM, V rows = k
      const uint64_t dq = umma_smem_desc(smem_u32(s.q[t]), 16, 1024);
      const uint64_t d_k0 = umma_smem_desc(smem_u32(s.ring[0]), 16, 1024);
      const uint64_t d_v0 = umma_smem_desc(smem_u32(s.ring[0]), kHalfBytes, 1024);
      const uint32_t s_tmem = tmem + kFwS + 128 * t, o_tmem = tmem + kFwO + 128 * t;
      uint32_t st = 0, phase = 0;        // ring stage and phase of K(u); V(u) is in the stage behind it
      uint32_t v_st = 0, v_phase = 0;    // V(u - 1)
      uint32_t nq = 0, np = 0, turns = 0;  // items with tiles; weights consumed; turns taken
      bool alive = true;
      FwdItem it;
      for (int rnd = 0, idx; alive && fwd_item(A, idx = snake_item(rnd, blockIdx.x, gridDim.x), it); ++rnd) {
        const PairTiles pt = pair_tiles(A, it, length_of(it.b));
        const KeyTiles kt = pt.list(t);
        bool first = true, pend = false, was_narrow = false;    // pend: the weights of entry u - 1 are this tile's
        int left = kt.n;
        for (int u = 0; u <= pt.n; ++u) {
          const bool more = u < pt.n, act = more && pt.active(kt, u), narrow = more && tile_narrow(A, kt, pt.tile(u));
          if (u > 0 && !wait_lean(&s.full[v_st], v_phase, cta_abort, limit, AF_FULL)) { alive = false; break; }
          if (more && !wait_lean(&s.full[st], phase, cta_abort, limit, AF_FULL)) { alive = false; break; }
          if (act && left == kt.n && !wait_lean(&s.q_full[t], nq & 1, cta_abort, limit, AF_Q_FULL)) { alive = false; break; }
          if (pend) {
            if (!wait_lean(&s.p_half[t], np & 1, cta_abort, limit, AF_P_HALF)) { alive = false; break; }
            // the epilogue of this tile's previous item has read O
            if (first && !wait_lean(&s.o_free[t], (nq & 1) ^ 1, cta_abort, limit, AF_O_FREE)) { alive = false; break; }
          }
          const uint64_t dv = d_v0 + v_st * (kTileBytes >> 4), dk = d_k0 + st * (kTileBytes >> 4);
          if (!wait_lean(&s.turn[t], (turns & 1) ^ (t ^ 1), cta_abort, limit, AF_TURN)) { alive = false; break; }
          ++turns;
          tc_fence_after_sync();
          if (pend) {
            const uint32_t add = first ? 0u : 1u;
            if (was_narrow) {
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kNarrow / 16; ++k) umma_ts(o_tmem, s_tmem + 8 * k, dv + k * (2048 >> 4), idesc_o, k ? 1u : add);
              }
            } else {
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_ts(o_tmem, s_tmem + 8 * k, dv + k * (2048 >> 4), idesc_o, k ? 1u : add);
              }
            }
            if (!wait_lean(&s.p_ready[t], np & 1, cta_abort, limit, AF_P_READY)) { alive = false; break; }
            ++np;
            if (!was_narrow) {
              tc_fence_after_sync();
              if (elect_one()) {
#pragma unroll
                for (int k = 4; k < 8; ++k) umma_ts(o_tmem, s_tmem + 8 * k, dv + k * (2048 >> 4), idesc_o, 1u);
              }
            }
            first = false;
          }
          if (act) {
            const uint32_t idesc = narrow ? idesc_sn : idesc_s;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
                umma_ss(s_tmem, dq + off, dk + off, idesc, k ? 1u : 0u);
              }
            }
            --left;
          }
          __syncwarp();
          if (elect_one()) {
            mbar_arrive(&s.turn[t ^ 1]);
            if (act) umma_commit(&s.s_full[t]);
            // the stages go back when both issuers' products that read them are complete (an issuer without products
            // on them only says that it is past them)
            if (u > 0) umma_commit(&s.empty[v_st]);
            if (more) umma_commit(&s.empty[st]);
            if (act && left == 0) umma_commit(&s.q_free[t]);
            // the tile's last weights have been consumed: its result is complete
            if (pend && !act && left == 0) umma_commit(&s.o_full[t]);
          }
          if (pend && !act && left == 0) ++nq;
          pend = act;
          was_narrow = narrow;
          if (more) {
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
          }
        }
      }
    }
  } else {
    // =========================== softmax of one tile, then its epilogue ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFwRegsSoftmax));
    const int t = (warp - 4) >> 2;
    const int row = ((warp & 3) << 5) + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + kFwS + 128 * t, o_tmem = tmem + lanes + kFwO + 128 * t;
    const float sl2 = args.scale_log2;
    const unsigned long long sl22 = f32x2(sl2, sl2);
    uint32_t ns = 0, no = 0, r = 0, meets = 0;
    // the tile's 128 threads meet (an mbarrier and not a named barrier: this wait, too, has a limit)
    auto meet = [&]() -> bool {
      mbar_arrive(&s.meet[t]);
      return wait_lean(&s.meet[t], meets++ & 1, cta_abort, limit, AF_MEET);
    };
    bool alive = true;
    FwdItem it;
    for (int rnd = 0, idx; alive && fwd_item(A, idx = snake_item(rnd, blockIdx.x, gridDim.x), it); ++rnd) {
      const int len = length_of(it.b);
      const PairTiles pt = pair_tiles(A, it, len);
      const KeyTiles kt = pt.list(t);
      const int i = it.block(t) * kBlock + row;
      const int p = i + A.off;
      const bool valid = i < A.Nq && p < len;
      float ref = -INFINITY, l = 0.f;
      for (int x = 0; x < kt.n; ++x, ++ns) {
        const int tile = kt.tile(x), j0 = tile << 7;
        if (!wait_lean(&s.s_full[t], ns & 1, cta_abort, limit, AF_S_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        const bool masked = tile_masked(A, kt, tile, len);
        const RowMask mask = row_mask(A, p, j0, len);
        if (masked) {
          if (j0 + 127 >= len && len < A.Nk) {
            // rows behind the sequence hold anything, and 0 * NaN is not 0: the value tile's become zero
            const uint32_t use = r + 2 * (tile == 0 && pt.sink ? 0 : tile - pt.lo + pt.sink) + 1;
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
        auto weights = [&](auto chunks) {
          constexpr int kChunks = decltype(chunks)::value;
          uint32_t v[kChunks][32];
#pragma unroll
          for (int c = 0; c < kChunks; ++c) tmem_ld32(s_tmem + 32 * c, v[c]);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              const uint32_t w = mask.word(32 * c);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[c][e] = (w & (1u << e)) ? v[c][e] : 0xff800000u;
            }
          }
          float mx[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) mx[x] = __uint_as_float(v[0][x]);
#pragma unroll
          for (int x = 4; x < 32 * kChunks; ++x) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(v[x >> 5][x & 31]));
          const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
          const bool grow = m > ref + kFwSlack;
          if (x == 0) {
            ref = m;
          } else if (__any_sync(0xffffffffu, grow)) {
            // S(u) is complete, and with it every product issued before it: O holds all earlier tiles
            const float next = fmaxf(ref, m);
            const float f = next == -INFINITY ? 1.f : ex2_approx(ref - next);
            ref = next;
            l *= f;
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
          unsigned long long sum = 0, sum2 = 0;          // two zeros each
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const unsigned long long y =
                  f32x2_fma(f32x2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), sl22, neg2);
              float2 w = f32x2_unpack(y);
              w.x = ex2_approx(w.x);
              w.y = ex2_approx(w.y);
              if (e & 1) sum2 = f32x2_add(sum2, f32x2(w.x, w.y));
              else sum = f32x2_add(sum, f32x2(w.x, w.y));
              pk[e] = pack2<kBf16>(w.x, w.y);
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
          const float2 both = f32x2_unpack(f32x2_add(sum, sum2));
          l += both.x + both.y;
        };
        if (tile_narrow(A, kt, tile)) weights(std::integral_constant<int, kNarrow / 32>{});
        else weights(std::integral_constant<int, 4>{});
      }
      if (!alive) break;
      r += 2 * pt.n;

      // ---- epilogue ----
      const bool has = kt.n > 0;
      if (has) {
        if (!wait_lean(&s.o_full[t], no & 1, cta_abort, limit, AF_O_FULL)) break;
        ++no;
        tc_fence_after_sync();
      }
      const bool some = valid && l != 0.f;      // (a NaN sum is written as it is)
      const float inv = some ? 1.f / l : 0.f;
      const bool lead = (tid & 127) == 0;
      if (it.block(t) < A.nqb) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (lead) tma_store_wait_read();               // the panel's previous store has read it
          if (!meet()) { alive = false; break; }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            if (has) {
              tmem_ld32(o_tmem + 64 * hf + 32 * c, o);
              tmem_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint4 w = make_uint4(0, 0, 0, 0);
              if (has && some) {
                w.x = pack2<kBf16>(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv);
                w.y = pack2<kBf16>(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv);
                w.z = pack2<kBf16>(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv);
                w.w = pack2<kBf16>(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv);
              }
              *reinterpret_cast<uint4*>(s.stage[t] + sw128_off(row, 4 * c + e)) = w;
            }
          }
          fence_proxy_async_smem();
          if (!meet()) { alive = false; break; }
          if (lead) {                                    // rows behind Nq lie outside the map and are not written
            tma_store_4d(&tm_out, s.stage[t], 64 * hf, it.block(t) * kBlock, it.h(t), it.b);
            tma_store_commit();
          }
        }
      }
      if (has) {
        tc_fence_before_sync();
        mbar_arrive(&s.o_free[t]);
      }
      if (i < A.Nq && args.lse)
        args.lse[((long long)it.b * A.Hq + it.h(t)) * A.Nq + i] =
            some ? (ref + log2f(l)) * 0.6931471805599453f : -INFINITY;
    }
    if ((tid & 127) == 0) tma_store_wait_read();
  }

  if (s.abort_flag) {
    // a role gave up: leave the copies and products in flight time to land before the CTA's memory goes
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    if (tid == 0) report_error(ctl, kErrBarrierTimeout, -1, -1, blockIdx.x, s.abort_flag);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 3) tmem_dealloc(tmem, 512);
}

cudaError_t launch_attn_fwd(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                            const CUtensorMap& tm_out, const AttnFwdArgs& args, int sms, cudaStream_t stream) {
  const int items = fwd_items(args.a), grid = items < sms ? items : sms;
  const int bytes = (int)sizeof(AttnFwdSmem) + 1024;
  auto kernel = bf16 ? attn_fwd_kernel<true> : attn_fwd_kernel<false>;
  static SmemOnce once[2];
  cudaError_t e = once[bf16].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kFwThreads, bytes, stream>>>(tm_q, tm_k, tm_v, tm_out, args);
  return cudaGetLastError();
}

cudaError_t attn_fwd_status(cudaStream_t stream, int out[8]) { return take_status(&g_attn_fwd_ctl, stream, out); }

}  // namespace lucid
