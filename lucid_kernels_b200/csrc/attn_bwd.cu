// Backward of the sliding-window attention with visible first keys, on sm_100a.
//
// With P_ij = exp(scale q_i.k_j - lse_i) over the visible pairs and delta_i = dO_i . O_i:
//     dS = P o (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
// Two passes: attn_dq_kernel owns a block of queries and streams its keys, attn_dkv_kernel owns a block of keys and
// streams the queries (of all heads that share it) that see it.  S and dO V^T are formed twice - seven products per
// pair of tiles where one pass needs five - and in return every sum stays in tensor memory, is added in a fixed order
// and leaves the chip once: no fp32 dQ in memory, no atomics, the same bits on every run.
#include <type_traits>
#include "attn.h"

namespace lucid {

static __device__ Control g_attn_bwd_ctl;

// ------------------------------------------------------------------------------------------------------------------
// Row statistics {lse in base 2, delta}, one row per warp: reads O and dO once, bound by HBM.
// ------------------------------------------------------------------------------------------------------------------
template <bool kBf16>
__global__ void __launch_bounds__(256) attn_stat_kernel(const AttnStatArgs args) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  const AttnShape& A = args.a;
  const int lane = threadIdx.x & 31;
  const int rows = A.nqb * kBlock;                       // padded rows per head
  const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= (long long)A.B * A.Hq * rows) return;
  const int i = (int)(r % rows), bh = (int)(r / rows), b = bh / A.Hq, h = bh % A.Hq;
  float2 st = make_float2(INFINITY, 0.f);                // a row without weight
  if (i < A.Nq) {
    const float lse = args.lse[(long long)bh * A.Nq + i];
    const elem_t* o = reinterpret_cast<const elem_t*>(args.out) + b * args.out_strides.b + (long long)i * args.out_strides.n +
                      h * args.out_strides.h;
    const elem_t* g = reinterpret_cast<const elem_t*>(args.dout) + b * args.dout_strides.b +
                      (long long)i * args.dout_strides.n + h * args.dout_strides.h;
    const uint2 ov = *reinterpret_cast<const uint2*>(o + lane * 4), gv = *reinterpret_cast<const uint2*>(g + lane * 4);
    const float2 o0 = unpack2<kBf16>(ov.x), o1 = unpack2<kBf16>(ov.y), g0 = unpack2<kBf16>(gv.x), g1 = unpack2<kBf16>(gv.y);
    float d = o0.x * g0.x + o0.y * g0.y + o1.x * g1.x + o1.y * g1.y;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
    if (lse != -INFINITY) st = make_float2(lse * kLog2e, d);
  }
  if (lane == 0) args.stat[r] = st;
}

cudaError_t launch_attn_stat(bool bf16, const AttnStatArgs& args, cudaStream_t stream) {
  const long long rows = (long long)args.a.B * args.a.Hq * args.a.nqb * kBlock;
  const unsigned grid = (unsigned)((rows + 7) / 8);
  if (bf16) attn_stat_kernel<true><<<grid, 256, 0, stream>>>(args);
  else attn_stat_kernel<false><<<grid, 256, 0, stream>>>(args);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------
// dQ.  Per key tile three products (S, dO V^T, dS K) against one exponential per pair: about balanced.  Warp roles
// (384 threads): warp 0 producer, warps 1, 2, 3 issue G = dO V^T, S = Q K^T and dS K (one warp per product stream),
// warps 4-11 form dS, 64 columns each group, over S columns they have consumed.  TMEM: S twice, G, dQ.
// ------------------------------------------------------------------------------------------------------------------
struct AttnDqSmem {
  alignas(1024) uint8_t q[kTileBytes];
  alignas(1024) uint8_t go[kTileBytes];            // dO
  alignas(1024) uint8_t kring[3][kTileBytes];
  alignas(1024) uint8_t vring[2][kTileBytes];
  alignas(8) uint64_t k_full[3];
  uint64_t k_empty[3], v_full[2], v_empty[2];
  uint64_t q_full, q_free, go_full, go_free;
  uint64_t s_full[2], g_full, g_free, w_ready[2], sbuf_free[2], acc_full, acc_free;
  uint32_t tmem_base;
  int abort_flag;
};

enum AttnBwdBar : int {
  AB_K_FULL = 501, AB_K_EMPTY, AB_V_FULL, AB_V_EMPTY, AB_Q_FULL, AB_Q_FREE, AB_GO_FULL, AB_GO_FREE, AB_S_FULL, AB_G_FULL,
  AB_G_FREE, AB_W_READY, AB_SBUF_FREE, AB_ACC_FULL, AB_ACC_FREE, AB_P_READY, AB_DS_READY, AB_DP_FULL
};

constexpr int kDqThreads = 384;
constexpr int kDqS = 0, kDqG = 256, kDqAcc = 384;

struct DqItem {
  int b, h, block;
};
__device__ __forceinline__ bool dq_item(const AttnShape& a, int idx, DqItem& it) {
  const int per = a.B * a.Hq;
  if (idx >= per * a.nqb) return false;
  it.block = a.nqb - 1 - idx / per;
  const int r = idx % per;
  it.b = r / a.Hq;
  it.h = r % a.Hq;
  return true;
}

template <bool kBf16>
__global__ void __launch_bounds__(kDqThreads, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
               const AttnBwdArgs args) {
  extern __shared__ uint8_t smem_raw[];
  AttnDqSmem& s = *reinterpret_cast<AttnDqSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const AttnShape& A = args.a;
  Control* ctl = &g_attn_bwd_ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned long long limit = args.wait_ns;
  volatile int* cta_abort = &s.abort_flag;

  if (tid == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.w_ready[i], 256);
      mbar_init(&s.sbuf_free[i], 1);
    }
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_free, 1);
    mbar_init(&s.go_full, 1);
    mbar_init(&s.go_free, 1);
    mbar_init(&s.g_full, 1);
    mbar_init(&s.g_free, 256);
    mbar_init(&s.acc_full, 1);
    mbar_init(&s.acc_free, 256);
    s.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s.tmem_base;
  constexpr int fmt = kBf16 ? 1 : 0;
  constexpr uint32_t idesc_kk = umma_idesc(fmt, 0, 0, 128, 128);
  constexpr uint32_t idesc_mn = umma_idesc(fmt, 0, 1, 128, 128);

  // `g` counts tiles, `it` items that have any, over all items of this CTA
#define DQ_ITEMS                                                                       \
  uint32_t g = 0, itn = 0;                                                             \
  bool alive = true;                                                                   \
  DqItem it;                                                                           \
  for (int rnd = 0, idx; alive && dq_item(A, idx = snake_item(rnd, blockIdx.x, gridDim.x), it); ++rnd)

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_do);
      DQ_ITEMS {
        const KeyTiles kt = key_tiles(A, it.block, attn_length(A, args.lengths, it.b));
        if (kt.n == 0) continue;
        const int hk = it.h / A.G;
        if (!wait_lean(&s.q_free, (itn & 1) ^ 1, cta_abort, limit, AB_Q_FREE)) break;
        mbar_expect_tx(&s.q_full, kTileBytes);
        tma_load_4d(s.q, &tm_q, &s.q_full, 0, it.block * kBlock, it.h, it.b);
        tma_load_4d(s.q + kHalfBytes, &tm_q, &s.q_full, 64, it.block * kBlock, it.h, it.b);
        if (!wait_lean(&s.go_free, (itn & 1) ^ 1, cta_abort, limit, AB_GO_FREE)) break;
        mbar_expect_tx(&s.go_full, kTileBytes);
        tma_load_4d(s.go, &tm_do, &s.go_full, 0, it.block * kBlock, it.h, it.b);
        tma_load_4d(s.go + kHalfBytes, &tm_do, &s.go_full, 64, it.block * kBlock, it.h, it.b);
        for (int u = 0; u < kt.n; ++u, ++g) {
          const int j = kt.tile(u), ks = g % 3, vs = g & 1;
          if (!wait_lean(&s.k_empty[ks], ((g / 3) & 1) ^ 1, cta_abort, limit, AB_K_EMPTY)) { alive = false; break; }
          mbar_expect_tx(&s.k_full[ks], kTileBytes);
          tma_load_4d(s.kring[ks], &tm_k, &s.k_full[ks], 0, j * kBlock, hk, it.b);
          tma_load_4d(s.kring[ks] + kHalfBytes, &tm_k, &s.k_full[ks], 64, j * kBlock, hk, it.b);
          if (!wait_lean(&s.v_empty[vs], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_V_EMPTY)) { alive = false; break; }
          mbar_expect_tx(&s.v_full[vs], kTileBytes);
          tma_load_4d(s.vring[vs], &tm_v, &s.v_full[vs], 0, j * kBlock, hk, it.b);
          tma_load_4d(s.vring[vs] + kHalfBytes, &tm_v, &s.v_full[vs], 64, j * kBlock, hk, it.b);
        }
        ++itn;
      }
    }
  } else if (warp == 1) {
    // G = dO V^T
    const uint64_t d_go = umma_smem_desc(smem_u32(s.go), 16, 1024);
    const uint64_t d_v0 = umma_smem_desc(smem_u32(s.vring[0]), 16, 1024);
    DQ_ITEMS {
      const KeyTiles kt = key_tiles(A, it.block, attn_length(A, args.lengths, it.b));
      if (kt.n == 0) continue;
      if (!wait_lean(&s.go_full, itn & 1, cta_abort, limit, AB_GO_FULL)) break;
      for (int u = 0; u < kt.n; ++u, ++g) {
        if (g > 0 && !wait_lean(&s.g_free, (g - 1) & 1, cta_abort, limit, AB_G_FREE)) { alive = false; break; }
        const uint32_t vs = g & 1;
        if (!wait_lean(&s.v_full[vs], (g >> 1) & 1, cta_abort, limit, AB_V_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        const uint64_t db = d_v0 + vs * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          umma_ss_w(tmem + kDqG, d_go + off, db + off, idesc_kk, k ? 1u : 0u);
        }
        umma_commit_w(&s.v_empty[vs]);
        umma_commit_w(&s.g_full);
      }
      if (!alive) break;
      umma_commit_w(&s.go_free);
      ++itn;
    }
  } else if (warp == 2) {
    // S = Q K^T, ahead of G as far as the two S buffers allow
    const uint64_t d_q = umma_smem_desc(smem_u32(s.q), 16, 1024);
    const uint64_t d_k0 = umma_smem_desc(smem_u32(s.kring[0]), 16, 1024);
    DQ_ITEMS {
      const KeyTiles kt = key_tiles(A, it.block, attn_length(A, args.lengths, it.b));
      if (kt.n == 0) continue;
      if (!wait_lean(&s.q_full, itn & 1, cta_abort, limit, AB_Q_FULL)) break;
      for (int u = 0; u < kt.n; ++u, ++g) {
        const uint32_t ks = g % 3, buf = g & 1;
        if (!wait_lean(&s.sbuf_free[buf], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_SBUF_FREE)) { alive = false; break; }
        if (!wait_lean(&s.k_full[ks], (g / 3) & 1, cta_abort, limit, AB_K_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        const uint64_t db = d_k0 + ks * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          umma_ss_w(tmem + kDqS + 128 * buf, d_q + off, db + off, idesc_kk, k ? 1u : 0u);
        }
        umma_commit_w(&s.s_full[buf]);
      }
      if (!alive) break;
      umma_commit_w(&s.q_free);
      ++itn;
    }
  } else if (warp == 3) {
    // dQ += dS K
    const uint64_t d_k0 = umma_smem_desc(smem_u32(s.kring[0]), kHalfBytes, 1024);
    DQ_ITEMS {
      const KeyTiles kt = key_tiles(A, it.block, attn_length(A, args.lengths, it.b));
      if (kt.n == 0) continue;
      for (int u = 0; u < kt.n; ++u, ++g) {
        const uint32_t ks = g % 3, buf = g & 1;
        if (!wait_lean(&s.w_ready[buf], (g >> 1) & 1, cta_abort, limit, AB_W_READY)) { alive = false; break; }
        if (u == 0 && !wait_lean(&s.acc_free, (itn & 1) ^ 1, cta_abort, limit, AB_ACC_FREE)) { alive = false; break; }
        tc_fence_after_sync();
        const uint64_t db = d_k0 + ks * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          // packed dS: k-steps 0-3 at columns 0-31, k-steps 4-7 at columns 64-95 of the S buffer
          const uint32_t a_col = (k < 4) ? k * 8 : 64 + (k - 4) * 8;
          umma_ts_w(tmem + kDqAcc, tmem + kDqS + 128 * buf + a_col, db + k * (2048 >> 4), idesc_mn, (u | k) ? 1u : 0u);
        }
        umma_commit_w(&s.k_empty[ks]);
        umma_commit_w(&s.sbuf_free[buf]);
      }
      if (!alive) break;
      umma_commit_w(&s.acc_full);
      ++itn;
    }
  } else {
    typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
    const int wg = (warp - 4) >> 2;                  // columns 64*wg .. 64*wg+63
    const int row = ((warp & 3) << 5) + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float sl2 = args.scale_log2;
    DQ_ITEMS {
      const int len = attn_length(A, args.lengths, it.b);
      const KeyTiles kt = key_tiles(A, it.block, len);
      const int i = it.block * kBlock + row, p = i + A.off;
      const float2 st = args.stat[((long long)it.b * A.Hq + it.h) * (A.nqb * kBlock) + i];
      for (int u = 0; u < kt.n; ++u, ++g) {
        const int tile = kt.tile(u), j0 = tile << 7;
        const uint32_t s_tmem = lanes + kDqS + 128 * (g & 1) + wg * 64, g_tmem = lanes + kDqG + wg * 64;
        if (!wait_lean(&s.g_full, g & 1, cta_abort, limit, AB_G_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        uint32_t gv0[32], gv1[32];
        tmem_ld32(g_tmem, gv0);
        tmem_ld32(g_tmem + 32, gv1);
        if (!wait_lean(&s.s_full[g & 1], (g >> 1) & 1, cta_abort, limit, AB_S_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        uint32_t sv0[32], sv1[32];
        tmem_ld32(s_tmem, sv0);
        tmem_ld32(s_tmem + 32, sv1);
        tmem_wait_ld();
        tc_fence_before_sync();
        mbar_arrive(&s.g_free);
        if (tile_masked(A, kt, tile, len)) {
          // outside: S = -inf and G = delta, so that dS = 0 * 0 whatever stood there
          const RowMask mask = row_mask(A, p, j0 + wg * 64, len);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const bool k0 = mask.sees(e), k1 = mask.sees(e + 32);
            sv0[e] = k0 ? sv0[e] : 0xff800000u;
            gv0[e] = k0 ? gv0[e] : __float_as_uint(st.y);
            sv1[e] = k1 ? sv1[e] : 0xff800000u;
            gv1[e] = k1 ? gv1[e] : __float_as_uint(st.y);
          }
          if (wg == 0 && j0 + 127 >= len && len < A.Nk && j0 + row >= len) {
            // key rows behind the sequence hold anything (k_full of this tile is complete: S has been formed)
            zero_tile_row(s.kring[g % 3], row);
          }
          __syncwarp();
          fence_proxy_async_smem();
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float a = ex2_approx(fmaf(__uint_as_float(sv0[2 * e]), sl2, -st.x)) * (__uint_as_float(gv0[2 * e]) - st.y);
          const float b = ex2_approx(fmaf(__uint_as_float(sv0[2 * e + 1]), sl2, -st.x)) * (__uint_as_float(gv0[2 * e + 1]) - st.y);
          pk[e] = pack2<kBf16>(a, b);
        }
        tmem_st16(s_tmem, pk);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float a = ex2_approx(fmaf(__uint_as_float(sv1[2 * e]), sl2, -st.x)) * (__uint_as_float(gv1[2 * e]) - st.y);
          const float b = ex2_approx(fmaf(__uint_as_float(sv1[2 * e + 1]), sl2, -st.x)) * (__uint_as_float(gv1[2 * e + 1]) - st.y);
          pk[e] = pack2<kBf16>(a, b);
        }
        tmem_st16(s_tmem + 16, pk);
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(&s.w_ready[g & 1]);
      }
      if (!alive) break;

      const bool has = kt.n > 0;
      if (has) {
        if (!wait_lean(&s.acc_full, itn & 1, cta_abort, limit, AB_ACC_FULL)) break;
        tc_fence_after_sync();
      }
      const bool some = has && st.x != INFINITY;
      elem_t* out = reinterpret_cast<elem_t*>(args.dq) + it.b * args.dq_strides.b + (long long)i * args.dq_strides.n +
                    it.h * args.dq_strides.h + wg * 64;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        if (has) {
          tmem_ld32(lanes + kDqAcc + wg * 64 + 32 * c, v);
          tmem_wait_ld();
        }
        if (i < A.Nq) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (some) {
              w.x = pack2<kBf16>(__uint_as_float(v[8 * e]) * args.scale, __uint_as_float(v[8 * e + 1]) * args.scale);
              w.y = pack2<kBf16>(__uint_as_float(v[8 * e + 2]) * args.scale, __uint_as_float(v[8 * e + 3]) * args.scale);
              w.z = pack2<kBf16>(__uint_as_float(v[8 * e + 4]) * args.scale, __uint_as_float(v[8 * e + 5]) * args.scale);
              w.w = pack2<kBf16>(__uint_as_float(v[8 * e + 6]) * args.scale, __uint_as_float(v[8 * e + 7]) * args.scale);
            }
            *reinterpret_cast<uint4*>(out + 32 * c + 8 * e) = w;
          }
        }
        __syncwarp();
      }
      if (has) {
        tc_fence_before_sync();
        mbar_arrive(&s.acc_free);
        ++itn;
      }
    }
  }
#undef DQ_ITEMS

  if (s.abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    if (tid == 0) report_error(ctl, kErrBarrierTimeout, -1, -1, blockIdx.x, s.abort_flag);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

cudaError_t launch_attn_dq(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                           const CUtensorMap& tm_do, const AttnBwdArgs& args, int sms, cudaStream_t stream) {
  const int items = args.a.B * args.a.Hq * args.a.nqb, grid = items < sms ? items : sms;
  const int bytes = (int)sizeof(AttnDqSmem) + 1024;
  auto kernel = bf16 ? attn_dq_kernel<true> : attn_dq_kernel<false>;
  static SmemOnce once[2];
  cudaError_t e = once[bf16].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kDqThreads, bytes, stream>>>(tm_q, tm_k, tm_v, tm_do, args);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------
// dK and dV.  Transposed tiles (rows = keys): S^T = K Q^T, G^T = V dO^T, then dV += P^T dO and dK += dS^T Q with P^T
// and dS^T packed over the S^T and G^T columns they were formed from; dV and dK take the other half of TMEM.  One
// buffer each suffices: warp 1 issues dV(q), S(q+1), ... and warp 2 dK(q), G(q+1), ..., so the exponentials of tile
// q + 1 run beside dK(q) and G(q+1), and what the rest of tile q needs beside dV(q) and S(q+1).
// Step q of an item = one block of queries of one of the G heads that share the key head.
// ------------------------------------------------------------------------------------------------------------------
struct AttnDkvSmem {
  alignas(1024) uint8_t k[kTileBytes];
  alignas(1024) uint8_t v[kTileBytes];
  alignas(1024) uint8_t qring[2][kTileBytes];
  alignas(1024) uint8_t gring[2][kTileBytes];      // dO
  alignas(16) float2 stat[2][kBlock];              // with the Q stage
  alignas(8) uint64_t q_full[2];
  uint64_t q_empty[2], go_full[2], go_empty[2];
  uint64_t k_full, k_free, v_full, v_free;
  uint64_t s_full, p_ready, dp_full, ds_ready, dv_full, dv_free, dk_full, dk_free;
  uint32_t tmem_base;
  int abort_flag;
};

constexpr int kDkvThreads = 384;
constexpr int kKvS = 0, kKvG = 128, kKvDv = 256, kKvDk = 384;

template <bool kBf16>
__global__ void __launch_bounds__(kDkvThreads, 1)
attn_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                const AttnBwdArgs args) {
  extern __shared__ uint8_t smem_raw[];
  AttnDkvSmem& s = *reinterpret_cast<AttnDkvSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const AttnShape& A = args.a;
  Control* ctl = &g_attn_bwd_ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned long long limit = args.wait_ns;
  volatile int* cta_abort = &s.abort_flag;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
      mbar_init(&s.go_full[i], 1);
      mbar_init(&s.go_empty[i], 2);
    }
    mbar_init(&s.k_full, 1);
    mbar_init(&s.k_free, 1);
    mbar_init(&s.v_full, 1);
    mbar_init(&s.v_free, 1);
    mbar_init(&s.s_full, 1);
    mbar_init(&s.p_ready, 256);
    mbar_init(&s.dp_full, 1);
    mbar_init(&s.ds_ready, 256);
    mbar_init(&s.dv_full, 1);
    mbar_init(&s.dv_free, 256);
    mbar_init(&s.dk_full, 1);
    mbar_init(&s.dk_free, 256);
    s.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s.tmem_base;
  constexpr int fmt = kBf16 ? 1 : 0;
  constexpr uint32_t idesc_kk = umma_idesc(fmt, 0, 0, 128, 128);
  constexpr uint32_t idesc_mn = umma_idesc(fmt, 0, 1, 128, 128);

  // `g` counts steps, `itn` items that have any; n = steps of the item
#define DKV_ITEMS                                                                                \
  uint32_t g = 0, itn = 0;                                                                       \
  bool alive = true;                                                                             \
  KvItem it;                                                                                     \
  for (int rnd = 0, idx; alive && kv_item(A, args.chunks, idx = snake_item(rnd, blockIdx.x, gridDim.x), it); ++rnd)
#define DKV_GEOMETRY                                                                             \
  const int len = attn_length(A, args.lengths, it.b);                                            \
  const QueryBlocks qb = item_blocks(A, it, len);                                                \
  const int nb = qb.last - qb.first + 1, n = nb > 0 ? nb * A.G : 0;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_do);
      DKV_ITEMS {
        DKV_GEOMETRY
        if (n == 0) continue;
        if (!wait_lean(&s.k_free, (itn & 1) ^ 1, cta_abort, limit, AB_K_EMPTY)) break;
        mbar_expect_tx(&s.k_full, kTileBytes);
        tma_load_4d(s.k, &tm_k, &s.k_full, 0, it.tile * kBlock, it.hk, it.b);
        tma_load_4d(s.k + kHalfBytes, &tm_k, &s.k_full, 64, it.tile * kBlock, it.hk, it.b);
        for (int q = 0; q < n; ++q, ++g) {
          const int h = it.hk * A.G + q / nb, blk = qb.first + q % nb, st = g & 1;
          if (!wait_lean(&s.q_empty[st], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_Q_FREE)) { alive = false; break; }
          mbar_expect_tx(&s.q_full[st], kTileBytes + kBlock * 8);
          tma_load_4d(s.qring[st], &tm_q, &s.q_full[st], 0, blk * kBlock, h, it.b);
          tma_load_4d(s.qring[st] + kHalfBytes, &tm_q, &s.q_full[st], 64, blk * kBlock, h, it.b);
          bulk_load(s.stat[st], args.stat + (((long long)it.b * A.Hq + h) * A.nqb + blk) * kBlock, kBlock * 8, &s.q_full[st]);
          if (q == 0) {
            if (!wait_lean(&s.v_free, (itn & 1) ^ 1, cta_abort, limit, AB_V_EMPTY)) { alive = false; break; }
            mbar_expect_tx(&s.v_full, kTileBytes);
            tma_load_4d(s.v, &tm_v, &s.v_full, 0, it.tile * kBlock, it.hk, it.b);
            tma_load_4d(s.v + kHalfBytes, &tm_v, &s.v_full, 64, it.tile * kBlock, it.hk, it.b);
          }
          if (!wait_lean(&s.go_empty[st], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_GO_FREE)) { alive = false; break; }
          mbar_expect_tx(&s.go_full[st], kTileBytes);
          tma_load_4d(s.gring[st], &tm_do, &s.go_full[st], 0, blk * kBlock, h, it.b);
          tma_load_4d(s.gring[st] + kHalfBytes, &tm_do, &s.go_full[st], 64, blk * kBlock, h, it.b);
        }
        ++itn;
      }
    }
  } else if (warp == 1) {
    // S^T(0); then dV(q), S^T(q+1)
    const uint64_t d_k = umma_smem_desc(smem_u32(s.k), 16, 1024);
    const uint64_t d_q0 = umma_smem_desc(smem_u32(s.qring[0]), 16, 1024);
    const uint64_t d_g0 = umma_smem_desc(smem_u32(s.gring[0]), kHalfBytes, 1024);
    DKV_ITEMS {
      DKV_GEOMETRY
      if (n == 0) continue;
      if (!wait_lean(&s.k_full, itn & 1, cta_abort, limit, AB_K_FULL)) break;
      auto issue_s = [&](uint32_t gq) -> bool {
        if (!wait_lean(&s.q_full[gq & 1], (gq >> 1) & 1, cta_abort, limit, AB_Q_FULL)) return false;
        tc_fence_after_sync();
        const uint64_t db = d_q0 + (gq & 1) * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          umma_ss_w(tmem + kKvS, d_k + off, db + off, idesc_kk, k ? 1u : 0u);
        }
        umma_commit_w(&s.s_full);
        return true;
      };
      if (!issue_s(g)) break;
      for (int q = 0; q < n; ++q, ++g) {
        if (!wait_lean(&s.p_ready, g & 1, cta_abort, limit, AB_P_READY)) { alive = false; break; }
        if (q == 0 && !wait_lean(&s.dv_free, (itn & 1) ^ 1, cta_abort, limit, AB_ACC_FREE)) { alive = false; break; }
        if (!wait_lean(&s.go_full[g & 1], (g >> 1) & 1, cta_abort, limit, AB_GO_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        const uint64_t db = d_g0 + (g & 1) * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t a_col = (k < 4) ? k * 8 : 64 + (k - 4) * 8;
          umma_ts_w(tmem + kKvDv, tmem + kKvS + a_col, db + k * (2048 >> 4), idesc_mn, (q | k) ? 1u : 0u);
        }
        umma_commit_w(&s.go_empty[g & 1]);
        if (q + 1 < n && !issue_s(g + 1)) { alive = false; break; }
      }
      if (!alive) break;
      umma_commit_w(&s.k_free);
      umma_commit_w(&s.dv_full);
      ++itn;
    }
  } else if (warp == 2) {
    // G^T(0); then dK(q), G^T(q+1)
    const uint64_t d_v = umma_smem_desc(smem_u32(s.v), 16, 1024);
    const uint64_t d_g0 = umma_smem_desc(smem_u32(s.gring[0]), 16, 1024);
    const uint64_t d_q0 = umma_smem_desc(smem_u32(s.qring[0]), kHalfBytes, 1024);
    DKV_ITEMS {
      DKV_GEOMETRY
      if (n == 0) continue;
      if (!wait_lean(&s.v_full, itn & 1, cta_abort, limit, AB_V_FULL)) break;
      auto issue_g = [&](uint32_t gq) -> bool {
        if (!wait_lean(&s.go_full[gq & 1], (gq >> 1) & 1, cta_abort, limit, AB_GO_FULL)) return false;
        tc_fence_after_sync();
        const uint64_t db = d_g0 + (gq & 1) * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
          umma_ss_w(tmem + kKvG, d_v + off, db + off, idesc_kk, k ? 1u : 0u);
        }
        umma_commit_w(&s.go_empty[gq & 1]);
        umma_commit_w(&s.dp_full);
        return true;
      };
      if (!issue_g(g)) break;
      for (int q = 0; q < n; ++q, ++g) {
        if (!wait_lean(&s.ds_ready, g & 1, cta_abort, limit, AB_DS_READY)) { alive = false; break; }
        if (q == 0 && !wait_lean(&s.dk_free, (itn & 1) ^ 1, cta_abort, limit, AB_ACC_FREE)) { alive = false; break; }
        tc_fence_after_sync();
        const uint64_t db = d_q0 + (g & 1) * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t a_col = (k < 4) ? k * 8 : 64 + (k - 4) * 8;
          umma_ts_w(tmem + kKvDk, tmem + kKvG + a_col, db + k * (2048 >> 4), idesc_mn, (q | k) ? 1u : 0u);
        }
        umma_commit_w(&s.q_empty[g & 1]);      // S^T(q) was complete before dS^T(q) could be formed
        if (q + 1 < n && !issue_g(g + 1)) { alive = false; break; }
      }
      if (!alive) break;
      umma_commit_w(&s.v_free);
      umma_commit_w(&s.dk_full);
      ++itn;
    }
  } else if (warp >= 4) {
    typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
    const int wg = (warp - 4) >> 2;                  // query columns 64*wg .. 64*wg+63
    const int row = ((warp & 3) << 5) + lane;        // key row
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_tmem = lanes + kKvS + wg * 64, g_tmem = lanes + kKvG + wg * 64;
    const float sl2 = args.scale_log2;
    DKV_ITEMS {
      DKV_GEOMETRY
      const int j = it.tile * kBlock + row;
      const bool key = j < len;
      const int j0 = it.tile * kBlock;
      for (int q = 0; q < n; ++q, ++g) {
        const int st = g & 1;
        const int p0 = (qb.first + q % nb) * kBlock + A.off;        // position of the block's first query
        const float2* stat = s.stat[st] + wg * 64;
        const bool masked = block_masked(A, j0, p0, len);
        const ColMask mask = col_mask(A, j, p0 + wg * 64, len);
        if (!wait_lean(&s.s_full, g & 1, cta_abort, limit, AB_S_FULL)) { alive = false; break; }
        // (for this thread's own reads of the statistics: the load that brought Q brought them)
        if (!wait_lean(&s.q_full[st], (g >> 1) & 1, cta_abort, limit, AB_Q_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        uint32_t v0[32], v1[32];
        tmem_ld32(s_tmem, v0);
        tmem_ld32(s_tmem + 32, v1);
        tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            v0[e] = mask.sees(e) ? v0[e] : 0xff800000u;
            v1[e] = mask.sees(e + 32) ? v1[e] : 0xff800000u;
          }
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float4 t = *reinterpret_cast<const float4*>(stat + 2 * e);
          const float a = ex2_approx(fmaf(__uint_as_float(v0[2 * e]), sl2, -t.x));
          const float b = ex2_approx(fmaf(__uint_as_float(v0[2 * e + 1]), sl2, -t.z));
          v0[2 * e] = __float_as_uint(a);
          v0[2 * e + 1] = __float_as_uint(b);
          pk[e] = pack2<kBf16>(a, b);
        }
        tmem_st16(s_tmem, pk);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float4 t = *reinterpret_cast<const float4*>(stat + 32 + 2 * e);
          const float a = ex2_approx(fmaf(__uint_as_float(v1[2 * e]), sl2, -t.x));
          const float b = ex2_approx(fmaf(__uint_as_float(v1[2 * e + 1]), sl2, -t.z));
          v1[2 * e] = __float_as_uint(a);
          v1[2 * e + 1] = __float_as_uint(b);
          pk[e] = pack2<kBf16>(a, b);
        }
        tmem_st16(s_tmem + 16, pk);
        tmem_wait_st();
        // Query rows behind the sequence hold anything, and 0 * NaN is not 0: they become zero in Q and dO before
        // the products that sum over them.  S^T and G^T, which read them as columns, are complete by then.
        const bool stale = p0 + 127 >= len && len < A.Nk;
        if (stale) {
          if (!wait_lean(&s.dp_full, g & 1, cta_abort, limit, AB_DP_FULL)) { alive = false; break; }
          if (wg == 0 && p0 + row >= len) {
            zero_tile_row(s.qring[st], row);
            zero_tile_row(s.gring[st], row);
          }
          __syncwarp();
          fence_proxy_async_smem();
        }
        tc_fence_before_sync();
        mbar_arrive(&s.p_ready);
        if (!stale && !wait_lean(&s.dp_full, g & 1, cta_abort, limit, AB_DP_FULL)) { alive = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t gv[16], w[8];
          tmem_ld16(g_tmem + 16 * c, gv);
          tmem_wait_ld();
          const uint32_t* pv = (c < 2) ? v0 + 16 * c : v1 + 16 * (c - 2);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 t = *reinterpret_cast<const float4*>(stat + 16 * c + 2 * e);
            float a = __uint_as_float(pv[2 * e]) * (__uint_as_float(gv[2 * e]) - t.y);
            float b = __uint_as_float(pv[2 * e + 1]) * (__uint_as_float(gv[2 * e + 1]) - t.w);
            if (masked) {
              const int x = 16 * c + 2 * e;
              a = mask.sees(x) ? a : 0.f;
              b = mask.sees(x + 1) ? b : 0.f;
            }
            w[e] = pack2<kBf16>(a, b);
          }
          tmem_st8(g_tmem + 8 * c, w);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(&s.ds_ready);
      }
      if (!alive) break;

      // ---- epilogue: this thread's key row, 64 of the 128 columns of dV and of dK ----
      const bool has = n > 0;
      const bool sums = args.chunks > 0 && it.tile == 0 && j < A.S;     // first keys: fp32 sums, joined afterwards
      const bool mine = j < A.Nk && (it.chunk < 0 || j < A.S);
#pragma unroll
      for (int which = 0; which < 2; ++which) {       // 0: dV, 1: dK
        if (has) {
          if (!wait_lean(which ? &s.dk_full : &s.dv_full, itn & 1, cta_abort, limit, AB_ACC_FULL)) {
            alive = false;
            break;
          }
          tc_fence_after_sync();
        }
        const float f = which ? args.scale : 1.f;
        const Strides& sd = which ? args.dk_strides : args.dv_strides;
        elem_t* out = reinterpret_cast<elem_t*>(which ? args.dk : args.dv) + it.b * sd.b + (long long)j * sd.n +
                      it.hk * sd.h + wg * 64;
        float* part = args.partial + ((((long long)(it.b * A.Hkv + it.hk) * (1 + args.chunks) + it.chunk + 1) * 2 + which) * A.S + j) * 128 +
                      wg * 64;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[32];
          if (has) {
            tmem_ld32(lanes + (which ? kKvDk : kKvDv) + wg * 64 + 32 * c, v);
            tmem_wait_ld();
          }
          if (!has || !key) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0u;
          }
          if (mine && sums) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<float4*>(part + 32 * c + 4 * e) =
                  make_float4(__uint_as_float(v[4 * e]) * f, __uint_as_float(v[4 * e + 1]) * f,
                              __uint_as_float(v[4 * e + 2]) * f, __uint_as_float(v[4 * e + 3]) * f);
          } else if (mine) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(out + 32 * c + 8 * e) =
                  make_uint4(pack2<kBf16>(__uint_as_float(v[8 * e]) * f, __uint_as_float(v[8 * e + 1]) * f),
                             pack2<kBf16>(__uint_as_float(v[8 * e + 2]) * f, __uint_as_float(v[8 * e + 3]) * f),
                             pack2<kBf16>(__uint_as_float(v[8 * e + 4]) * f, __uint_as_float(v[8 * e + 5]) * f),
                             pack2<kBf16>(__uint_as_float(v[8 * e + 6]) * f, __uint_as_float(v[8 * e + 7]) * f));
          }
          __syncwarp();
        }
        if (has) {
          tc_fence_before_sync();
          mbar_arrive(which ? &s.dk_free : &s.dv_free);
        }
      }
      if (has) ++itn;
    }
  }
#undef DKV_ITEMS
#undef DKV_GEOMETRY

  if (s.abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    if (tid == 0) report_error(ctl, kErrBarrierTimeout, -1, -1, blockIdx.x, s.abort_flag);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// The first keys' rows: the tile's own sums and those of the chunks, added in order.
template <bool kBf16>
__global__ void __launch_bounds__(128) attn_first_keys_kernel(const AttnBwdArgs args) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  const AttnShape& A = args.a;
  const int j = blockIdx.x, which = blockIdx.y, bh = blockIdx.z, b = bh / A.Hkv, hk = bh % A.Hkv;
  const float* p = args.partial + (((long long)bh * (1 + args.chunks) * 2 + which) * A.S + j) * 128 + threadIdx.x;
  const long long step = (long long)2 * A.S * 128;
  float sum = 0.f;
#pragma unroll 8
  for (int c = 0; c <= args.chunks; ++c) sum += p[c * step];
  const Strides& sd = which ? args.dk_strides : args.dv_strides;
  elem_t* out = reinterpret_cast<elem_t*>(which ? args.dk : args.dv) + b * sd.b + (long long)j * sd.n + hk * sd.h;
  if constexpr (kBf16) out[threadIdx.x] = __float2bfloat16_rn(sum);
  else out[threadIdx.x] = __float2half_rn(sum);
}

cudaError_t launch_attn_dkv(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                            const CUtensorMap& tm_do, const AttnBwdArgs& args, int sms, cudaStream_t stream) {
  const AttnShape& a = args.a;
  const int items = kv_items(a), grid = items < sms ? items : sms;
  const int bytes = (int)sizeof(AttnDkvSmem) + 1024;
  auto kernel = bf16 ? attn_dkv_kernel<true> : attn_dkv_kernel<false>;
  static SmemOnce once[2];
  cudaError_t e = once[bf16].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kDkvThreads, bytes, stream>>>(tm_q, tm_k, tm_v, tm_do, args);
  if ((e = cudaGetLastError()) != cudaSuccess || args.chunks == 0) return e;
  const dim3 sum_grid(a.S < a.Nk ? a.S : a.Nk, 2, a.B * a.Hkv);
  if (bf16) attn_first_keys_kernel<true><<<sum_grid, 128, 0, stream>>>(args);
  else attn_first_keys_kernel<false><<<sum_grid, 128, 0, stream>>>(args);
  return cudaGetLastError();
}

cudaError_t attn_bwd_status(cudaStream_t stream, int out[8]) { return take_status(&g_attn_bwd_ctl, stream, out); }

}  // namespace lucid
