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
// Row statistics {log2(sum of exponentials / unit), -delta / unit}, delta = dO . (O + what its rounding took off): as the dK/dV
// kernel wants them, whose weights are `unit` times P (below).  Reads each once, bound by HBM.  Eight lanes per row, four rows
// per warp and round.
// ------------------------------------------------------------------------------------------------------------------
// P^T enters its product times 2^kWeightBits, and dV leaves divided by that: fp16 loses bits of weights below 2^-14, which is
// what a row of some ten thousand keys has; none is above 1 but for the rounding of very large scores, for which there is room.
// dS, which has no such bound, is formed from them with its other
// factor divided (part of an fma), and rounded as it is.  (Products with the unit in the dK/dV kernel took it 4 % longer.)
template <bool kBf16>
constexpr int kWeightBits = kBf16 ? 0 : 12;

constexpr int kStatRows = 8;             // rows of a warp (4, 16 and 32: 3, 3 and 10 % slower at 64k)

template <bool kBf16>
__global__ void __launch_bounds__(256) attn_stat_kernel(const AttnStatArgs args) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  launch_dependents();
  const AttnShape& A = args.a;
  const int lane = threadIdx.x & 31, ch = lane & 7;
  const long long base = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * kStatRows;     // of the padded rows of all heads
  if (base >= (long long)A.B * A.Hq * A.nqb * kBlock) return;
  const int rows = A.nqb * kBlock;
  const int i0 = (int)(base % rows), bh = (int)(base / rows), b = bh / A.Hq, h = bh % A.Hq;
  const elem_t* o = reinterpret_cast<const elem_t*>(args.out) + b * args.out_strides.b + h * args.out_strides.h + ch * 8;
  const elem_t* g = reinterpret_cast<const elem_t*>(args.dout) + b * args.dout_strides.b + h * args.dout_strides.h + ch * 8;
  const long long tile = base >> 7;
  const int rest_step = rest_rows(A) * 8;
  const elem_t* rest = reinterpret_cast<const elem_t*>(args.rest) + tile * 16 * rest_step + ch * rest_step;
#pragma unroll
  for (int y = 0; y < kStatRows / 4; ++y) {
    const int r = 4 * y + (lane >> 3), i = i0 + r;
    float d = 0.f;
    if (i < A.Nq) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 ov = *reinterpret_cast<const uint4*>(o + (long long)i * args.out_strides.n + 64 * c);
        const uint4 gv = *reinterpret_cast<const uint4*>(g + (long long)i * args.dout_strides.n + 64 * c);
        uint4 rv = make_uint4(0, 0, 0, 0);
        if (args.rest) rv = *reinterpret_cast<const uint4*>(rest + 8 * c * rest_step + (i & 127) * 8);
        const uint32_t ow[4] = {ov.x, ov.y, ov.z, ov.w}, gw[4] = {gv.x, gv.y, gv.z, gv.w}, rw[4] = {rv.x, rv.y, rv.z, rv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = unpack2<kBf16>(ow[e]), q = unpack2<kBf16>(gw[e]), l = unpack2<kBf16>(rw[e]);
          d += (a.x + l.x) * q.x + (a.y + l.y) * q.y;
        }
      }
    }
#pragma unroll
    for (int m = 4; m > 0; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
    if (ch == 0) {
      const float lse = i < A.Nq ? args.lse[(long long)bh * A.Nq + i] : -INFINITY;
      const bool weight = lse != -INFINITY;                // (a row without weight: P = 0 from +infinity)
      float* st = args.stat + tile * (2 * kBlock) + (i & 127);
      st[0] = weight ? lse * kLog2e - kWeightBits<kBf16> : INFINITY;
      st[kBlock] = weight ? -d / (1 << kWeightBits<kBf16>) : 0.f;
    }
  }
}

cudaError_t launch_attn_stat(bool bf16, const AttnStatArgs& args, cudaStream_t stream) {
  const long long rows = (long long)args.a.B * args.a.Hq * args.a.nqb * kBlock;
  const unsigned grid = (unsigned)((rows + 8 * kStatRows - 1) / (8 * kStatRows));
  if (bf16) attn_stat_kernel<true><<<grid, 256, 0, stream>>>(args);
  else attn_stat_kernel<false><<<grid, 256, 0, stream>>>(args);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------------------------------------
// Shared by both kernels
// ------------------------------------------------------------------------------------------------------------------
enum AttnBwdBar : int {
  AB_K_FULL = 501, AB_K_EMPTY, AB_V_FULL, AB_V_EMPTY, AB_Q_FULL, AB_Q_FREE, AB_GO_FULL, AB_GO_FREE, AB_S_FULL, AB_G_FULL,
  AB_G_FREE, AB_W_READY, AB_SBUF_FREE, AB_ACC_FULL, AB_ACC_FREE, AB_P_READY, AB_DS_READY, AB_DP_FULL, AB_SLOT_FULL,
  AB_SLOT_FREE, AB_PANEL
};

constexpr int kBwThreads = 384;

// A whole group of eight products: A K-major in shared memory, B K-major
__device__ __forceinline__ void issue_kk(uint32_t d_tmem, uint64_t da, uint64_t db, uint32_t idesc) {
  if (elect_one()) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
      umma_ss(d_tmem, da + off, db + off, idesc, k ? 1u : 0u);
    }
  }
}
// A packed in tensor memory (k-steps 0-3 at columns 0-31, 4-7 at columns 64-95), B with rows = k
__device__ __forceinline__ void issue_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t idesc, uint32_t add) {
  if (elect_one()) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      umma_ts(d_tmem, a_tmem + (k < 4 ? 8 * k : 32 + 8 * k), db + k * (2048 >> 4), idesc, k ? 1u : add);
  }
}

// The same in two parts: k-steps 0, 1, 4, 5 (the first 32 columns of both halves' threads), then 2, 3, 6, 7
template <int kPart>
__device__ __forceinline__ void issue_ts_part(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t idesc, uint32_t add) {
  if (elect_one()) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int k = 2 * kPart + (x & 1) + 4 * (x >> 1);
      umma_ts(d_tmem, a_tmem + (k < 4 ? 8 * k : 32 + 8 * k), db + k * (2048 >> 4), idesc, x ? 1u : add);
    }
  }
}

// 64 fp32 columns of this thread's row, from tensor memory, times `f`, as 16-bit values into the warp's panel (32 rows x 64
// columns; zeros unless `some`); `loaded` is called when the tensor memory has been read.
template <bool kBf16, class Loaded>
__device__ __forceinline__ void stage_row(uint32_t t_addr, bool some, float f, uint8_t* panel, int lane, Loaded loaded) {
  uint32_t o[2][32];
  tmem_ld32(t_addr, o[0]);
  tmem_ld32(t_addr + 32, o[1]);
  tmem_wait_ld();
  loaded();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t* v = o[e >> 2] + 8 * (e & 3);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (some) {
      w.x = pack2<kBf16>(__uint_as_float(v[0]) * f, __uint_as_float(v[1]) * f);
      w.y = pack2<kBf16>(__uint_as_float(v[2]) * f, __uint_as_float(v[3]) * f);
      w.z = pack2<kBf16>(__uint_as_float(v[4]) * f, __uint_as_float(v[5]) * f);
      w.w = pack2<kBf16>(__uint_as_float(v[6]) * f, __uint_as_float(v[7]) * f);
    }
    *reinterpret_cast<uint4*>(panel + sw128_off(lane, e)) = w;
  }
  __syncwarp();
}
// The panel's rows to memory, four whole lines per instruction; row r is written where lo <= r < hi.  `zero`: zeros instead.
template <class elem_t>
__device__ __forceinline__ void store_panel(const uint8_t* panel, bool zero, elem_t* out, long long row_stride, int lo, int hi, int lane) {
#pragma unroll 4
  for (int y = 0; y < 8; ++y) {
    const int r = 4 * y + (lane >> 3);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (!zero) w = *reinterpret_cast<const uint4*>(panel + sw128_off(r, lane & 7));
    if (r >= lo && r < hi) *reinterpret_cast<uint4*>(out + r * row_stride + (lane & 7) * 8) = w;
  }
  __syncwarp();
}

// ------------------------------------------------------------------------------------------------------------------
// dQ.  Per key tile three products (S, dO V^T, dS K) against one exponential per pair: about balanced.  Warp roles
// (384 threads): warp 0 producer (and works out the items), warps 1, 2, 3 issue G = dO V^T, S = Q K^T and dS K (one warp per
// product stream), warps 4-11 form dS, 64 columns each group, over S columns they have consumed.  TMEM: S twice, G, dQ.
// Results leave through a stage of the V ring that the producer passes over at the end of an item (no product reads it
// then): per warp a panel of 32 rows x 64 columns, read back in rows.
// ------------------------------------------------------------------------------------------------------------------
struct DqSlot {
  int n;                 // key tiles, -1: no more items
  int b, h, block, len, sink, lo, p_lo, p_hi;
  __device__ __forceinline__ KeyTiles list() const {
    KeyTiles t;
    t.n = n;
    t.sink = sink;
    t.lo = lo;
    t.p_lo = p_lo;
    t.p_hi = p_hi;
    return t;
  }
};

struct AttnDqSmem {
  alignas(1024) uint8_t q[kTileBytes];
  alignas(1024) uint8_t go[kTileBytes];            // dO
  alignas(1024) uint8_t kring[3][kTileBytes];
  alignas(1024) uint8_t vring[2][kTileBytes];
  alignas(16) float stat[2][2 * kBlock];           // with the slot: the rows' statistics
  alignas(8) uint64_t k_full[3];
  uint64_t k_empty[3], v_full[2], v_empty[2], slot_full[2], slot_free[2];
  uint64_t q_full, q_free, go_full, go_free, panel_done;
  uint64_t s_full[2], g_full, g_free, w_ready[2], sbuf_free[2], acc_full, acc_free;
  DqSlot slot[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(AttnDqSmem) <= 232448, "shared memory of a CTA");

constexpr int kDqS = 0, kDqG = 256, kDqAcc = 384;

// The V ring's stages in turn, with one passed over behind every item that has tiles
struct VTurn {
  uint32_t at = 0, used0 = 0, used1 = 0;      // stage of the next use; loads of each stage so far
  __device__ __forceinline__ uint32_t stage() const { return at & 1; }
  __device__ __forceinline__ uint32_t used() const { return (at & 1) ? used1 : used0; }
  __device__ __forceinline__ void use() {
    if (at & 1) ++used1;
    else ++used0;
    ++at;
  }
};

template <bool kBf16>
__global__ void __launch_bounds__(kBwThreads, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
               const AttnBwdArgs args) {
  // (no room to round the base up: the kernel has no static shared memory, and the window starts on 1 KiB)
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  AttnDqSmem& s = *reinterpret_cast<AttnDqSmem*>(smem_raw);
  const AttnShape& A = args.a;
  Control* ctl = &g_attn_bwd_ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned long long limit = args.wait_ns;
  volatile int* cta_abort = &s.abort_flag;

  if (smem_u32(smem_raw) & 1023) {       // (operand tiles would be misread)
    if (tid == 0) report_error(ctl, kErrAborted, -1, -1, blockIdx.x, 0);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.slot_full[i], 1);
      mbar_init(&s.slot_free[i], 11);      // three issuing and eight dS warps
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.w_ready[i], 256);
      mbar_init(&s.sbuf_free[i], 1);
    }
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_free, 1);
    mbar_init(&s.go_full, 1);
    mbar_init(&s.go_free, 1);
    mbar_init(&s.panel_done, 8);
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
  // The statistics' kernel may still be running until here.  From here on the dK/dV kernel, which needs them too but
  // nothing of this one, may take SMs that have no items left.
  wait_for_primary();
  launch_dependents();
  const uint32_t tmem = s.tmem_base;
  constexpr int fmt = kBf16 ? 1 : 0;
  constexpr uint32_t idesc_kk = umma_idesc(fmt, 0, 0, 128, 128);
  constexpr uint32_t idesc_mn = umma_idesc(fmt, 0, 1, 128, 128);

  // `g` counts tiles, `itn` items that have any, over all items of this CTA
  uint32_t g = 0, itn = 0, slots = 0;
  bool alive = true;
  auto next = [&]() -> const DqSlot* {
    if (!alive || !wait_lean(&s.slot_full[slots & 1], (slots >> 1) & 1, cta_abort, limit, AB_SLOT_FULL)) return nullptr;
    const DqSlot* slot = &s.slot[slots & 1];
    return slot->n < 0 ? nullptr : slot;
  };
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.slot_free[slots & 1]);
    ++slots;
  };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_do);
      VTurn vt;
      int passed = -1;           // the stage the previous item's results leave through
      const int per = A.B * A.Hq;
      for (int rnd = 0; alive; ++rnd, ++slots) {
        const int idx = snake_item(rnd, blockIdx.x, gridDim.x), sl = rnd & 1;
        if (!wait_lane(&s.slot_free[sl], ((rnd >> 1) & 1) ^ 1, cta_abort, limit, AB_SLOT_FREE)) break;
        DqSlot& x = s.slot[sl];
        if (idx >= per * A.nqb) {
          x.n = -1;
          mbar_arrive(&s.slot_full[sl]);
          break;
        }
        // blocks from the last to the first (under full causality the last ones take longest), heads side by side
        const int block = A.nqb - 1 - idx / per, r = idx % per, b = r / A.Hq, h = r % A.Hq, hk = h / A.G;
        const int len = attn_length(A, args.lengths, b);
        const KeyTiles kt = key_tiles(A, block, len);
        x.n = kt.n;
        x.b = b;
        x.h = h;
        x.block = block;
        x.len = len;
        x.sink = kt.sink;
        x.lo = kt.lo;
        x.p_lo = kt.p_lo;
        x.p_hi = kt.p_hi;
        mbar_expect_tx(&s.slot_full[sl], 2 * kBlock * 4);
        bulk_load(s.stat[sl], args.stat + (((long long)b * A.Hq + h) * A.nqb + block) * (2 * kBlock), 2 * kBlock * 4, &s.slot_full[sl]);
        if (kt.n == 0) continue;
        if (!wait_lane(&s.q_free, (itn & 1) ^ 1, cta_abort, limit, AB_Q_FREE)) break;
        mbar_expect_tx(&s.q_full, kTileBytes);
        tma_load_4d(s.q, &tm_q, &s.q_full, 0, block * kBlock, h, b);
        tma_load_4d(s.q + kHalfBytes, &tm_q, &s.q_full, 64, block * kBlock, h, b);
        if (!wait_lane(&s.go_free, (itn & 1) ^ 1, cta_abort, limit, AB_GO_FREE)) break;
        mbar_expect_tx(&s.go_full, kTileBytes);
        tma_load_4d(s.go, &tm_do, &s.go_full, 0, block * kBlock, h, b);
        tma_load_4d(s.go + kHalfBytes, &tm_do, &s.go_full, 64, block * kBlock, h, b);
        for (int u = 0; u < kt.n; ++u, ++g) {
          const int j = kt.tile(u), ks = g % 3, vs = vt.stage();
          if (!wait_lane(&s.k_empty[ks], ((g / 3) & 1) ^ 1, cta_abort, limit, AB_K_EMPTY)) { alive = false; break; }
          mbar_expect_tx(&s.k_full[ks], kTileBytes);
          tma_load_4d(s.kring[ks], &tm_k, &s.k_full[ks], 0, j * kBlock, hk, b);
          tma_load_4d(s.kring[ks] + kHalfBytes, &tm_k, &s.k_full[ks], 64, j * kBlock, hk, b);
          if (!wait_lane(&s.v_empty[vs], (vt.used() & 1) ^ 1, cta_abort, limit, AB_V_EMPTY)) { alive = false; break; }
          if (vs == passed) {
            // (itn items have passed a stage so far; the last of them has to be through with it)
            if (!wait_lane(&s.panel_done, (itn - 1) & 1, cta_abort, limit, AB_PANEL)) { alive = false; break; }
            passed = -1;
          }
          mbar_expect_tx(&s.v_full[vs], kTileBytes);
          tma_load_4d(s.vring[vs], &tm_v, &s.v_full[vs], 0, j * kBlock, hk, b);
          tma_load_4d(s.vring[vs] + kHalfBytes, &tm_v, &s.v_full[vs], 64, j * kBlock, hk, b);
          vt.use();
        }
        // (an item of one tile that did not come to the stage the item before passed over: wait here, one at a time)
        if (alive && passed >= 0 && !wait_lane(&s.panel_done, (itn - 1) & 1, cta_abort, limit, AB_PANEL)) break;
        passed = vt.stage();
        ++vt.at;
        ++itn;
      }
    }
  } else if (warp == 1) {
    // G = dO V^T
    const uint64_t d_go = umma_smem_desc(smem_u32(s.go), 16, 1024);
    const uint64_t d_v0 = umma_smem_desc(smem_u32(s.vring[0]), 16, 1024);
    VTurn vt;
    while (const DqSlot* x = next()) {
      const int n = x->n;
      done();
      if (n == 0) continue;
      if (!wait_lean(&s.go_full, itn & 1, cta_abort, limit, AB_GO_FULL)) break;
      for (int u = 0; u < n; ++u, ++g) {
        if (g > 0 && !wait_lean(&s.g_free, (g - 1) & 1, cta_abort, limit, AB_G_FREE)) { alive = false; break; }
        const uint32_t vs = vt.stage();
        if (!wait_lean(&s.v_full[vs], vt.used() & 1, cta_abort, limit, AB_V_FULL)) { alive = false; break; }
        vt.use();
        tc_fence_after_sync();
        issue_kk(tmem + kDqG, d_go, d_v0 + vs * (kTileBytes >> 4), idesc_kk);
        umma_commit_w(&s.v_empty[vs]);
        umma_commit_w(&s.g_full);
      }
      if (!alive) break;
      ++vt.at;
      umma_commit_w(&s.go_free);
      ++itn;
    }
  } else if (warp == 2) {
    // S = Q K^T, ahead of G as far as the two S buffers allow
    const uint64_t d_q = umma_smem_desc(smem_u32(s.q), 16, 1024);
    const uint64_t d_k0 = umma_smem_desc(smem_u32(s.kring[0]), 16, 1024);
    while (const DqSlot* x = next()) {
      const int n = x->n;
      done();
      if (n == 0) continue;
      if (!wait_lean(&s.q_full, itn & 1, cta_abort, limit, AB_Q_FULL)) break;
      for (int u = 0; u < n; ++u, ++g) {
        const uint32_t ks = g % 3, buf = g & 1;
        if (!wait_lean(&s.sbuf_free[buf], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_SBUF_FREE)) { alive = false; break; }
        if (!wait_lean(&s.k_full[ks], (g / 3) & 1, cta_abort, limit, AB_K_FULL)) { alive = false; break; }
        tc_fence_after_sync();
        issue_kk(tmem + kDqS + 128 * buf, d_q, d_k0 + ks * (kTileBytes >> 4), idesc_kk);
        umma_commit_w(&s.s_full[buf]);
      }
      if (!alive) break;
      umma_commit_w(&s.q_free);
      ++itn;
    }
  } else if (warp == 3) {
    // dQ += dS K
    const uint64_t d_k0 = umma_smem_desc(smem_u32(s.kring[0]), kHalfBytes, 1024);
    while (const DqSlot* x = next()) {
      const int n = x->n;
      done();
      if (n == 0) continue;
      for (int u = 0; u < n; ++u, ++g) {
        const uint32_t ks = g % 3, buf = g & 1;
        if (!wait_lean(&s.w_ready[buf], (g >> 1) & 1, cta_abort, limit, AB_W_READY)) { alive = false; break; }
        if (u == 0 && !wait_lean(&s.acc_free, (itn & 1) ^ 1, cta_abort, limit, AB_ACC_FREE)) { alive = false; break; }
        tc_fence_after_sync();
        issue_ts(tmem + kDqAcc, tmem + kDqS + 128 * buf, d_k0 + ks * (kTileBytes >> 4), idesc_mn, u ? 1u : 0u);
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
    const unsigned long long sl22 = f32x2(sl2, sl2);
    uint32_t v_at = 0;                               // the V ring's turn, for the stage that is passed over
    while (const DqSlot* x = next()) {
      const KeyTiles kt = x->list();
      const int len = x->len, block = x->block, b = x->b, h = x->h;
      const int i = block * kBlock + row, p = i + A.off;
      // (a query that sees one key has dS = 0 exactly, not the difference of two nearly equal sums)
      const float lse2 = sees_one(A, p) ? INFINITY : s.stat[slots & 1][row] + kWeightBits<kBf16>;
      const float delta = -s.stat[slots & 1][kBlock + row] * (1 << kWeightBits<kBf16>);
      done();
      const unsigned long long nlse2 = f32x2(-lse2, -lse2), ndelta = f32x2(-delta, -delta);
      for (int u = 0; u < kt.n; ++u, ++g) {
        const int tile = kt.tile(u), j0 = tile << 7;
        const uint32_t s_tmem = lanes + kDqS + 128 * (g & 1) + wg * 64, g_tmem = lanes + kDqG + wg * 64;
        auto form = [&](auto some_masked) -> bool {
          constexpr bool kMasked = decltype(some_masked)::value;
          if (!wait_lean(&s.g_full, g & 1, cta_abort, limit, AB_G_FULL)) return false;
          tc_fence_after_sync();
          uint32_t gv[2][32], sv[2][32];
          tmem_ld32(g_tmem, gv[0]);
          tmem_ld32(g_tmem + 32, gv[1]);
          if (!wait_lean(&s.s_full[g & 1], (g >> 1) & 1, cta_abort, limit, AB_S_FULL)) return false;
          tc_fence_after_sync();
          tmem_ld32(s_tmem, sv[0]);
          tmem_ld32(s_tmem + 32, sv[1]);
          tmem_wait_ld();
          tc_fence_before_sync();
          mbar_arrive(&s.g_free);
          uint32_t words[2] = {~0u, ~0u};
          if constexpr (kMasked) {
            const RowMask mask = row_mask(A, p, j0 + wg * 64, len);
            words[0] = mask.word(0);
            words[1] = mask.word(32);
            if (wg == 0 && j0 + 127 >= len && len < A.Nk && j0 + row >= len) {
              // key rows behind the sequence hold anything (k_full of this tile is complete: S has been formed)
              zero_tile_row(s.kring[g % 3], row);
            }
            __syncwarp();
            fence_proxy_async_smem();
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
            if (kMasked && __all_sync(0xffffffffu, words[c] == 0u)) {
#pragma unroll
              for (int e = 0; e < 16; ++e) pk[e] = 0u;
            } else {
              if constexpr (kMasked) {
                // outside: S = -inf and G = delta, so that dS = 0 * 0 whatever stood there
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  sv[c][e] = (words[c] & (1u << e)) ? sv[c][e] : 0xff800000u;
                  gv[c][e] = (words[c] & (1u << e)) ? gv[c][e] : __float_as_uint(delta);
                }
              }
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float2 w = f32x2_unpack(f32x2_fma(f32x2(__uint_as_float(sv[c][2 * e]), __uint_as_float(sv[c][2 * e + 1])), sl22, nlse2));
                const unsigned long long d =
                    f32x2_add(f32x2(__uint_as_float(gv[c][2 * e]), __uint_as_float(gv[c][2 * e + 1])), ndelta);
                w = f32x2_unpack(f32x2_mul(f32x2(ex2_approx(w.x), ex2_approx(w.y)), d));
                pk[e] = pack2<kBf16>(w.x, w.y);
              }
            }
            tmem_st16(s_tmem + 16 * c, pk);
          }
          tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(&s.w_ready[g & 1]);
          return true;
        };
        alive = tile_masked(A, kt, tile, len) ? form(std::true_type{}) : form(std::false_type{});
        if (!alive) break;
      }
      if (!alive) break;

      // ---- this warp's 32 rows, 64 columns ----
      const bool has = kt.n > 0;
      v_at += kt.n;
      uint8_t* panel = s.vring[v_at & 1] + (warp - 4) * 4096;
      if (has) {
        if (!wait_lean(&s.acc_full, itn & 1, cta_abort, limit, AB_ACC_FULL)) break;
        tc_fence_after_sync();
        stage_row<kBf16>(lanes + kDqAcc + wg * 64, lse2 != INFINITY, args.scale, panel, lane, [&]() {
          tc_fence_before_sync();
          mbar_arrive(&s.acc_free);
        });
      }
      elem_t* out = reinterpret_cast<elem_t*>(args.dq) + b * args.dq_strides.b +
                    (long long)(block * kBlock + ((warp & 3) << 5)) * args.dq_strides.n + h * args.dq_strides.h + wg * 64;
      store_panel(panel, !has, out, args.dq_strides.n, 0, A.Nq - block * kBlock - ((warp & 3) << 5), lane);
      if (has) {
        fence_proxy_async_smem();
        if (lane == 0) mbar_arrive(&s.panel_done);
        ++v_at;
        ++itn;
      }
    }
  }

  if (s.abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  // (reported once every role is here: this thread's own role may have ended long before another's wait ran out)
  if (tid == 0 && s.abort_flag) report_error(ctl, kErrBarrierTimeout, -1, -1, blockIdx.x, s.abort_flag);
  if (warp == 1) tmem_dealloc(tmem, 512);
}

cudaError_t launch_attn_dq(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                           const CUtensorMap& tm_do, const AttnBwdArgs& args, int sms, cudaStream_t stream) {
  const int items = args.a.B * args.a.Hq * args.a.nqb, grid = items < sms ? items : sms;
  const int bytes = (int)sizeof(AttnDqSmem);
  auto kernel = bf16 ? attn_dq_kernel<true> : attn_dq_kernel<false>;
  static SmemOnce once[2];
  cudaError_t e = once[bf16].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  return launch_early(kernel, dim3(grid), kBwThreads, bytes, stream, tm_q, tm_k, tm_v, tm_do, args);
}

// ------------------------------------------------------------------------------------------------------------------
// dK and dV.  Transposed tiles (rows = keys): S^T = K Q^T, G^T = V dO^T, then dV += P^T dO and dK += dS^T Q with P^T
// and dS^T packed over the S^T and G^T columns they were formed from; dV and dK take the other half of TMEM.  One
// buffer each suffices: warp 1 issues dV(q), S(q+1), ... and warp 2 dK(q), G(q+1), ..., so the exponentials of tile
// q + 1 run beside dK(q) and G(q+1), and what the rest of tile q needs beside dV(q) and S(q+1).
// Step q of an item = one block of queries of one of the G heads that share the key head.
// ------------------------------------------------------------------------------------------------------------------
struct DkvSlot {
  int nb;                // blocks of queries per head, -1: no more items
  int b, hk, tile, chunk, first, len;
};

struct AttnDkvSmem {
  alignas(1024) uint8_t k[kTileBytes];
  alignas(1024) uint8_t v[kTileBytes];
  alignas(1024) uint8_t qring[2][kTileBytes];
  alignas(1024) uint8_t gring[2][kTileBytes];      // dO
  alignas(1024) uint8_t stage[kTileBytes];         // per warp a panel of 32 rows x 64 columns
  alignas(16) float stat[2][2 * kBlock];           // with the Q stage: the rows' statistics
  alignas(8) uint64_t q_full[2];
  uint64_t q_empty[2], go_full[2], go_empty[2], slot_full[2], slot_free[2];
  uint64_t k_full, k_free, v_full, v_free;
  uint64_t s_full, p_half, p_ready, dp_full, ds_ready, dv_full, dv_free, dk_full, dk_free;
  DkvSlot slot[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(AttnDkvSmem) <= 232448, "shared memory of a CTA");

constexpr int kKvS = 0, kKvG = 128, kKvDv = 256, kKvDk = 384;

template <bool kBf16>
__global__ void __launch_bounds__(kBwThreads, 1)
attn_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                const AttnBwdArgs args) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  AttnDkvSmem& s = *reinterpret_cast<AttnDkvSmem*>(smem_raw);
  const AttnShape& A = args.a;
  Control* ctl = &g_attn_bwd_ctl;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned long long limit = args.wait_ns;
  volatile int* cta_abort = &s.abort_flag;

  if (smem_u32(smem_raw) & 1023) {
    if (tid == 0) report_error(ctl, kErrAborted, -1, -1, blockIdx.x, 0);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
      mbar_init(&s.go_full[i], 1);
      mbar_init(&s.go_empty[i], 2);
      mbar_init(&s.slot_full[i], 1);
      mbar_init(&s.slot_free[i], 10);      // two issuing and eight P / dS warps
    }
    mbar_init(&s.k_full, 1);
    mbar_init(&s.k_free, 1);
    mbar_init(&s.v_full, 1);
    mbar_init(&s.v_free, 1);
    mbar_init(&s.s_full, 1);
    mbar_init(&s.p_half, 256);
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
  if (!args.after_dq) wait_for_primary();
  launch_dependents();
  const uint32_t tmem = s.tmem_base;
  constexpr int fmt = kBf16 ? 1 : 0;
  constexpr uint32_t idesc_kk = umma_idesc(fmt, 0, 0, 128, 128);
  constexpr uint32_t idesc_mn = umma_idesc(fmt, 0, 1, 128, 128);

  // `g` counts steps, `itn` items that have any
  uint32_t g = 0, itn = 0, slots = 0;
  bool alive = true;
  auto next = [&]() -> const DkvSlot* {
    if (!alive || !wait_lean(&s.slot_full[slots & 1], (slots >> 1) & 1, cta_abort, limit, AB_SLOT_FULL)) return nullptr;
    const DkvSlot* slot = &s.slot[slots & 1];
    return slot->nb < 0 ? nullptr : slot;
  };
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.slot_free[slots & 1]);
    ++slots;
  };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_do);
      KvItem it;
      for (int rnd = 0; alive; ++rnd) {
        const int sl = rnd & 1;
        if (!wait_lane(&s.slot_free[sl], ((rnd >> 1) & 1) ^ 1, cta_abort, limit, AB_SLOT_FREE)) break;
        DkvSlot& x = s.slot[sl];
        if (!kv_item(A, args.chunks, snake_item(rnd, blockIdx.x, gridDim.x), it)) {
          x.nb = -1;
          mbar_arrive(&s.slot_full[sl]);
          break;
        }
        const int len = attn_length(A, args.lengths, it.b);
        const QueryBlocks qb = item_blocks(A, it, len);
        const int nb = imax(0, qb.last - qb.first + 1);
        x.nb = nb;
        x.b = it.b;
        x.hk = it.hk;
        x.tile = it.tile;
        x.chunk = it.chunk;
        x.first = qb.first;
        x.len = len;
        mbar_arrive(&s.slot_full[sl]);
        if (nb == 0) continue;
        if (!wait_lane(&s.k_free, (itn & 1) ^ 1, cta_abort, limit, AB_K_EMPTY)) break;
        mbar_expect_tx(&s.k_full, kTileBytes);
        tma_load_4d(s.k, &tm_k, &s.k_full, 0, it.tile * kBlock, it.hk, it.b);
        tma_load_4d(s.k + kHalfBytes, &tm_k, &s.k_full, 64, it.tile * kBlock, it.hk, it.b);
        bool v_loaded = false;
        for (int h = it.hk * A.G; h < it.hk * A.G + A.G && alive; ++h) {
          const float* stat = args.stat + ((long long)it.b * A.Hq + h) * A.nqb * (2 * kBlock);
          for (int blk = qb.first; blk <= qb.last; ++blk, ++g) {
            const int st = g & 1;
            if (!wait_lane(&s.q_empty[st], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_Q_FREE)) { alive = false; break; }
            mbar_expect_tx(&s.q_full[st], kTileBytes + 2 * kBlock * 4);
            tma_load_4d(s.qring[st], &tm_q, &s.q_full[st], 0, blk * kBlock, h, it.b);
            tma_load_4d(s.qring[st] + kHalfBytes, &tm_q, &s.q_full[st], 64, blk * kBlock, h, it.b);
            bulk_load(s.stat[st], stat + (long long)blk * (2 * kBlock), 2 * kBlock * 4, &s.q_full[st]);
            if (!v_loaded) {
              if (!wait_lane(&s.v_free, (itn & 1) ^ 1, cta_abort, limit, AB_V_EMPTY)) { alive = false; break; }
              mbar_expect_tx(&s.v_full, kTileBytes);
              tma_load_4d(s.v, &tm_v, &s.v_full, 0, it.tile * kBlock, it.hk, it.b);
              tma_load_4d(s.v + kHalfBytes, &tm_v, &s.v_full, 64, it.tile * kBlock, it.hk, it.b);
              v_loaded = true;
            }
            if (!wait_lane(&s.go_empty[st], ((g >> 1) & 1) ^ 1, cta_abort, limit, AB_GO_FREE)) { alive = false; break; }
            mbar_expect_tx(&s.go_full[st], kTileBytes);
            tma_load_4d(s.gring[st], &tm_do, &s.go_full[st], 0, blk * kBlock, h, it.b);
            tma_load_4d(s.gring[st] + kHalfBytes, &tm_do, &s.go_full[st], 64, blk * kBlock, h, it.b);
          }
        }
        ++itn;
      }
    }
  } else if (warp == 1) {
    // S^T(0); then dV(q), S^T(q+1)
    const uint64_t d_k = umma_smem_desc(smem_u32(s.k), 16, 1024);
    const uint64_t d_q0 = umma_smem_desc(smem_u32(s.qring[0]), 16, 1024);
    const uint64_t d_g0 = umma_smem_desc(smem_u32(s.gring[0]), kHalfBytes, 1024);
    while (const DkvSlot* x = next()) {
      const int n = x->nb * A.G;
      done();
      if (n == 0) continue;
      if (!wait_lean(&s.k_full, itn & 1, cta_abort, limit, AB_K_FULL)) break;
      auto issue_s = [&](uint32_t gq) -> bool {
        if (!wait_lean(&s.q_full[gq & 1], (gq >> 1) & 1, cta_abort, limit, AB_Q_FULL)) return false;
        tc_fence_after_sync();
        issue_kk(tmem + kKvS, d_k, d_q0 + (gq & 1) * (kTileBytes >> 4), idesc_kk);
        umma_commit_w(&s.s_full);
        return true;
      };
      if (!issue_s(g)) break;
      for (int q = 0; q < n; ++q, ++g) {
        if (!wait_lean(&s.go_full[g & 1], (g >> 1) & 1, cta_abort, limit, AB_GO_FULL)) { alive = false; break; }
        if (q == 0 && !wait_lean(&s.dv_free, (itn & 1) ^ 1, cta_abort, limit, AB_ACC_FREE)) { alive = false; break; }
        if (!wait_lean(&s.p_half, g & 1, cta_abort, limit, AB_P_READY)) { alive = false; break; }
        tc_fence_after_sync();
        const uint64_t db = d_g0 + (g & 1) * (kTileBytes >> 4);
        issue_ts_part<0>(tmem + kKvDv, tmem + kKvS, db, idesc_mn, q ? 1u : 0u);
        if (!wait_lean(&s.p_ready, g & 1, cta_abort, limit, AB_P_READY)) { alive = false; break; }
        tc_fence_after_sync();
        issue_ts_part<1>(tmem + kKvDv, tmem + kKvS, db, idesc_mn, 1u);
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
    while (const DkvSlot* x = next()) {
      const int n = x->nb * A.G;
      done();
      if (n == 0) continue;
      if (!wait_lean(&s.v_full, itn & 1, cta_abort, limit, AB_V_FULL)) break;
      auto issue_g = [&](uint32_t gq) -> bool {
        if (!wait_lean(&s.go_full[gq & 1], (gq >> 1) & 1, cta_abort, limit, AB_GO_FULL)) return false;
        tc_fence_after_sync();
        issue_kk(tmem + kKvG, d_v, d_g0 + (gq & 1) * (kTileBytes >> 4), idesc_kk);
        umma_commit_w(&s.go_empty[gq & 1]);
        umma_commit_w(&s.dp_full);
        return true;
      };
      if (!issue_g(g)) break;
      for (int q = 0; q < n; ++q, ++g) {
        if (q == 0 && !wait_lean(&s.dk_free, (itn & 1) ^ 1, cta_abort, limit, AB_ACC_FREE)) { alive = false; break; }
        if (!wait_lean(&s.ds_ready, g & 1, cta_abort, limit, AB_DS_READY)) { alive = false; break; }
        tc_fence_after_sync();
        issue_ts(tmem + kKvDk, tmem + kKvG, d_q0 + (g & 1) * (kTileBytes >> 4), idesc_mn, q ? 1u : 0u);
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
    constexpr float kUnit = 1 << kWeightBits<kBf16>;
    const unsigned long long sl22 = f32x2(sl2, sl2), minus = f32x2(-1.f, -1.f), part = f32x2(1.f / kUnit, 1.f / kUnit);
    uint8_t* panel = s.stage + (warp - 4) * 4096;
    while (const DkvSlot* x = next()) {
      const int nb = x->nb, n = nb * A.G, len = x->len, tile = x->tile, chunk = x->chunk, b = x->b, hk = x->hk, first = x->first;
      done();
      const int j0 = tile * kBlock, j = j0 + row;
      int blk = first;
      for (int q = 0; q < n; ++q, ++g) {
        const int st = g & 1;
        const int p0 = blk * kBlock + A.off;         // position of the block's first query
        if (++blk == first + nb) blk = first;
        const float* stat = s.stat[st] + wg * 64;
        auto form = [&](auto some_masked) -> bool {
          constexpr bool kMasked = decltype(some_masked)::value;
          uint32_t words[2] = {~0u, ~0u};
          if constexpr (kMasked) {
            const ColMask mask = col_mask(A, j, p0 + wg * 64, len);
            words[0] = mask.word(0);
            words[1] = mask.word(32);
          }
          if (!wait_lean(&s.s_full, g & 1, cta_abort, limit, AB_S_FULL)) return false;
          // (for this thread's own reads of the statistics: the load that brought Q brought them)
          if (!wait_lean(&s.q_full[st], (g >> 1) & 1, cta_abort, limit, AB_Q_FULL)) return false;
          tc_fence_after_sync();
          uint32_t v[2][32];
          tmem_ld32(s_tmem, v[0]);
          tmem_ld32(s_tmem + 32, v[1]);
          tmem_wait_ld();
          // Query rows behind the sequence hold anything, and 0 * NaN is not 0: they become zero in Q and dO before
          // the products that sum over them; so do, in Q, those of queries that see one key, whose dS is 0 exactly.  S^T and
          // G^T, which read them as columns, are complete by then.
          const bool stale = kMasked && p0 + 127 >= len && len < A.Nk;
          const bool cleared = stale || (kMasked && (sees_one(A, p0) || sees_one(A, p0 + 127)));
          if (cleared) {
            if (!wait_lean(&s.dp_full, g & 1, cta_abort, limit, AB_DP_FULL)) return false;
            if (wg == 0) {
              if (p0 + row >= len || sees_one(A, p0 + row)) zero_tile_row(s.qring[st], row);
              if (p0 + row >= len) zero_tile_row(s.gring[st], row);
            }
            __syncwarp();
            fence_proxy_async_smem();
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
            bool empty = false;
            if constexpr (kMasked) {
              empty = __all_sync(0xffffffffu, words[c] == 0u);
              if (!__all_sync(0xffffffffu, words[c] == ~0u)) {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[c][e] = (words[c] & (1u << e)) ? v[c][e] : 0xff800000u;
              }
            }
            if (kMasked && empty) {
#pragma unroll
              for (int e = 0; e < 32; ++e) v[c][e] = 0u;
#pragma unroll
              for (int e = 0; e < 16; ++e) pk[e] = 0u;
            } else {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float4 t = *reinterpret_cast<const float4*>(stat + 32 * c + 2 * e);
              float2 w = f32x2_unpack(f32x2_fma(f32x2(t.x, t.y), minus,
                                                f32x2_mul(f32x2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), sl22)));
              float2 y = f32x2_unpack(f32x2_fma(f32x2(t.z, t.w), minus,
                                                f32x2_mul(f32x2(__uint_as_float(v[c][2 * e + 2]), __uint_as_float(v[c][2 * e + 3])), sl22)));
              w.x = ex2_approx(w.x);
              w.y = ex2_approx(w.y);
              y.x = ex2_approx(y.x);
              y.y = ex2_approx(y.y);
              v[c][2 * e] = __float_as_uint(w.x);
              v[c][2 * e + 1] = __float_as_uint(w.y);
              v[c][2 * e + 2] = __float_as_uint(y.x);
              v[c][2 * e + 3] = __float_as_uint(y.y);
              pk[e] = pack2<kBf16>(w.x, w.y);
              pk[e + 1] = pack2<kBf16>(y.x, y.y);
            }
            }
            tmem_st16(s_tmem + 16 * c, pk);
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(c ? &s.p_ready : &s.p_half);
          }
          if (!cleared && !wait_lean(&s.dp_full, g & 1, cta_abort, limit, AB_DP_FULL)) return false;
          tc_fence_after_sync();
          uint32_t ga[16], gb[16];
          auto ds = [&](uint32_t (&cur)[16], uint32_t (&nxt)[16], int c) {
            if (c < 3) tmem_ld16(g_tmem + 16 * (c + 1), nxt);
            uint32_t w[8];
            const uint32_t* pv = v[c >> 1] + 16 * (c & 1);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float4 t = *reinterpret_cast<const float4*>(stat + kBlock + 16 * c + 2 * e);
              float2 a = f32x2_unpack(f32x2_mul(f32x2(__uint_as_float(pv[2 * e]), __uint_as_float(pv[2 * e + 1])),
                                                f32x2_fma(f32x2(__uint_as_float(cur[2 * e]), __uint_as_float(cur[2 * e + 1])), part, f32x2(t.x, t.y))));
              float2 d = f32x2_unpack(f32x2_mul(f32x2(__uint_as_float(pv[2 * e + 2]), __uint_as_float(pv[2 * e + 3])),
                                                f32x2_fma(f32x2(__uint_as_float(cur[2 * e + 2]), __uint_as_float(cur[2 * e + 3])), part, f32x2(t.z, t.w))));
              if (kMasked && stale) {          // (elsewhere G is finite, and 0 * G is 0)
                const uint32_t m = words[c >> 1] >> (16 * (c & 1) + 2 * e);
                a.x = (m & 1u) ? a.x : 0.f;
                a.y = (m & 2u) ? a.y : 0.f;
                d.x = (m & 4u) ? d.x : 0.f;
                d.y = (m & 8u) ? d.y : 0.f;
              }
              w[e] = pack2<kBf16>(a.x, a.y);
              w[e + 1] = pack2<kBf16>(d.x, d.y);
            }
            if (c < 3) tmem_wait_ld();
            tmem_st8(g_tmem + 8 * c, w);
          };
          tmem_ld16(g_tmem, ga);
          tmem_wait_ld();
          ds(ga, gb, 0);
          ds(gb, ga, 1);
          ds(ga, gb, 2);
          ds(gb, ga, 3);
          tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(&s.ds_ready);
          return true;
        };
        alive = block_masked(A, j0, p0, len) ? form(std::true_type{}) : form(std::false_type{});
        if (!alive) break;
      }
      if (!alive) break;

      // ---- epilogue: this warp's 32 key rows, 64 of the 128 columns of dV and of dK ----
      const bool has = n > 0, key = j < len;
      const int r0 = j0 + ((warp & 3) << 5);
      const bool joined = args.chunks > 0 && tile == 0;          // the first keys' rows: fp32 sums, joined afterwards
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {                  // 0: dV, 1: dK
        const uint32_t t_addr = lanes + (which ? kKvDk : kKvDv) + wg * 64;
        const float f = which ? args.scale : 1.f / kUnit;
        if (has) {
          if (!wait_lean(which ? &s.dk_full : &s.dv_full, itn & 1, cta_abort, limit, AB_ACC_FULL)) { alive = false; break; }
          tc_fence_after_sync();
        }
        if (joined) {
          float* part = args.partial + ((((long long)(b * A.Hkv + hk) * (1 + args.chunks) + chunk + 1) * 2 + which) * A.S + j) * 128 + wg * 64;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[16];
            if (has) {
              tmem_ld16(t_addr + 16 * c, o);
              tmem_wait_ld();
            }
            if (j < A.S && j < A.Nk) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<float4*>(part + 16 * c + 4 * e) =
                    has && key ? make_float4(__uint_as_float(o[4 * e]) * f, __uint_as_float(o[4 * e + 1]) * f,
                                             __uint_as_float(o[4 * e + 2]) * f, __uint_as_float(o[4 * e + 3]) * f)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            __syncwarp();
          }
        }
        if (has)
          stage_row<kBf16>(t_addr, key, f, panel, lane, [&]() {
            tc_fence_before_sync();
            mbar_arrive(which ? &s.dk_free : &s.dv_free);
          });
        if (chunk < 0) {
          const Strides& sd = which ? args.dk_strides : args.dv_strides;
          elem_t* out = reinterpret_cast<elem_t*>(which ? args.dk : args.dv) + b * sd.b + (long long)r0 * sd.n + hk * sd.h + wg * 64;
          store_panel(panel, !has, out, sd.n, joined ? A.S - r0 : 0, A.Nk - r0, lane);
        }
      }
      if (has) ++itn;
    }
  }

  if (args.after_dq) wait_for_primary();       // what follows this kernel follows the dQ kernel as well
  if (s.abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  // (reported once every role is here: this thread's own role may have ended long before another's wait ran out)
  if (tid == 0 && s.abort_flag) report_error(ctl, kErrBarrierTimeout, -1, -1, blockIdx.x, s.abort_flag);
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// The first keys' rows: the tile's own sums and those of the chunks, added in order.
template <bool kBf16>
__global__ void __launch_bounds__(128) attn_first_keys_kernel(const AttnBwdArgs args) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  wait_for_primary();
  const AttnShape& A = args.a;
  const int bh = blockIdx.x, which = blockIdx.y, j = blockIdx.z, b = bh / A.Hkv, hk = bh % A.Hkv;
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
  const int bytes = (int)sizeof(AttnDkvSmem);
  auto kernel = bf16 ? attn_dkv_kernel<true> : attn_dkv_kernel<false>;
  static SmemOnce once[2];
  cudaError_t e = once[bf16].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  e = launch_early(kernel, dim3(grid), kBwThreads, bytes, stream, tm_q, tm_k, tm_v, tm_do, args);
  if (e != cudaSuccess || args.chunks == 0) return e;
  const dim3 sum_grid(a.B * a.Hkv, 2, a.S < a.Nk ? a.S : a.Nk);     // (S <= 128; batch times heads may pass 65535)
  return launch_early(bf16 ? attn_first_keys_kernel<true> : attn_first_keys_kernel<false>, sum_grid, 128, 0, stream, args);
}

cudaError_t attn_bwd_status(cudaStream_t stream, int out[8]) { return take_status(&g_attn_bwd_ctl, stream, out); }

}  // namespace lucid
