// Single-token attention over a paged key/value cache, and the LUCID solve's next row with the attention that reads it.
//
// The cache is read once and dominates everything: 512 bytes per key and head against one multiply-add per element and
// query, so the kernel is bound by HBM (long contexts) or by latency (short ones), and the tensor work is small: the
// G query heads that share a key head are the rows of one 16-row matrix instruction (mma.sync; a tcgen05 tile has 128
// rows, of which 8 would be in use).  Keys are split over CTAs (`splits` chunks per sequence and key head); each warp
// streams blocks of 16 keys through a ring of its own (cp.async, page by page) with a running maximum and sum, and the
// warps of a CTA meet in shared memory.  Up to 8 chunks are the CTAs of one cluster and meet there too, each CTA taking a
// share of the columns from its peers' shared memory: one launch, no scratch memory.  One long sequence alone needs more
// CTAs than that to draw on the whole HBM; its chunks meet in a second kernel.
//
// LUCID: with t_j = k_scale^2 k_n.k_j the solve's newest row is v'_n = exp(-t_n) v_n - sum_{j<n} exp(t_j - t_n) v'_j, an
// unnormalised attention of k_n over the rows before it.  So k_n is one more row of the same matrix instruction: one
// pass over the cache serves the solve and the attention, whose own weight on v'_n is added when both sums are known.
#include <type_traits>
#include "attn.h"

namespace lucid {

static __device__ Control g_paged_ctl;

constexpr int kPaWarps = 4, kPaStages = 2, kPaKeys = 16;
// (two stages - one block on its way while one is worked on - and three CTAs per SM; three stages and two CTAs took 106 us
// where this takes 99 on 32 ragged sequences of up to 16384 keys, and 22 us against 16.5 on 12 of up to 3001)
constexpr int kPaStageBytes = 2 * kPaKeys * 256;               // K block, V block
constexpr int kPaRow = 132;                                    // floats of a partial sum: 128 sums, maximum, sum, 2 unused
constexpr int kPaMinChunk = 64;                                // keys of a split: at least one block per warp

struct PagedAttnSmem {
  alignas(128) uint8_t q[16 * 256];
  alignas(128) uint8_t ring[kPaWarps][kPaStages][kPaStageBytes];
  int valid[kPaWarps][kPaStages];                              // bit r: row r of the block is a key
  float ml[kPaWarps][16][2];
  float chunk_ml[16][2];                                       // the CTA's own maximum and sum of each row
  float self[16];                                              // LUCID: row . k_n, unscaled
};

// What a sequence shows its newest query; LUCID: the rows before the newest one.
__device__ __forceinline__ Visible visible(const PagedAttnArgs& a, bool lucid, int len) {
  return cache_visible(a.W, a.S, lucid ? len - 1 : len, a.c.table_width << a.c.page_shift);
}
__device__ __forceinline__ int chunk_keys(int n, int splits) {
  const int even = (n + splits - 1) / splits;
  const int c = (even + kPaMinChunk - 1) / kPaMinChunk * kPaMinChunk;
  return c < kPaMinChunk ? kPaMinChunk : c;
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes global -> shared; `bytes` 0 writes zeros and reads nothing
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
// rows of 256 bytes, 16-byte chunks XOR-permuted by the row: eight rows' equal chunks fall into eight bank groups
__device__ __forceinline__ uint32_t row256(int row, int chunk) { return row * 256 + ((chunk ^ (row & 7)) << 4); }

// Page of a position, or -1.
__device__ __forceinline__ long long page_of(const PagedCache& c, int b, int pos) {
  const int i = pos >> c.page_shift;
  if (pos < 0 || i >= c.table_width) return -1;
  const long long p = __ldg(c.table + b * c.table_stride + i);
  return p < c.pages ? p : -1;
}

template <typename elem_t>
__device__ __forceinline__ float as_float(elem_t x) {
  if constexpr (std::is_same<elem_t, __nv_bfloat16>::value) return __bfloat162float(x);
  else return __half2float(x);
}
template <typename elem_t>
__device__ __forceinline__ elem_t as_elem(float x) {
  if constexpr (std::is_same<elem_t, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
// LUCID's closing step for one column, given the joined sums over the rows before the newest:
// v'_n from k_n's row (reference km, sum ka) and t_n; then a query row's result with its weight on v'_n.
__device__ __forceinline__ float lucid_new_value(float tn, float vn, float km, float ka) {
  float v = ex2_approx(-tn) * vn;
  if (km != -INFINITY) v -= ex2_approx(km - tn) * ka;
  return v;
}
__device__ __forceinline__ float lucid_output(float sn, float v_new, float m, float l, float a) {
  const float mm = fmaxf(m, sn);
  const float f = m == -INFINITY ? 0.f : ex2_approx(m - mm), w = ex2_approx(sn - mm);
  return (a * f + w * v_new) / (l * f + w);
}

// kCluster: the grid's x dimension is one cluster of `splits` CTAs (1, 2, 4 or 8)
template <bool kBf16, bool kLucid, bool kCluster>
__global__ void __launch_bounds__(kPaWarps * 32, kPagedPerSm) paged_attn_kernel(const PagedAttnArgs args) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  extern __shared__ uint8_t smem_raw[];
  PagedAttnSmem& s = *reinterpret_cast<PagedAttnSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const PagedCache& c = args.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x, b = blockIdx.z;
  const int chunks = (args.G + 15) / 16, hk = blockIdx.y / chunks, rc = blockIdx.y % chunks;
  const int heads = imin(16, args.G - 16 * rc);                // query rows of this CTA
  const int rows = heads + (kLucid ? 1 : 0);
  const int len = __ldg(args.lens + b);
  const Visible vis = visible(args, kLucid, len);
  const int chunk = chunk_keys(vis.n, args.splits);
  const int begin = split * chunk, end = imin(vis.n, begin + chunk);
  if (!kLucid && split == 0 && tid == 0 && len > (c.table_width << c.page_shift)) report_error(&g_paged_ctl, kErrBadPage, b, len - 1, len - 1, 0);
  if constexpr (!kCluster) {
    launch_dependents();
    if (begin >= end) return;                                  // an empty chunk: the second kernel does not read it
  }

  // ---- this warp's blocks: begin + (4 i + warp) * 16 ----
  const int first = begin + warp * kPaKeys, stride = kPaWarps * kPaKeys;
  const int blocks = first < end ? (end - first + stride - 1) / stride : 0;
  uint8_t* ring = s.ring[warp][0];
  auto load = [&](int i) {
    const int st = i % kPaStages;
    if (i < blocks) {
      // lanes 0-15: the row of the cache of one key each
      const int v = first + i * stride + (lane & 15);
      long long page = -1;
      int pos = 0;
      if (v < end) {
        pos = vis.pos(v);
        page = page_of(c, b, pos);
        if (page < 0 && lane < 16) report_error(&g_paged_ctl, kErrBadPage, b, pos, pos, 0);
      }
      const bool ok = page >= 0;
      const long long slot = pos & ((1 << c.page_shift) - 1);
      const long long ko = ok ? page * c.k_page + slot * c.k_row + hk * c.k_head : 0;
      const long long vo = ok ? page * c.v_page + slot * c.v_row + hk * c.v_head : 0;
      const unsigned mask = __ballot_sync(0xffffffffu, ok);
      if (lane == 0) s.valid[warp][st] = mask & 0xffff;
      const uint32_t dst = smem_u32(ring + st * kPaStageBytes);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int r = 2 * x + (lane >> 4), ch = lane & 15;
        const long long kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
        const int bytes = (mask >> r) & 1 ? 16 : 0;
        cp_async16(dst + row256(r, ch), reinterpret_cast<const elem_t*>(c.k) + kr + 8 * ch, bytes);
        cp_async16(dst + kPaKeys * 256 + row256(r, ch), reinterpret_cast<const elem_t*>(c.v) + vr + 8 * ch, bytes);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kPaStages - 1; ++i) load(i);
  // ---- queries (and k_n) into shared memory, then into fragments, while the first blocks are on their way ----
  for (int x = tid; x < 256; x += kPaWarps * 32) {
    const int r = x >> 4, ch = x & 15;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < heads) {
      w = *reinterpret_cast<const uint4*>(reinterpret_cast<const elem_t*>(args.q) + b * args.q_b +
                                          (hk * args.G + 16 * rc + r) * args.q_h + 8 * ch);
    } else if (kLucid && r == heads) {
      const long long page = page_of(c, b, len - 1);
      if (page >= 0)
        w = *reinterpret_cast<const uint4*>(reinterpret_cast<const elem_t*>(c.k) + page * c.k_page +
                                            ((len - 1) & ((1 << c.page_shift) - 1)) * c.k_row + hk * c.k_head + 8 * ch);
    }
    *reinterpret_cast<uint4*>(s.q + row256(r, ch)) = w;
  }
  __syncthreads();
  if constexpr (kLucid && kCluster) {
    for (int r = warp; r < rows; r += kPaWarps) {
      const uint32_t at = (lane & 1) * 8;
      const uint2 x = *reinterpret_cast<const uint2*>(s.q + row256(r, lane >> 1) + at);
      const uint2 y = *reinterpret_cast<const uint2*>(s.q + row256(heads, lane >> 1) + at);
      const float2 x0 = unpack2<kBf16>(x.x), x1 = unpack2<kBf16>(x.y), y0 = unpack2<kBf16>(y.x), y1 = unpack2<kBf16>(y.y);
      float dot = (x0.x * y0.x + x0.y * y0.y) + (x1.x * y1.x + x1.y * y1.y);
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
      if (lane == 0) s.self[r] = dot;
    }
  }
  uint32_t qf[8][4];
#pragma unroll
  for (int k = 0; k < 8; ++k) ldmatrix4(qf[k], smem_u32(s.q) + row256(lane & 15, 2 * k + (lane >> 4)));

  const int r0 = lane >> 2, r1 = r0 + 8;                       // the fragment rows of this lane
  const float sc0 = (kLucid && r0 == heads) ? args.lucid_log2 : args.scale_log2;
  const float sc1 = (kLucid && r1 == heads) ? args.lucid_log2 : args.scale_log2;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float acc[16][4];
#pragma unroll
  for (int n = 0; n < 16; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;

  for (int i = 0; i < blocks; ++i) {
    cp_async_wait<kPaStages - 2>();
    __syncwarp();
    load(i + kPaStages - 1);
    const int st = i % kPaStages;
    const uint32_t kb = smem_u32(ring + st * kPaStageBytes), vb = kb + kPaKeys * 256;
    const int valid = s.valid[warp][st];
    float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};      // keys 0-7, keys 8-15
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t bk[4];
      ldmatrix4(bk, kb + row256((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
      mma16816<kBf16>(sa, qf[k], bk[0], bk[1]);
      mma16816<kBf16>(sb, qf[k], bk[2], bk[3]);
    }
    const int col = (lane & 3) * 2;
    const bool c0 = (valid >> col) & 1, c1 = (valid >> (col + 1)) & 1, c2 = (valid >> (col + 8)) & 1, c3 = (valid >> (col + 9)) & 1;
    sa[0] = c0 ? sa[0] * sc0 : -INFINITY;
    sa[1] = c1 ? sa[1] * sc0 : -INFINITY;
    sb[0] = c2 ? sb[0] * sc0 : -INFINITY;
    sb[1] = c3 ? sb[1] * sc0 : -INFINITY;
    sa[2] = c0 ? sa[2] * sc1 : -INFINITY;
    sa[3] = c1 ? sa[3] * sc1 : -INFINITY;
    sb[2] = c2 ? sb[2] * sc1 : -INFINITY;
    sb[3] = c3 ? sb[3] * sc1 : -INFINITY;
    float n0 = fmaxf(fmaxf(sa[0], sa[1]), fmaxf(sb[0], sb[1])), n1 = fmaxf(fmaxf(sa[2], sa[3]), fmaxf(sb[2], sb[3]));
    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2));
    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2));
    if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
      n0 = fmaxf(n0, m0);
      n1 = fmaxf(n1, m1);
      const float f0 = n0 == -INFINITY ? 1.f : ex2_approx(m0 - n0), f1 = n1 == -INFINITY ? 1.f : ex2_approx(m1 - n1);
      m0 = n0;
      m1 = n1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        acc[n][0] *= f0;
        acc[n][1] *= f0;
        acc[n][2] *= f1;
        acc[n][3] *= f1;
      }
    }
    const float z0 = m0 == -INFINITY ? 0.f : m0 - kTopWeight<kBf16>, z1 = m1 == -INFINITY ? 0.f : m1 - kTopWeight<kBf16>;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sa[e] = ex2_approx(sa[e] - z0);
      sb[e] = ex2_approx(sb[e] - z0);
      sa[e + 2] = ex2_approx(sa[e + 2] - z1);
      sb[e + 2] = ex2_approx(sb[e + 2] - z1);
    }
    const uint32_t pf[4] = {pack2<kBf16>(sa[0], sa[1]), pack2<kBf16>(sa[2], sa[3]), pack2<kBf16>(sb[0], sb[1]),
                            pack2<kBf16>(sb[2], sb[3])};
    // the sums of the weights as they are rounded: the result is a mean of values even where one weight is nearly all
    float e0 = 0.f, e1 = 0.f, f0 = 0.f, f1 = 0.f;
    add_halves<kBf16>(e0, e1, pf[0]);
    add_halves<kBf16>(e0, e1, pf[2]);
    add_halves<kBf16>(f0, f1, pf[1]);
    add_halves<kBf16>(f0, f1, pf[3]);
    l0 += e0 + e1;
    l1 += f0 + f1;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      uint32_t bv[4];      // keys 0-7 and 8-15 of columns 16n .. 16n+7, then of 16n+8 .. 16n+15
      ldmatrix4_trans(bv, vb + row256(lane & 15, 2 * n + (lane >> 4)));
      mma16816<kBf16>(acc[2 * n], pf, bv[0], bv[1]);
      mma16816<kBf16>(acc[2 * n + 1], pf, bv[2], bv[3]);
    }
    __syncwarp();
  }
  cp_async_wait<0>();

  // ---- the four warps' sums ----
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  __syncthreads();
  float* mine = reinterpret_cast<float*>(ring);                // 16 x 128 sums of this warp
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    const int col = 8 * n + (lane & 3) * 2;
    *reinterpret_cast<float2*>(mine + r0 * 128 + col) = make_float2(acc[n][0], acc[n][1]);
    *reinterpret_cast<float2*>(mine + r1 * 128 + col) = make_float2(acc[n][2], acc[n][3]);
  }
  if ((lane & 3) == 0) {
    s.ml[warp][r0][0] = m0 - kTopWeight<kBf16>;        // (what the sums are relative to)
    s.ml[warp][r0][1] = l0;
    s.ml[warp][r1][0] = m1 - kTopWeight<kBf16>;
    s.ml[warp][r1][1] = l1;
  }
  __syncthreads();
  float* joined = reinterpret_cast<float*>(s.ring[0][1]);      // rows x 128 of this CTA (the stage behind warp 0's sums)
  for (int r = 0; r < rows; ++r) {
    float m = -INFINITY, l = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < kPaWarps; ++w) m = fmaxf(m, s.ml[w][r][0]);
    const float z = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kPaWarps; ++w) {
      const float f = ex2_approx(s.ml[w][r][0] - z);
      l += f * s.ml[w][r][1];
      a += f * reinterpret_cast<const float*>(s.ring[w][0])[r * 128 + tid];
    }
    if constexpr (kCluster) {
      joined[r * 128 + tid] = a;
      if (tid == 0) s.chunk_ml[r][0] = m;
      if (tid == 1) s.chunk_ml[r][1] = l;
    } else {
      const int total = args.G + (kLucid ? 1 : 0);
      float* p = args.partial + ((((long long)b * args.Hkv + hk) * total + 16 * rc + r) * args.splits + split) * kPaRow;
      p[tid] = a;
      if (tid == 0) p[128] = m;
      if (tid == 1) p[129] = l;
    }
  }
  if constexpr (kCluster) {
    cluster_sync_all();
    // this CTA's share: columns split * per .. + per - 1 of every row
    const int n = args.splits, per = 128 / n, col = split * per + tid % per;
    const uint32_t a_joined = smem_u32(joined) + col * 4, a_ml = smem_u32(s.chunk_ml);
    auto join = [&](int r, float& m, float& l, float& a) {
      float pm[8], pl[8], pa[8];
      m = -INFINITY;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if (x < n) {
          const uint32_t at = mapa_u32(a_ml + r * 8, x);
          pm[x] = ld_cluster(at);
          pl[x] = ld_cluster(at + 4);
          pa[x] = ld_cluster(mapa_u32(a_joined + r * 512, x));
        } else {
          pm[x] = -INFINITY;
          pl[x] = pa[x] = 0.f;
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) m = fmaxf(m, pm[x]);
      const float z = m == -INFINITY ? 0.f : m;
      l = a = 0.f;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float f = ex2_approx(pm[x] - z);
        l += f * pl[x];
        a += f * pa[x];
      }
    };
    elem_t v_stored = as_elem<elem_t>(0.f);
    long long page = -1;
    float m, l, a;
    if constexpr (kLucid) {
      if (len > 0) page = page_of(c, b, len - 1);
      join(heads, m, l, a);
      if (page >= 0) {
        const float vn = as_float(reinterpret_cast<const elem_t*>(args.v_new)[b * args.v_b + hk * args.v_h + col]);
        // the attention reads v'_n as the cache keeps it
        v_stored = as_elem<elem_t>(lucid_new_value(s.self[heads] * args.lucid_log2, vn, m, a));
        if (tid < per)
          reinterpret_cast<elem_t*>(c.v)[page * c.v_page + ((len - 1) & ((1 << c.page_shift) - 1)) * c.v_row + hk * c.v_head + col] = v_stored;
      } else if (len > 0 && tid == 0) {
        report_error(&g_paged_ctl, kErrBadPage, b, len - 1, len - 1, 0);
      }
    }
    for (int r = tid / per; r < heads; r += n) {
      join(r, m, l, a);
      float o = l != 0.f ? a / l : 0.f;
      if constexpr (kLucid) o = page >= 0 ? lucid_output(s.self[r] * args.scale_log2, as_float(v_stored), m, l, a) : 0.f;
      reinterpret_cast<elem_t*>(args.out)[((long long)b * args.Hq + hk * args.G + 16 * rc + r) * 128 + col] = as_elem<elem_t>(o);
    }
    cluster_sync_all();                                        // no CTA leaves while a peer reads its sums
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Joins the chunks of one row; LUCID: also of k_n's row, from which v'_n follows, and adds v'_n's own share.
// One CTA per (query head of a key head, key head, sequence), eight groups of 128 threads (one column each); LUCID: half of
// them on k_n's row.
// ------------------------------------------------------------------------------------------------------------------
constexpr int kJoinGroups = 8, kPaMaxSplits = kPagedMaxSplits;

__device__ __forceinline__ float block_sum(float x, float* red) {       // 128 threads of one group use the result
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  __syncthreads();
  if (lane == 0) red[warp] = x;
  __syncthreads();
  const int g = (warp >> 2) << 2;
  return (red[g] + red[g + 1]) + (red[g + 2] + red[g + 3]);
}

// Maximum, sum and this thread's column of a row's chunks, joined by `groups` groups of 128 threads (this thread is in
// group `g`; every thread of the CTA calls it with its own row).  w: this row's weights, red: the groups' sums.
__device__ __forceinline__ void join_row(const float* p, int n, int g, int groups, float& m, float& l, float& a,
                                         float* w, float (*red)[128], float* ml) {
  const int d = threadIdx.x & 127, t = g * 128 + d, lane = threadIdx.x & 31;
  // the chunks' maxima and sums, all at once; a warp of each row's first group joins them
  if (t < n) {
    w[t] = p[(long long)t * kPaRow + 128];
    w[kPaMaxSplits + t] = p[(long long)t * kPaRow + 129];
  }
  __syncthreads();
  if (t < 32) {
    float mm = -INFINITY;
    for (int c = lane; c < n; c += 32) mm = fmaxf(mm, w[c]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
    const float z = mm == -INFINITY ? 0.f : mm;
    float sum = 0.f;
    for (int c = lane; c < n; c += 32) {
      const float f = ex2_approx(w[c] - z);
      w[c] = f;
      sum += f * w[kPaMaxSplits + c];
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) {
      ml[0] = mm;
      ml[1] = sum;
    }
  }
  __syncthreads();
  float acc = 0.f;
#pragma unroll 16
  for (int c = g; c < n; c += groups) acc += w[c] * p[(long long)c * kPaRow + d];
  red[g][d] = acc;
  __syncthreads();
  m = ml[0];
  l = ml[1];
  a = 0.f;
  for (int x = 0; x < groups; ++x) a += red[x][d];
}

template <bool kBf16, bool kLucid>
__global__ void __launch_bounds__(128 * kJoinGroups) paged_join_kernel(const PagedAttnArgs args) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  constexpr int kRows = kLucid ? 2 : 1, kGroups = kJoinGroups / kRows;
  __shared__ float red[kRows][kGroups][128];
  __shared__ float weights[kRows][2 * kPaMaxSplits], ml[kRows][2], sums[kRows][128];
  __shared__ float red1[4 * kJoinGroups];
  const int row = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, d = threadIdx.x & 127;
  const int which = (threadIdx.x >> 7) / kGroups, g = (threadIdx.x >> 7) % kGroups;     // which row this group joins
  wait_for_primary();
  const int len = __ldg(args.lens + b);
  const Visible vis = visible(args, kLucid, len);
  const int chunk = chunk_keys(vis.n, args.splits);
  const int n = (vis.n + chunk - 1) / chunk;                   // chunks that were written
  const int total = args.G + (kLucid ? 1 : 0);
  const float* part = args.partial + (((long long)b * args.Hkv + hk) * total) * args.splits * kPaRow;
  float m, l, a;
  join_row(part + (long long)(which ? args.G : row) * args.splits * kPaRow, n, g, kGroups, m, l, a, weights[which], red[which], ml[which]);
  float o;
  if constexpr (!kLucid) {
    o = l != 0.f ? a / l : 0.f;
  } else {
    const PagedCache& c = args.c;
    const long long page = len > 0 ? page_of(c, b, len - 1) : -1;
    const long long slot = len > 0 ? (len - 1) & ((1 << c.page_shift) - 1) : 0;
    if (len > 0 && page < 0 && threadIdx.x == 0) report_error(&g_paged_ctl, kErrBadPage, b, len - 1, len - 1, 0);
    if (g == 0) sums[which][d] = a;
    __syncthreads();
    const float km = ml[1][0], ka = sums[1][d];
    m = ml[0][0];
    l = ml[0][1];
    a = sums[0][d];
    o = 0.f;
    if (page >= 0) {                                           // (uniform in the CTA)
      const float kn = as_float(reinterpret_cast<const elem_t*>(c.k)[page * c.k_page + slot * c.k_row + hk * c.k_head + d]);
      const float qn = as_float(reinterpret_cast<const elem_t*>(args.q)[b * args.q_b + (hk * args.G + row) * args.q_h + d]);
      const float vn = as_float(reinterpret_cast<const elem_t*>(args.v_new)[b * args.v_b + hk * args.v_h + d]);
      const float tn = block_sum(kn * kn, red1) * args.lucid_log2;
      const float sn = block_sum(qn * kn, red1) * args.scale_log2;
      // the attention reads v'_n as the cache keeps it
      const elem_t stored = as_elem<elem_t>(lucid_new_value(tn, vn, km, ka));
      if (row == 0 && threadIdx.x < 128)
        reinterpret_cast<elem_t*>(c.v)[page * c.v_page + slot * c.v_row + hk * c.v_head + d] = stored;
      o = lucid_output(sn, as_float(stored), m, l, a);
    }
  }
  if (threadIdx.x < 128)
    reinterpret_cast<elem_t*>(args.out)[((long long)b * args.Hq + hk * args.G + row) * 128 + d] = as_elem<elem_t>(o);
}

size_t paged_attn_partial_bytes(int B, int Hq, int Hkv, bool lucid, int splits) {
  if (splits <= kPagedCluster) return 0;
  return (size_t)B * (Hq + (lucid ? Hkv : 0)) * splits * kPaRow * sizeof(float);
}

template <bool kBf16, bool kLucid>
static cudaError_t launch_typed(const PagedAttnArgs& args, cudaStream_t stream) {
  const int bytes = (int)sizeof(PagedAttnSmem) + 128;
  const bool cluster = args.splits <= kPagedCluster;
  auto kernel = cluster ? paged_attn_kernel<kBf16, kLucid, true> : paged_attn_kernel<kBf16, kLucid, false>;
  static SmemOnce once[2];
  cudaError_t e = once[cluster].set(reinterpret_cast<const void*>(kernel), bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(args.splits, args.Hkv * ((args.G + 15) / 16), args.B);
  cfg.blockDim = dim3(kPaWarps * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = args.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  if ((e = cudaLaunchKernelEx(&cfg, kernel, args)) != cudaSuccess || cluster) return e;
  // the second kernel's CTAs may start while the first one's are still at work; they wait for them on the device
  cfg.gridDim = dim3(args.G, args.Hkv, args.B);
  cfg.blockDim = dim3(128 * kJoinGroups);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<kBf16, kLucid>, args);
}

cudaError_t launch_paged_attn(bool bf16, bool lucid, const PagedAttnArgs& args, cudaStream_t stream) {
  if (bf16) return lucid ? launch_typed<true, true>(args, stream) : launch_typed<true, false>(args, stream);
  return lucid ? launch_typed<false, true>(args, stream) : launch_typed<false, false>(args, stream);
}

cudaError_t paged_attn_status(cudaStream_t stream, int out[8]) { return take_status(&g_paged_ctl, stream, out); }

}  // namespace lucid
