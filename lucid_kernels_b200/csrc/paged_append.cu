// Appends new tokens' keys and values to a paged cache, rotating keys (and the tokens' queries) by their position on
// the way:  (x1, x2) -> (x1 cos a - x2 sin a, x2 cos a + x1 sin a),  a = position * inv_freq.
//
// Bound by HBM (each row is read once and written once) or, for a handful of tokens, by latency.  A warp owns one token
// and some of its heads, four head rows at a time, 8 lanes a row, each lane the two 16-byte pieces that rotate into
// one another.  The angle is a product in 64 bits reduced to a fraction of a turn there: at position 10^6 a product in 32
// bits is off by up to 0.03 radians (half of its spacing there, 2^-4).  Tables of sines would be 512 bytes to read per token; computing them costs a lane
// two angles per token.
#include <type_traits>
#include "attn.h"

namespace lucid {

static __device__ Control g_append_ctl;

constexpr int kApWarps = 4, kAhead = 4;

// Last b with cu[b] <= tok < cu[b + 1], or -1 (behind the last sequence).  Whole warp; a 32-way search.
__device__ __forceinline__ int find_sequence(const int* cu, int B, int tok, int lane) {
  int lo = 0, n = B;                                  // the answer, if any, is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int at = lo + lane * step;                  // first sequence of this lane's piece
    const bool past = lane * step < n && __ldg(cu + at) <= tok;
    const unsigned m = __ballot_sync(0xffffffffu, past);
    if (m == 0) return -1;
    const int last = 31 - __clz(m);
    const int nlo = lo + last * step;
    n = imin(step, lo + n - nlo);
    lo = nlo;
  }
  return (tok >= __ldg(cu + lo) && tok < __ldg(cu + lo + 1)) ? lo : -1;
}

template <bool kBf16>
__device__ __forceinline__ void rotate_pieces(uint4& a, uint4& b, const float2* cs, int ca, int cb, bool interleaved) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
  uint32_t* pb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 x = unpack2<kBf16>(pa[e]), y = unpack2<kBf16>(pb[e]);
    if (interleaved) {                                // pairs (2i, 2i + 1): both pieces rotate within themselves
      const float2 r = cs[4 * ca + e], t = cs[4 * cb + e];
      pa[e] = pack2<kBf16>(x.x * r.x - x.y * r.y, x.y * r.x + x.x * r.y);
      pb[e] = pack2<kBf16>(y.x * t.x - y.y * t.y, y.y * t.x + y.x * t.y);
    } else {                                          // pairs (i, i + rot / 2)
      const float2 r = cs[8 * ca + 2 * e], t = cs[8 * ca + 2 * e + 1];
      pa[e] = pack2<kBf16>(x.x * r.x - y.x * r.y, x.y * t.x - y.y * t.y);
      pb[e] = pack2<kBf16>(y.x * r.x + x.x * r.y, y.y * t.x + x.y * t.y);
    }
  }
}

template <bool kBf16>
__global__ void __launch_bounds__(kApWarps * 32) paged_append_kernel(const AppendArgs args, int parts) {
  typedef typename std::conditional<kBf16, __nv_bfloat16, __half>::type elem_t;
  __shared__ float2 cs_all[kApWarps][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * kApWarps + warp;
  const int tok = (int)(unit / parts), part = (int)(unit % parts);
  if (tok >= args.T) return;
  // rows of the token: Hkv keys, Hkv values, Hq queries; a lane's two pieces of its row in each of kAhead rounds are
  // requested first, everything that says where they go and how they turn is worked out meanwhile
  const int half = args.inv_freq ? args.rot / 16 : 0, l8 = lane & 7;
  const bool turn = l8 < half;
  const int ca = turn ? l8 : 2 * half + 2 * (l8 - half), cb = turn ? l8 + half : ca + 1;
  const int nv = args.v ? args.Hkv : 0, rows = args.Hkv + nv + (args.q ? args.Hq : 0);
  const int row0 = part * 4 + (lane >> 3), step = parts * 4;
  auto source = [&](int r) -> const elem_t* {
    if (r < args.Hkv) return reinterpret_cast<const elem_t*>(args.k) + tok * args.k_tok + r * args.k_head;
    if (r < args.Hkv + nv) return reinterpret_cast<const elem_t*>(args.v) + tok * args.v_tok + (r - args.Hkv) * args.v_head;
    return reinterpret_cast<const elem_t*>(args.q) + tok * args.q_tok + (r - args.Hkv - nv) * args.q_head;
  };
  uint4 x[kAhead], y[kAhead];
  auto request = [&](int r) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (r + e * step >= rows) break;
      const elem_t* src = source(r + e * step);
      x[e] = *reinterpret_cast<const uint4*>(src + 8 * ca);
      y[e] = *reinterpret_cast<const uint4*>(src + 8 * cb);
    }
  };
  request(row0);
  const int b = args.cu ? find_sequence(args.cu, args.B, tok, lane) : tok;
  long long pos = -1;
  if (b >= 0) pos = (long long)__ldg(args.cache_lens + b) + (args.cu ? tok - __ldg(args.cu + b) : 0);
  // the row of the cache this token goes to
  const PagedCache& c = args.c;
  long long page = -1;
  if (pos >= 0 && (pos >> c.page_shift) < c.table_width) page = __ldg(c.table + b * c.table_stride + (pos >> c.page_shift));
  const bool ok = page >= 0 && page < c.pages;
  if (b >= 0 && !ok && lane == 0 && part == 0) report_error(&g_append_ctl, kErrBadPage, b, tok, (int)pos, 0);
  const long long slot = ok ? (pos & ((1 << c.page_shift) - 1)) : 0;
  float2* cs = cs_all[warp];
  if (args.inv_freq && b >= 0) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = lane + 32 * e;
      if (i < args.rot / 2) {
        // fraction of a turn, then the functions of pi times it
        const double turns = (double)pos * (double)__ldg(args.inv_freq + i) * 0.15915494309189533577;
        float sn, cn;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
        cs[i] = make_float2(cn, sn);
      }
    }
  }
  __syncwarp();
  for (int r = row0; r < rows; r += kAhead * step) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int re = r + e * step;
      if (re >= rows) break;
      elem_t* dst = nullptr;
      if (re < args.Hkv) {
        if (ok) dst = reinterpret_cast<elem_t*>(c.k) + page * c.k_page + slot * c.k_row + re * c.k_head;
      } else if (re < args.Hkv + nv) {
        if (ok) dst = reinterpret_cast<elem_t*>(c.v) + page * c.v_page + slot * c.v_row + (re - args.Hkv) * c.v_head;
      } else {
        dst = reinterpret_cast<elem_t*>(args.q_out) + ((long long)tok * args.Hq + re - args.Hkv - nv) * 128;
      }
      if (!dst) continue;
      if (b < 0) x[e] = y[e] = make_uint4(0, 0, 0, 0);        // queries behind the last sequence come back as zeros
      else if (turn && (re < args.Hkv || re >= args.Hkv + nv)) rotate_pieces<kBf16>(x[e], y[e], cs, ca, cb, args.interleaved != 0);
      *reinterpret_cast<uint4*>(dst + 8 * ca) = x[e];
      *reinterpret_cast<uint4*>(dst + 8 * cb) = y[e];
    }
    request(r + kAhead * step);
  }
}

// A warp takes four head rows of a token, or all of them.  Four, while the warps that makes fit the SMs at once (80 registers: six
// CTAs an SM) as often as a warp with all rows has rounds of kAhead to do; beyond that its repeated lookups cost more than
// its shorter chain saves.  Four against all, us, 8/4 query/key heads: 8 tokens 3.0 and 3.9, 768 4.1 and 4.7, 1024 5.6 and 4.7,
// 3500 11.5 and 7.0, 9000 25.4 and 14.9; 32/8 heads: 640 7.8 and 8.2, 1024 10.4 and 8.2; 4/1 heads: 1536 4.1 and 4.3,
// 2048 5.7 and 4.6.
constexpr int kApPerSm = 6;

cudaError_t launch_paged_append(bool bf16, const AppendArgs& args, int sms, cudaStream_t stream) {
  const int rows = args.Hkv + (args.v ? args.Hkv : 0) + (args.q ? args.Hq : 0);
  const int groups = (rows + 3) / 4;
  const int parts = (long long)args.T * imin(groups, kAhead) <= (long long)kApPerSm * kApWarps * sms ? groups : 1;
  const long long units = (long long)args.T * parts;
  const unsigned grid = (unsigned)((units + kApWarps - 1) / kApWarps);
  if (bf16) paged_append_kernel<true><<<grid, kApWarps * 32, 0, stream>>>(args, parts);
  else paged_append_kernel<false><<<grid, kApWarps * 32, 0, stream>>>(args, parts);
  return cudaGetLastError();
}

cudaError_t paged_append_status(cudaStream_t stream, int out[8]) { return take_status(&g_append_ctl, stream, out); }

}  // namespace lucid
