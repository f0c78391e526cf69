// C ABI of the windowed attention, the paged cache and its readers: argument checks, tensor maps and launches.
#include <math.h>
#include <string.h>

#include "attn.h"
#include "host.h"

namespace lucid {

static bool good_scale(float s) { return s > 0.0f && s < 1e18f; }

static int make_shape(AttnShape* a, int B, int Nq, int Nk, int Hq, int Hkv, int D, int dtype, int window, int sinks) {
  if (B <= 0 || Nq <= 0 || Nk < Nq || Hq <= 0 || Hkv <= 0 || D != kBlock || Nk > (1 << 28)) return LUCID_E_BAD_SHAPE;
  if (Hq % Hkv) return LUCID_E_BAD_HEADS;
  if (sinks < 0 || sinks > kMaxSinks) return LUCID_E_BAD_SHAPE;
  if (dtype != LUCID_DTYPE_FP16 && dtype != LUCID_DTYPE_BF16) return LUCID_E_BAD_DTYPE;
  if ((long long)B * Hq * ((Nk + 127) / 128 + 2) > (1ll << 30) / kBlock) return LUCID_E_BAD_SHAPE;
  a->B = B;
  a->Nq = Nq;
  a->Nk = Nk;
  a->Hq = Hq;
  a->Hkv = Hkv;
  a->G = Hq / Hkv;
  a->off = Nk - Nq;
  // a window as long as the keys hides nothing
  a->W = window < 0 || window >= Nk ? kNoWindow : window;
  a->S = a->W == kNoWindow ? 0 : sinks;
  a->nqb = (Nq + 127) / 128;
  a->nkb = (Nk + 127) / 128;
  return 0;
}

static size_t stat_bytes(const AttnShape& a) { return (size_t)a.B * a.Hq * a.nqb * kBlock * sizeof(float2); }
static size_t partial_bytes(const AttnShape& a) {
  const int c = sink_chunks(a);
  return c ? (size_t)a.B * a.Hkv * (1 + c) * 2 * a.S * kBlock * sizeof(float) : 0;
}

static int check_cache(const lucid_paged_cache* c, int B, int Hkv, PagedCache* out) {
  if (!c || !c->k || !c->v || !c->block_table) return LUCID_E_NULL_POINTER;
  if (c->pages <= 0 || c->table_width <= 0 || c->page_rows <= 0 || c->page_rows > 65536 ||
      (c->page_rows & (c->page_rows - 1)))
    return LUCID_E_BAD_PAGE;
  if ((long long)c->table_width * c->page_rows > (1ll << 30)) return LUCID_E_BAD_SHAPE;
  int rc;
  // {page, row, head} strides; their extents
  if ((rc = check_tensor(c->k, c->k_strides, c->pages, c->page_rows, Hkv))) return rc;
  if ((rc = check_tensor(c->v, c->v_strides, c->pages, c->page_rows, Hkv))) return rc;
  if (B > 1 && c->table_stride < c->table_width) return LUCID_E_BAD_STRIDE;
  out->k = c->k;
  out->v = c->v;
  out->k_page = c->k_strides[0];
  out->k_row = c->k_strides[1];
  out->k_head = c->k_strides[2];
  out->v_page = c->v_strides[0];
  out->v_row = c->v_strides[1];
  out->v_head = c->v_strides[2];
  out->table = c->block_table;
  out->table_stride = c->table_stride;
  out->table_width = c->table_width;
  out->pages = c->pages;
  out->page_shift = 0;
  while ((1 << out->page_shift) < c->page_rows) ++out->page_shift;
  return 0;
}

// rows of tokens: {token, head} strides, 16-byte pieces
static int check_rows(const void* p, const int64_t st[2], long long T, int H) {
  if (!p || !st) return LUCID_E_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(p) % 16) return LUCID_E_BAD_ALIGNMENT;
  if (st[0] < 0 || st[1] < 0 || (T > 1 && st[0] % 8) || (H > 1 && st[1] % 8)) return LUCID_E_BAD_ALIGNMENT;
  return 0;
}

// How many chunks a sequence's keys are dealt out in, from what the host knows: the capacity of the block table, not the
// lengths.  One wave of CTAs (two per SM) at least; with several sequences up to four, because their lengths differ and
// the longest would run alone at the end; no chunk under 256 keys while that still fills the SMs, under 64 ever.
static int paged_splits(int B, int Hkv, int G, long long keys) {
  int sms = sm_count();
  if (sms <= 0) {
    (void)cudaGetLastError();
    sms = 148;
  }
  const long long base = (long long)B * Hkv * ((G + 15) / 16), wave = 2ll * sms;
  long long n = (wave + base - 1) / base;
  if (B > 1) {
    long long more = (4 * wave + base - 1) / base;
    if (more > 32) more = 32;
    if (more > n) n = more;
  }
  const long long by256 = (keys + 255) / 256, by64 = (keys + 63) / 64;
  long long most = by256;
  if (base * by256 < wave) most = by64 < (wave + base - 1) / base ? by64 : (wave + base - 1) / base;
  if (n > most) n = most;
  if (n > 128) n = 128;
  return n < 1 ? 1 : (int)n;
}
static long long paged_keys(int page_rows, int table_width, int window, int sinks, bool lucid) {
  const long long cap = (long long)page_rows * table_width;
  if (lucid || window < 0) return cap;
  return cap < (long long)window + sinks ? cap : (long long)window + sinks;
}

}  // namespace lucid

using namespace lucid;

extern "C" {

int lucid_window_attn_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int64_t q_strides[3],
                          const int64_t k_strides[3], const int64_t v_strides[3], const int64_t out_strides[3], int B,
                          int Nq, int Nk, int Hq, int Hkv, int D, int dtype, int window, int sinks, float scale,
                          const int32_t* lengths, void* cuda_stream) {
  AttnFwdArgs args;
  int rc;
  if ((rc = make_shape(&args.a, B, Nq, Nk, Hq, Hkv, D, dtype, window, sinks))) return rc;
  if (!good_scale(scale)) return LUCID_E_BAD_SCALE;
  if ((rc = check_tensor(q, q_strides, B, Nq, Hq)) || (rc = check_tensor(k, k_strides, B, Nk, Hkv)) ||
      (rc = check_tensor(v, v_strides, B, Nk, Hkv)) || (rc = check_tensor(out, out_strides, B, Nq, Hq)))
    return rc;
  if (!lse) return LUCID_E_NULL_POINTER;
  const int sms = sm_count();
  if (sms <= 0) return LUCID_E_NO_DEVICE;
  const bool bf16 = dtype == LUCID_DTYPE_BF16;
  CUtensorMap tm_q, tm_k, tm_v;
  if ((rc = bshd_map(&tm_q, bf16, q, q_strides, B, Nq, Hq, 128)) || (rc = bshd_map(&tm_k, bf16, k, k_strides, B, Nk, Hkv, 128)) ||
      (rc = bshd_map(&tm_v, bf16, v, v_strides, B, Nk, Hkv, 128)))
    return rc;
  args.lengths = lengths;
  args.out = out;
  args.out_strides = Strides{out_strides[0], out_strides[1], out_strides[2]};
  args.lse = lse;
  args.scale_log2 = scale * kLog2e;
  args.wait_ns = wait_limit_ns();
  return (int)launch_attn_fwd(bf16, tm_q, tm_k, tm_v, args, sms, static_cast<cudaStream_t>(cuda_stream));
}

size_t lucid_window_attn_bwd_workspace_bytes(int B, int Nq, int Nk, int Hq, int Hkv, int window, int sinks) {
  AttnShape a;
  if (make_shape(&a, B, Nq, Nk, Hq, Hkv, kBlock, LUCID_DTYPE_BF16, window, sinks)) return 0;
  return stat_bytes(a) + partial_bytes(a);
}

int lucid_window_attn_bwd(const void* q, const void* k, const void* v, const void* out, const float* lse, const void* dout,
                          void* dq, void* dk, void* dv, const int64_t q_strides[3], const int64_t k_strides[3],
                          const int64_t v_strides[3], const int64_t out_strides[3], const int64_t dout_strides[3],
                          const int64_t dq_strides[3], const int64_t dk_strides[3], const int64_t dv_strides[3], int B, int Nq,
                          int Nk, int Hq, int Hkv, int D, int dtype, int window, int sinks, float scale,
                          const int32_t* lengths, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  AttnBwdArgs args;
  memset(&args, 0, sizeof(args));
  int rc;
  if ((rc = make_shape(&args.a, B, Nq, Nk, Hq, Hkv, D, dtype, window, sinks))) return rc;
  if (!good_scale(scale)) return LUCID_E_BAD_SCALE;
  if ((rc = check_tensor(q, q_strides, B, Nq, Hq)) || (rc = check_tensor(k, k_strides, B, Nk, Hkv)) ||
      (rc = check_tensor(v, v_strides, B, Nk, Hkv)) || (rc = check_tensor(out, out_strides, B, Nq, Hq)) ||
      (rc = check_tensor(dout, dout_strides, B, Nq, Hq)))
    return rc;
  if (dq && (rc = check_tensor(dq, dq_strides, B, Nq, Hq))) return rc;
  if ((dk == nullptr) != (dv == nullptr)) return LUCID_E_NULL_POINTER;
  if (dk && ((rc = check_tensor(dk, dk_strides, B, Nk, Hkv)) || (rc = check_tensor(dv, dv_strides, B, Nk, Hkv)))) return rc;
  if (!lse || !workspace) return LUCID_E_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return LUCID_E_BAD_ALIGNMENT;
  if (workspace_bytes < stat_bytes(args.a) + partial_bytes(args.a)) return LUCID_E_WORKSPACE_TOO_SMALL;
  const int sms = sm_count();
  if (sms <= 0) return LUCID_E_NO_DEVICE;
  const bool bf16 = dtype == LUCID_DTYPE_BF16;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  CUtensorMap tm_q, tm_k, tm_v, tm_do;
  if ((rc = bshd_map(&tm_q, bf16, q, q_strides, B, Nq, Hq, 128)) || (rc = bshd_map(&tm_k, bf16, k, k_strides, B, Nk, Hkv, 128)) ||
      (rc = bshd_map(&tm_v, bf16, v, v_strides, B, Nk, Hkv, 128)) ||
      (rc = bshd_map(&tm_do, bf16, dout, dout_strides, B, Nq, Hq, 128)))
    return rc;
  float2* stat = static_cast<float2*>(workspace);
  AttnStatArgs sa;
  sa.a = args.a;
  sa.lengths = lengths;
  sa.out = out;
  sa.dout = dout;
  sa.out_strides = Strides{out_strides[0], out_strides[1], out_strides[2]};
  sa.dout_strides = Strides{dout_strides[0], dout_strides[1], dout_strides[2]};
  sa.lse = lse;
  sa.stat = stat;
  cudaError_t e = launch_attn_stat(bf16, sa, stream);
  if (e != cudaSuccess) return (int)e;
  args.lengths = lengths;
  args.stat = stat;
  args.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + stat_bytes(args.a));
  args.chunks = sink_chunks(args.a);
  args.scale = scale;
  args.scale_log2 = scale * kLog2e;
  args.wait_ns = wait_limit_ns();
  if (dq) {
    args.dq = dq;
    args.dq_strides = Strides{dq_strides[0], dq_strides[1], dq_strides[2]};
    if ((e = launch_attn_dq(bf16, tm_q, tm_k, tm_v, tm_do, args, sms, stream)) != cudaSuccess) return (int)e;
  }
  if (dk) {
    args.dk = dk;
    args.dv = dv;
    args.dk_strides = Strides{dk_strides[0], dk_strides[1], dk_strides[2]};
    args.dv_strides = Strides{dv_strides[0], dv_strides[1], dv_strides[2]};
    if ((e = launch_attn_dkv(bf16, tm_q, tm_k, tm_v, tm_do, args, sms, stream)) != cudaSuccess) return (int)e;
  }
  return 0;
}

int lucid_paged_append(const void* k, const void* v, const void* q, void* q_out, const int64_t k_strides[2],
                       const int64_t v_strides[2], const int64_t q_strides[2], const lucid_paged_cache* cache,
                       const int32_t* cache_lens, const int32_t* cu_seqlens, const float* inv_freq, int B, int T, int Hq,
                       int Hkv, int D, int rotated, int interleaved, int dtype, void* cuda_stream) {
  AppendArgs args;
  memset(&args, 0, sizeof(args));
  int rc;
  if (B <= 0 || T <= 0 || Hkv <= 0 || D != kBlock || (q && Hq <= 0)) return LUCID_E_BAD_SHAPE;
  if (!cu_seqlens && T != B) return LUCID_E_BAD_SHAPE;
  if ((long long)T * (2 * (long long)Hkv + (q ? Hq : 0)) > (1ll << 31)) return LUCID_E_BAD_SHAPE;
  if (dtype != LUCID_DTYPE_FP16 && dtype != LUCID_DTYPE_BF16) return LUCID_E_BAD_DTYPE;
  if (inv_freq && (rotated <= 0 || rotated > D || rotated % 16)) return LUCID_E_BAD_ROTATION;
  if (!cache_lens || (q && (!q_out || !inv_freq))) return LUCID_E_NULL_POINTER;
  if ((rc = check_cache(cache, B, Hkv, &args.c))) return rc;
  if ((rc = check_rows(k, k_strides, T, Hkv))) return rc;
  if (v && (rc = check_rows(v, v_strides, T, Hkv))) return rc;
  if (q && ((rc = check_rows(q, q_strides, T, Hq)) || reinterpret_cast<uintptr_t>(q_out) % 16))
    return rc ? rc : LUCID_E_BAD_ALIGNMENT;
  if (sm_count() <= 0) return LUCID_E_NO_DEVICE;
  args.k = k;
  args.v = v;
  args.q = q;
  args.q_out = q_out;
  args.k_tok = k_strides[0];
  args.k_head = k_strides[1];
  if (v) {
    args.v_tok = v_strides[0];
    args.v_head = v_strides[1];
  }
  if (q) {
    args.q_tok = q_strides[0];
    args.q_head = q_strides[1];
  }
  args.cache_lens = cache_lens;
  args.cu = cu_seqlens;
  args.inv_freq = inv_freq;
  args.B = B;
  args.T = T;
  args.Hq = q ? Hq : 0;
  args.Hkv = Hkv;
  args.rot = inv_freq ? rotated : 0;
  args.interleaved = interleaved ? 1 : 0;
  return (int)launch_paged_append(dtype == LUCID_DTYPE_BF16, args, static_cast<cudaStream_t>(cuda_stream));
}

size_t lucid_paged_attn_workspace_bytes(int B, int Hq, int Hkv, int page_rows, int table_width, int window, int sinks,
                                        int lucid_step) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || page_rows <= 0 || table_width <= 0) return 0;
  const int n = paged_splits(B, Hkv, Hq / Hkv, paged_keys(page_rows, table_width, window, sinks, lucid_step != 0));
  return paged_attn_partial_bytes(B, Hq, Hkv, lucid_step != 0, n);
}

static int paged_attn(const void* q, const void* v_new, void* out, const int64_t q_strides[2], const int64_t v_strides[2],
                      const lucid_paged_cache* cache, const int32_t* seq_lens, int B, int Hq, int Hkv, int D, int dtype,
                      int window, int sinks, float scale, float k_scale, bool lucid_step, void* workspace,
                      size_t workspace_bytes, void* cuda_stream) {
  PagedAttnArgs args;
  memset(&args, 0, sizeof(args));
  int rc;
  if (B <= 0 || B > 65535 || Hq <= 0 || Hkv <= 0 || D != kBlock || sinks < 0) return LUCID_E_BAD_SHAPE;
  if (Hq % Hkv || (lucid_step && Hq / Hkv > 15)) return LUCID_E_BAD_HEADS;
  const int G = Hq / Hkv;
  if ((long long)Hkv * ((G + 15) / 16) > 65535) return LUCID_E_BAD_HEADS;
  if (dtype != LUCID_DTYPE_FP16 && dtype != LUCID_DTYPE_BF16) return LUCID_E_BAD_DTYPE;
  if (!good_scale(scale) || (lucid_step && !good_scale(k_scale))) return LUCID_E_BAD_SCALE;
  if (!seq_lens || !out) return LUCID_E_NULL_POINTER;
  if ((rc = check_cache(cache, B, Hkv, &args.c))) return rc;
  if ((rc = check_rows(q, q_strides, B, Hq))) return rc;
  if (lucid_step && (rc = check_rows(v_new, v_strides, B, Hkv))) return rc;
  if (reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16) return LUCID_E_BAD_ALIGNMENT;
  args.splits = paged_splits(B, Hkv, G, paged_keys(cache->page_rows, cache->table_width, window, sinks, lucid_step));
  const size_t need = paged_attn_partial_bytes(B, Hq, Hkv, lucid_step, args.splits);
  if (need && !workspace) return LUCID_E_NULL_POINTER;
  if (workspace_bytes < need) return LUCID_E_WORKSPACE_TOO_SMALL;
  if (sm_count() <= 0) return LUCID_E_NO_DEVICE;
  args.q = q;
  args.q_b = q_strides[0];
  args.q_h = q_strides[1];
  args.v_new = v_new;
  if (lucid_step) {
    args.v_b = v_strides[0];
    args.v_h = v_strides[1];
  }
  args.out = out;
  args.lens = seq_lens;
  args.partial = static_cast<float*>(workspace);
  args.B = B;
  args.Hq = Hq;
  args.Hkv = Hkv;
  args.G = G;
  args.W = window < 0 ? kNoWindow : window;
  args.S = sinks;
  args.scale_log2 = scale * kLog2e;
  args.lucid_log2 = k_scale * k_scale * kLog2e;
  return (int)launch_paged_attn(dtype == LUCID_DTYPE_BF16, lucid_step, args, static_cast<cudaStream_t>(cuda_stream));
}

int lucid_paged_window_attn(const void* q, void* out, const int64_t q_strides[2], const lucid_paged_cache* cache,
                            const int32_t* seq_lens, int B, int Hq, int Hkv, int D, int dtype, int window, int sinks,
                            float scale, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  return paged_attn(q, nullptr, out, q_strides, nullptr, cache, seq_lens, B, Hq, Hkv, D, dtype, window, sinks, scale, 1.0f,
                    false, workspace, workspace_bytes, cuda_stream);
}

int lucid_paged_lucid_attn(const void* q, const void* v, void* out, const int64_t q_strides[2], const int64_t v_strides[2],
                           const lucid_paged_cache* cache, const int32_t* seq_lens, int B, int Hq, int Hkv, int D, int dtype,
                           float k_scale, float scale, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  return paged_attn(q, v, out, q_strides, v_strides, cache, seq_lens, B, Hq, Hkv, D, dtype, -1, 0, scale, k_scale, true,
                    workspace, workspace_bytes, cuda_stream);
}

int lucid_attn_status(void* cuda_stream, int32_t out[8]) {
  if (!out) return LUCID_E_NULL_POINTER;
  cudaError_t (*const take[4])(cudaStream_t, int*) = {attn_fwd_status, attn_bwd_status, paged_append_status, paged_attn_status};
  memset(out, 0, 8 * sizeof(int32_t));
  for (int i = 0; i < 4; ++i) {
    int st[8];
    const cudaError_t e = take[i](static_cast<cudaStream_t>(cuda_stream), st);
    if (e != cudaSuccess) return (int)e;
    if (st[0] != 0 && out[0] == 0) {
      out[0] = st[0];
      out[1] = i;
      for (int w = 1; w < 6; ++w) out[1 + w] = st[w];
    }
  }
  return 0;
}

}  // extern "C"
