// C ABI of the windowed attention, the paged cache and its readers: argument checks, tensor maps and launches.
#include <math.h>
#include <string.h>

#include "attn.h"
#include "host.h"

namespace lucid {

static bool good_scale(float s) { return s > 0.0f && s < 1e18f; }

static int make_shape(AttnShape* a, const lucid_window_attn_desc* d) {
  if (!d) return LUCID_E_NULL_POINTER;
  const int B = d->B, Nq = d->Nq, Nk = d->Nk, Hq = d->Hq, Hkv = d->Hkv, D = d->D, dtype = d->dtype, window = d->window,
            sinks = d->sinks;
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

static size_t stat_bytes(const AttnShape& a) { return (size_t)a.B * a.Hq * a.nqb * 2 * kBlock * sizeof(float); }
static size_t partial_bytes(const AttnShape& a) {
  const int c = sink_chunks(a);
  return c ? (size_t)a.B * a.Hkv * (1 + c) * 2 * a.S * kBlock * sizeof(float) : 0;
}

static int check_cache(const lucid_paged_cache_desc* c, int B, int Hkv, const void* k, const void* v, const int32_t* table,
                       PagedCache* out) {
  if (!k || !v || !table) return LUCID_E_NULL_POINTER;
  if (c->pages <= 0 || c->table_width <= 0 || c->page_rows <= 0 || c->page_rows > 65536 ||
      (c->page_rows & (c->page_rows - 1)))
    return LUCID_E_BAD_PAGE;
  if ((long long)c->table_width * c->page_rows > (1ll << 30)) return LUCID_E_BAD_SHAPE;
  int rc;
  // {page, row, head} strides; their extents
  if ((rc = check_tensor(k, c->k_strides, c->pages, c->page_rows, Hkv))) return rc;
  if ((rc = check_tensor(v, c->v_strides, c->pages, c->page_rows, Hkv))) return rc;
  if (B > 1 && c->table_stride < c->table_width) return LUCID_E_BAD_STRIDE;
  out->k = const_cast<void*>(k);
  out->v = const_cast<void*>(v);
  out->k_page = c->k_strides[0];
  out->k_row = c->k_strides[1];
  out->k_head = c->k_strides[2];
  out->v_page = c->v_strides[0];
  out->v_row = c->v_strides[1];
  out->v_head = c->v_strides[2];
  out->table = table;
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
// lengths.  A cluster's worth (8, or what leaves a chunk 64 keys) where that fills the SMs or the keys are so few that a second launch
// costs more than it gains; otherwise one wave of CTAs.
static int paged_splits(int B, int Hkv, int G, long long keys) {
  int sms = sm_count();
  if (sms <= 0) {
    (void)cudaGetLastError();
    sms = 148;
  }
  const long long base = (long long)B * Hkv * ((G + 15) / 16), wave = (long long)kPagedPerSm * sms;
  const long long full = (wave + base - 1) / base;
  if (full <= kPagedCluster || keys <= 4096) {
    int n = 1;
    while (n < kPagedCluster && n * 64 < keys) n *= 2;
    return n;
  }
  long long n = full, most = (keys + 255) / 256;
  if (n > most) n = most;
  return (int)(n > kPagedMaxSplits ? kPagedMaxSplits : n);
}
static int paged_splits(const lucid_paged_attn_desc* d, bool lucid_step) {
  long long keys = (long long)d->cache.page_rows * d->cache.table_width;
  if (!lucid_step && d->window >= 0 && keys > (long long)d->window + d->sinks) keys = (long long)d->window + d->sinks;
  return paged_splits(d->B, d->Hkv, d->Hq / d->Hkv, keys);
}

}  // namespace lucid

using namespace lucid;

extern "C" {

int lucid_window_attn_fwd(const lucid_window_attn_desc* d, const void* q, const void* k, const void* v, void* out,
                          void* rest, float* lse, const int32_t* lengths, void* cuda_stream) {
  AttnFwdArgs args;
  int rc;
  if ((rc = make_shape(&args.a, d))) return rc;
  if (!good_scale(d->scale)) return LUCID_E_BAD_SCALE;
  const int B = d->B, Nq = d->Nq, Nk = d->Nk, Hq = d->Hq, Hkv = d->Hkv;
  if ((rc = check_tensor(q, d->q_strides, B, Nq, Hq)) || (rc = check_tensor(k, d->k_strides, B, Nk, Hkv)) ||
      (rc = check_tensor(v, d->v_strides, B, Nk, Hkv)) || (rc = check_tensor(out, d->out_strides, B, Nq, Hq)))
    return rc;
  if (rest && !lse) return LUCID_E_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(rest) % 16) return LUCID_E_BAD_ALIGNMENT;
  const int sms = sm_count();
  if (sms <= 0) return LUCID_E_NO_DEVICE;
  const bool bf16 = d->dtype == LUCID_DTYPE_BF16;
  CUtensorMap tm_q, tm_k, tm_v;
  if ((rc = bshd_map(&tm_q, bf16, q, d->q_strides, B, Nq, Hq, 128)) || (rc = bshd_map(&tm_k, bf16, k, d->k_strides, B, Nk, Hkv, 128)) ||
      (rc = bshd_map(&tm_v, bf16, v, d->v_strides, B, Nk, Hkv, 128)))
    return rc;
  args.lengths = lengths;
  args.out = out;
  args.out_strides = Strides{d->out_strides[0], d->out_strides[1], d->out_strides[2]};
  args.rest = rest;
  args.lse = lse;
  args.scale_log2 = d->scale * kLog2e;
  args.wait_ns = wait_limit_ns();
  // (inference) single tiles with split keys where all of them fit the SMs at once: a CTA then has half as many steps in a row
  args.split = !lse && fwd_items(args.a, true) <= sms ? 1 : 0;
  args.parts = args.split ? fwd_parts(args.a, bf16, sms) : 1;
  return (int)launch_attn_fwd(bf16, tm_q, tm_k, tm_v, args, sms, static_cast<cudaStream_t>(cuda_stream));
}

size_t lucid_window_attn_rest_bytes(const lucid_window_attn_desc* d) {
  AttnShape a;
  if (make_shape(&a, d)) return 0;
  return (size_t)a.B * a.Hq * a.nqb * rest_rows(a) * kBlock * 2;
}

size_t lucid_window_attn_bwd_workspace_bytes(const lucid_window_attn_desc* d) {
  AttnShape a;
  if (make_shape(&a, d)) return 0;
  return stat_bytes(a) + partial_bytes(a);
}

int lucid_window_attn_bwd(const lucid_window_attn_desc* d, const void* q, const void* k, const void* v, const void* out,
                          const void* rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, const int32_t* lengths,
                          void* workspace, size_t workspace_bytes, void* cuda_stream) {
  AttnBwdArgs args;
  memset(&args, 0, sizeof(args));
  int rc;
  if ((rc = make_shape(&args.a, d))) return rc;
  if (!good_scale(d->scale)) return LUCID_E_BAD_SCALE;
  const int B = d->B, Nq = d->Nq, Nk = d->Nk, Hq = d->Hq, Hkv = d->Hkv;
  if ((rc = check_tensor(q, d->q_strides, B, Nq, Hq)) || (rc = check_tensor(k, d->k_strides, B, Nk, Hkv)) ||
      (rc = check_tensor(v, d->v_strides, B, Nk, Hkv)) || (rc = check_tensor(out, d->out_strides, B, Nq, Hq)) ||
      (rc = check_tensor(dout, d->dout_strides, B, Nq, Hq)))
    return rc;
  if (dq && (rc = check_tensor(dq, d->dq_strides, B, Nq, Hq))) return rc;
  if ((dk == nullptr) != (dv == nullptr)) return LUCID_E_NULL_POINTER;
  if (dk && ((rc = check_tensor(dk, d->dk_strides, B, Nk, Hkv)) || (rc = check_tensor(dv, d->dv_strides, B, Nk, Hkv)))) return rc;
  if (!lse || !workspace) return LUCID_E_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 || reinterpret_cast<uintptr_t>(rest) % 16) return LUCID_E_BAD_ALIGNMENT;
  if (workspace_bytes < stat_bytes(args.a) + partial_bytes(args.a)) return LUCID_E_WORKSPACE_TOO_SMALL;
  const int sms = sm_count();
  if (sms <= 0) return LUCID_E_NO_DEVICE;
  const bool bf16 = d->dtype == LUCID_DTYPE_BF16;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  CUtensorMap tm_q, tm_k, tm_v, tm_do;
  if ((rc = bshd_map(&tm_q, bf16, q, d->q_strides, B, Nq, Hq, 128)) || (rc = bshd_map(&tm_k, bf16, k, d->k_strides, B, Nk, Hkv, 128)) ||
      (rc = bshd_map(&tm_v, bf16, v, d->v_strides, B, Nk, Hkv, 128)) ||
      (rc = bshd_map(&tm_do, bf16, dout, d->dout_strides, B, Nq, Hq, 128)))
    return rc;
  float* stat = static_cast<float*>(workspace);
  AttnStatArgs sa;
  sa.a = args.a;
  sa.lengths = lengths;
  sa.out = out;
  sa.rest = rest;
  sa.dout = dout;
  sa.out_strides = Strides{d->out_strides[0], d->out_strides[1], d->out_strides[2]};
  sa.dout_strides = Strides{d->dout_strides[0], d->dout_strides[1], d->dout_strides[2]};
  sa.lse = lse;
  sa.stat = stat;
  cudaError_t e = launch_attn_stat(bf16, sa, stream);
  if (e != cudaSuccess) return (int)e;
  args.lengths = lengths;
  args.stat = stat;
  args.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + stat_bytes(args.a));
  args.chunks = sink_chunks(args.a);
  args.scale = d->scale;
  args.scale_log2 = d->scale * kLog2e;
  args.wait_ns = wait_limit_ns();
  if (dq) {
    args.dq = dq;
    args.dq_strides = Strides{d->dq_strides[0], d->dq_strides[1], d->dq_strides[2]};
    if ((e = launch_attn_dq(bf16, tm_q, tm_k, tm_v, tm_do, args, sms, stream)) != cudaSuccess) return (int)e;
  }
  if (dk) {
    args.after_dq = dq ? 1 : 0;
    args.dk = dk;
    args.dv = dv;
    args.dk_strides = Strides{d->dk_strides[0], d->dk_strides[1], d->dk_strides[2]};
    args.dv_strides = Strides{d->dv_strides[0], d->dv_strides[1], d->dv_strides[2]};
    if ((e = launch_attn_dkv(bf16, tm_q, tm_k, tm_v, tm_do, args, sms, stream)) != cudaSuccess) return (int)e;
  }
  return 0;
}

int lucid_paged_append(const lucid_paged_append_desc* d, const void* k, const void* v, const void* q, void* q_out,
                       void* k_cache, void* v_cache, const int32_t* block_table, const int32_t* cache_lens,
                       const int32_t* cu_seqlens, const float* inv_freq, void* cuda_stream) {
  AppendArgs args;
  memset(&args, 0, sizeof(args));
  int rc;
  if (!d) return LUCID_E_NULL_POINTER;
  const int B = d->B, T = d->T, Hq = d->Hq, Hkv = d->Hkv;
  if (B <= 0 || T <= 0 || Hkv <= 0 || d->D != kBlock || (q && Hq <= 0)) return LUCID_E_BAD_SHAPE;
  if (!cu_seqlens && T != B) return LUCID_E_BAD_SHAPE;
  if ((long long)T * (2 * (long long)Hkv + (q ? Hq : 0)) > (1ll << 31)) return LUCID_E_BAD_SHAPE;
  if (d->dtype != LUCID_DTYPE_FP16 && d->dtype != LUCID_DTYPE_BF16) return LUCID_E_BAD_DTYPE;
  if (inv_freq && (d->rotated <= 0 || d->rotated > d->D || d->rotated % 16)) return LUCID_E_BAD_ROTATION;
  if (!cache_lens || (q && (!q_out || !inv_freq))) return LUCID_E_NULL_POINTER;
  if ((rc = check_cache(&d->cache, B, Hkv, k_cache, v_cache, block_table, &args.c))) return rc;
  if ((rc = check_rows(k, d->k_strides, T, Hkv))) return rc;
  if (v && (rc = check_rows(v, d->v_strides, T, Hkv))) return rc;
  if (q && ((rc = check_rows(q, d->q_strides, T, Hq)) || reinterpret_cast<uintptr_t>(q_out) % 16))
    return rc ? rc : LUCID_E_BAD_ALIGNMENT;
  const int sms = sm_count();
  if (sms <= 0) return LUCID_E_NO_DEVICE;
  args.k = k;
  args.v = v;
  args.q = q;
  args.q_out = q_out;
  args.k_tok = d->k_strides[0];
  args.k_head = d->k_strides[1];
  if (v) {
    args.v_tok = d->v_strides[0];
    args.v_head = d->v_strides[1];
  }
  if (q) {
    args.q_tok = d->q_strides[0];
    args.q_head = d->q_strides[1];
  }
  args.cache_lens = cache_lens;
  args.cu = cu_seqlens;
  args.inv_freq = inv_freq;
  args.B = B;
  args.T = T;
  args.Hq = q ? Hq : 0;
  args.Hkv = Hkv;
  args.rot = inv_freq ? d->rotated : 0;
  args.interleaved = d->interleaved ? 1 : 0;
  return (int)launch_paged_append(d->dtype == LUCID_DTYPE_BF16, args, sms, static_cast<cudaStream_t>(cuda_stream));
}

size_t lucid_paged_attn_workspace_bytes(const lucid_paged_attn_desc* d, int lucid_step) {
  if (!d || d->B <= 0 || d->Hkv <= 0 || d->Hq <= 0 || d->Hq % d->Hkv || d->cache.page_rows <= 0 || d->cache.table_width <= 0)
    return 0;
  return paged_attn_partial_bytes(d->B, d->Hq, d->Hkv, lucid_step != 0, paged_splits(d, lucid_step != 0));
}

static int paged_attn(const lucid_paged_attn_desc* d, const void* q, const void* v_new, void* out, const void* k_cache,
                      const void* v_cache, const int32_t* table, const int32_t* seq_lens, bool lucid_step, void* workspace,
                      size_t workspace_bytes, void* cuda_stream) {
  PagedAttnArgs args;
  memset(&args, 0, sizeof(args));
  int rc;
  if (!d) return LUCID_E_NULL_POINTER;
  const int B = d->B, Hq = d->Hq, Hkv = d->Hkv;
  if (B <= 0 || B > 65535 || Hq <= 0 || Hkv <= 0 || d->D != kBlock || (!lucid_step && d->sinks < 0)) return LUCID_E_BAD_SHAPE;
  if (Hq % Hkv || (lucid_step && Hq / Hkv > 15)) return LUCID_E_BAD_HEADS;
  const int G = Hq / Hkv;
  if ((long long)Hkv * ((G + 15) / 16) > 65535) return LUCID_E_BAD_HEADS;
  if (d->dtype != LUCID_DTYPE_FP16 && d->dtype != LUCID_DTYPE_BF16) return LUCID_E_BAD_DTYPE;
  if (!good_scale(d->scale) || (lucid_step && !good_scale(d->k_scale))) return LUCID_E_BAD_SCALE;
  if (!seq_lens || !out) return LUCID_E_NULL_POINTER;
  if ((rc = check_cache(&d->cache, B, Hkv, k_cache, v_cache, table, &args.c))) return rc;
  if ((rc = check_rows(q, d->q_strides, B, Hq))) return rc;
  if (lucid_step && (rc = check_rows(v_new, d->v_strides, B, Hkv))) return rc;
  if (reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16) return LUCID_E_BAD_ALIGNMENT;
  args.splits = paged_splits(d, lucid_step);
  const size_t need = paged_attn_partial_bytes(B, Hq, Hkv, lucid_step, args.splits);
  if (need && !workspace) return LUCID_E_NULL_POINTER;
  if (workspace_bytes < need) return LUCID_E_WORKSPACE_TOO_SMALL;
  if (sm_count() <= 0) return LUCID_E_NO_DEVICE;
  args.q = q;
  args.q_b = d->q_strides[0];
  args.q_h = d->q_strides[1];
  args.v_new = v_new;
  if (lucid_step) {
    args.v_b = d->v_strides[0];
    args.v_h = d->v_strides[1];
  }
  args.out = out;
  args.lens = seq_lens;
  args.partial = static_cast<float*>(workspace);
  args.B = B;
  args.Hq = Hq;
  args.Hkv = Hkv;
  args.G = G;
  args.W = lucid_step || d->window < 0 ? kNoWindow : d->window;
  args.S = lucid_step ? 0 : d->sinks;
  args.scale_log2 = d->scale * kLog2e;
  args.lucid_log2 = lucid_step ? d->k_scale * d->k_scale * kLog2e : 0.0f;
  return (int)launch_paged_attn(d->dtype == LUCID_DTYPE_BF16, lucid_step, args, static_cast<cudaStream_t>(cuda_stream));
}

int lucid_paged_window_attn(const lucid_paged_attn_desc* desc, const void* q, void* out, const void* k_cache,
                            const void* v_cache, const int32_t* block_table, const int32_t* seq_lens, void* workspace,
                            size_t workspace_bytes, void* cuda_stream) {
  return paged_attn(desc, q, nullptr, out, k_cache, v_cache, block_table, seq_lens, false, workspace, workspace_bytes,
                    cuda_stream);
}

int lucid_paged_lucid_attn(const lucid_paged_attn_desc* desc, const void* q, const void* v, void* out, const void* k_cache,
                           void* v_cache, const int32_t* block_table, const int32_t* seq_lens, void* workspace,
                           size_t workspace_bytes, void* cuda_stream) {
  return paged_attn(desc, q, v, out, k_cache, v_cache, block_table, seq_lens, true, workspace, workspace_bytes, cuda_stream);
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
