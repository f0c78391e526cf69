// Argument blocks and host launchers of the windowed attention kernels (attn_fwd.cu, attn_bwd.cu) and of the paged
// cache's kernels (paged_append.cu, paged_attn.cu).
#pragma once
#include <atomic>
#include <utility>

#include "attn_geometry.h"
#include "common.cuh"

namespace lucid {

// Device-side errors of these kernels: the first one since the last read, one record per source file and device.
//   kErrBarrierTimeout as in the solve; kErrBadPage: a position whose page is outside the pool or the block table
enum : int { kErrBadPage = 4 };

struct AttnFwdArgs {
  AttnShape a;
  int split;              // (without lse) items are single tiles of queries whose keys are split between the CTA's two halves
  int parts;              // (with split) CTAs of a cluster that share an item's keys: 1, 2, 4 or 8
  const int* lengths;     // (B) valid positions, or null
  void* out;              // (B, Nq, Hq, 128)
  Strides out_strides;
  void* rest;             // or null: (B, Hq, nqb, 16, rest_rows, 8) 16-bit, what the rounding of `out` took off (needs lse)
  float* lse;             // or null; (B, Hq, Nq) natural log of the row's sum of exponentials, -inf for an empty row
  float scale_log2;       // scale * log2(e)
  unsigned long long wait_ns;
};

struct AttnBwdArgs {
  AttnShape a;
  const int* lengths;
  const float* stat;      // (B, Hq, nqb, 2, 128): lse in base 2 (+inf: row without weight), -delta, in the units of attn_stat_kernel
  void* dq;
  Strides dq_strides;
  void *dk, *dv;
  Strides dk_strides, dv_strides;
  float* partial;         // (B * Hkv, 1 + chunks, 2, S, 128) fp32 sums of the first keys' rows {dK, dV}
  int chunks;
  int after_dq;           // dK/dV: launched behind the dQ kernel (else behind the statistics)
  float scale, scale_log2;
  unsigned long long wait_ns;
};

struct AttnStatArgs {
  AttnShape a;
  const int* lengths;
  const void *out, *rest, *dout;     // rest: of the forward, or null
  Strides out_strides, dout_strides;
  const float* lse;
  float* stat;
};

// The most CTAs that share an item's keys, for few items of long lists (split, without lse).
int fwd_parts(const AttnShape& a, bool bf16, int sms);
cudaError_t launch_attn_fwd(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                            const AttnFwdArgs& args, int sms, cudaStream_t stream);
cudaError_t launch_attn_stat(bool bf16, const AttnStatArgs& args, cudaStream_t stream);
cudaError_t launch_attn_dq(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                           const CUtensorMap& tm_do, const AttnBwdArgs& args, int sms, cudaStream_t stream);
cudaError_t launch_attn_dkv(bool bf16, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                            const CUtensorMap& tm_do, const AttnBwdArgs& args, int sms, cudaStream_t stream);

// Status words of the kernels of one source file on the current device (synchronises the stream, then clears them).
cudaError_t attn_fwd_status(cudaStream_t stream, int out[8]);
cudaError_t attn_bwd_status(cudaStream_t stream, int out[8]);
cudaError_t paged_append_status(cudaStream_t stream, int out[8]);
cudaError_t paged_attn_status(cudaStream_t stream, int out[8]);

// Sets a kernel's dynamic shared memory limit once per device (a kernel's attribute, not a call's).
struct SmemOnce {
  std::atomic<unsigned long long> done{0};
  cudaError_t set(const void* kernel, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

// A launch that may begin before the kernel in front of it has ended (the kernel itself waits for what it needs).
template <class... P, class... A>
inline cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, int bytes, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// For the source files' own status records.
inline cudaError_t take_status(const void* symbol, cudaStream_t stream, int out[8]) {
  Control c;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&c, symbol, sizeof(c), 0, cudaMemcpyDeviceToHost, stream);
  if (e != cudaSuccess) return e;
  if ((e = cudaStreamSynchronize(stream)) != cudaSuccess) return e;
  for (int i = 0; i < 7; ++i) out[i] = c.status[i];
  out[7] = 0;
  if (c.status[0] != 0) {
    static const Control zero = {};
    e = cudaMemcpyToSymbolAsync(symbol, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  }
  return e;
}

// Row `row` of a tile's two 64-column panels becomes zero (generic proxy; the caller fences).
__device__ __forceinline__ void zero_tile_row(uint8_t* tile, int row) {
  uint4* a = reinterpret_cast<uint4*>(tile + row * 128);
  uint4* b = reinterpret_cast<uint4*>(tile + kHalfBytes + row * 128);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    a[c] = make_uint4(0, 0, 0, 0);
    b[c] = make_uint4(0, 0, 0, 0);
  }
}
// valid positions of sequence b
__device__ __forceinline__ int attn_length(const AttnShape& a, const int* lengths, int b) {
  if (!lengths) return a.Nk;
  const int n = __ldg(lengths + b);
  return n < 0 ? 0 : (n < a.Nk ? n : a.Nk);
}

// ---- paged cache ----------------------------------------------------------------------------------------------
struct PagedCache {
  void *k, *v;                  // (pages, page, Hkv, 128)
  long long k_page, k_row, k_head, v_page, v_row, v_head;   // element strides
  const int* table;             // (B, table_width)
  long long table_stride;
  int table_width, pages;
  int page_shift;               // page = 1 << page_shift
};

struct AppendArgs {
  PagedCache c;
  const void *k, *v, *q;        // (T, Hkv, 128), (T, Hkv, 128) or null, (T, Hq, 128) or null
  long long k_tok, k_head, v_tok, v_head, q_tok, q_head;
  void* q_out;                  // (T, Hq, 128) contiguous, or null
  const int *cache_lens, *cu;   // (B), (B + 1) or null: one token per sequence
  const float* inv_freq;        // (rot / 2) or null: no rotation
  int B, T, Hq, Hkv, rot;       // rot: leading elements of a head that are rotated
  int interleaved;
};

struct PagedAttnArgs {
  PagedCache c;
  const void* q;                // (B, Hq, 128)
  long long q_b, q_h;
  const void* v_new;            // (B, Hkv, 128), LUCID only
  long long v_b, v_h;
  void* out;                    // (B, Hq, 128) contiguous
  const int* lens;              // (B)
  float* partial;               // split partial sums
  int B, Hq, Hkv, G, W, S, splits;
  float scale_log2, lucid_log2; // scale * log2(e); k_scale^2 * log2(e)
};

// up to this many chunks of a sequence are one cluster's CTAs (and then a power of two)
constexpr int kPagedCluster = 8, kPagedMaxSplits = 128, kPagedPerSm = 3;

cudaError_t launch_paged_append(bool bf16, const AppendArgs& args, int sms, cudaStream_t stream);
cudaError_t launch_paged_attn(bool bf16, bool lucid, const PagedAttnArgs& args, cudaStream_t stream);
size_t paged_attn_partial_bytes(int B, int Hq, int Hkv, bool lucid, int splits);

}  // namespace lucid
