// Host helpers shared by the C entry points: device query, tensor checks, tensor maps.
#pragma once
#include "../../include/lucid_b200.h"
#include "common.cuh"
#include "tmap.h"

namespace lucid {

// time limit of every device-side wait (lucid_set_wait_limit_ns)
unsigned long long wait_limit_ns();

// The driver's tensor-map call needs a current context, and a thread that has made no runtime call that needs one (an
// autograd worker, say) has none: make the current device's primary context current, once per thread and device.
inline cudaError_t ensure_context() {
  static thread_local int ready = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || ready == dev) return e;
  // (makes and binds the context since CUDA 12, and is allowed while a stream is being captured)
  if ((e = cudaSetDevice(dev)) != cudaSuccess) return e;
  ready = dev;
  return cudaSuccess;
}

inline int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 0 || dev >= 64) dev = 0;
  if (cached[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    cached[dev] = n;
  }
  return cached[dev];
}

// st = element strides {batch, sequence, head}; ext = the extents of those dimensions.  A zero stride in a
// dimension of extent > 1 is an expanded (broadcast) tensor: the tensor maps cannot express it, and writing
// through one would alias.
inline int check_tensor(const void* p, const int64_t st[3], int B, int N, int H) {
  if (!p || !st) return LUCID_E_NULL_POINTER;
  if (reinterpret_cast<uintptr_t>(p) % 16) return LUCID_E_BAD_ALIGNMENT;
  const int ext[3] = {B, N, H};
  for (int i = 0; i < 3; ++i) {
    if (st[i] % 8 || st[i] < 0) return LUCID_E_BAD_ALIGNMENT;
    if (st[i] == 0 && ext[i] > 1) return LUCID_E_BAD_STRIDE;
  }
  return 0;
}

// (B, N, H, 128) tensor -> 4-D map {d, n, h, b}
inline int bshd_map(CUtensorMap* m, bool bf16, const void* p, const int64_t st[3], int B, int N, int H,
                    uint32_t box_rows) {
  if (cudaError_t e = ensure_context()) return (int)e;
  uint64_t dims[4] = {(uint64_t)kBlock, (uint64_t)N, (uint64_t)H, (uint64_t)B};
  // size-1 dimensions may carry any stride; give them a harmless valid one.  (Zero strides of longer
  // dimensions never get here: check_tensor refuses them.)
  uint64_t sn = (uint64_t)st[1] * 2, sh = (uint64_t)st[2] * 2, sb = (uint64_t)st[0] * 2;
  if (N == 1) sn = 256;
  if (H == 1) sh = 256;
  if (B == 1) sb = 256;
  if (sn == 0 || sh == 0 || sb == 0) return LUCID_E_BAD_STRIDE;
  uint64_t strides[3] = {sn, sh, sb};
  return make_tmap_16bit(m, bf16, p, 4, dims, strides, box_rows) ? LUCID_E_TENSOR_MAP : 0;
}

}  // namespace lucid
