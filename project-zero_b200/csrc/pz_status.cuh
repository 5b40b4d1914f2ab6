// pz_status.cuh — how the C entries outside pz_capi.cu report a failure
// (pz_last_error / pz_last_error_detail), and what they share on the host.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/pz_sampling.h"

namespace pz {

// Records the status (and the reason) for this thread and returns it.
pz_status report(pz_status s, const char *msg);
pz_status report_cuda(cudaError_t e);

// SMs of the current device, looked up once per device (148 where the
// lookup fails).
int current_sms();

// Lets a kernel use `bytes` of dynamic shared memory on the current device,
// once per device (`ready`: a bit per device, the kernel's own).
inline cudaError_t allow_smem(const void *kernel, int bytes, std::atomic<uint64_t> *ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && ((ready->load(std::memory_order_acquire) >> dev) & 1u)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) ready->fetch_or(1ull << dev, std::memory_order_release);
  return e;
}

// Bytes of B rows of V elements, `ld` elements apart.
inline uint64_t rows_bytes(int B, int V, int64_t ld, size_t es) {
  return (static_cast<uint64_t>(B - 1) * static_cast<uint64_t>(ld) + static_cast<uint64_t>(V)) * es;
}
// Whether two spans of memory share a byte.
inline bool overlap(const void *a, uint64_t na, const void *b, uint64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}
inline bool misaligned(const void *p, size_t es) { return reinterpret_cast<uintptr_t>(p) % es != 0; }
inline size_t elem_bytes(pz_dtype t) { return t == PZ_DTYPE_BF16 ? 2 : 4; }

}  // namespace pz
