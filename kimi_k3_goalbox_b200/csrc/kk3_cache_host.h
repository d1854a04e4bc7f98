// kk3_cache_host.h - host helpers shared by the translation units of the paged latent cache.
#pragma once

#include <cuda_runtime.h>
#include <stdio.h>

#include <atomic>

#include "kk3_cache.cuh"

namespace kk3 {

// KK3_OK, or KK3_ERR_CUDA with the reason on stderr (the sticky error is taken, so that it is reported once)
int cache_cuda(cudaError_t e, const char* what);
// a non-null pointer on an n-byte boundary
inline bool cache_aligned(const void* p, size_t n) { return p && (uintptr_t)p % n == 0; }
// queries that the kernels can read: 16-byte aligned rows
inline bool cache_queries(const void* ql, int64_t ql_token, int64_t ql_head, const void* qp, int64_t qp_token, int64_t qp_head) {
  return cache_aligned(ql, 16) && cache_aligned(qp, 16) && ((ql_token | ql_head | qp_token | qp_head) & 7) == 0 && ql_token >= 0 &&
         ql_head >= 0 && qp_token >= 0 && qp_head >= 0;
}
// a scale whose product with log2(e), on which the softmax runs, is finite in FP32 (3.40e38 / 1.4427)
inline bool cache_scale(float scale) { return scale >= -2.35e38f && scale <= 2.35e38f; }
// checks a kk3_cache and turns it into the kernels' form
int cache_pages(const kk3_cache* c, CachePages* out, int* error_word);
// attention (kk3_cache_tc.cu): tiles of kPairRows rows by CTA pairs, of kFewRows by single CTAs; a.workers of them
int attend_pair(const kk3_cache* c, const AttendArgs& a, cudaStream_t st);
int attend_few(const kk3_cache* c, const AttendArgs& a, cudaStream_t st);
// SMs of the current device, looked up once per device
int cache_sms(int* sms);

// Allow `kernel` its dynamic shared memory on the current device, once per device (`done`: a zeroed array of
// kCacheMaxDevices flags that belongs to the kernel; setting an attribute twice does no harm).
constexpr int kCacheMaxDevices = 64;
template <class K>
int cache_allow_smem(K kernel, size_t bytes, std::atomic<bool>* done, const char* what) {
  int dev = 0;
  int rc = cache_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  if (dev < kCacheMaxDevices && done[dev].load(std::memory_order_acquire)) return KK3_OK;
  rc = cache_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), what);
  if (rc == KK3_OK && dev < kCacheMaxDevices) done[dev].store(true, std::memory_order_release);
  return rc;
}

// Launch a kernel that follows another of the same call on the stream: its launch overlaps the end of the one
// before, and it begins with cache_follow().
template <class K, class... Args>
int cache_launch_after(K kernel, dim3 grid, int threads, cudaStream_t st, const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cache_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

}  // namespace kk3
