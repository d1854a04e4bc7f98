// kk3_cache_host.h - host helpers shared by the translation units of the paged latent cache.
#pragma once

#include <cuda_runtime.h>
#include <stdio.h>

#include "kk3_cache.cuh"

namespace kk3 {

// KK3_OK, or KK3_ERR_CUDA with the reason on stderr (the sticky error is taken, so that it is reported once)
int cache_cuda(cudaError_t e, const char* what);
// a non-null pointer on an n-byte boundary
inline bool cache_aligned(const void* p, size_t n) { return p && (uintptr_t)p % n == 0; }
// checks a kk3_cache and turns it into the kernels' form
int cache_pages(const kk3_cache* c, CachePages* out, int* error_word);
// SMs of the current device
int cache_sms(int* sms);

}  // namespace kk3
