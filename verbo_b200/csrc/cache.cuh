// Launch-side view of the paged cache (include/verbo_cache.h), shared by
// cache_pages.cu, cache_attend.cu and cache_capi.cpp.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "verbo_cache.h"

namespace vb {

constexpr int kCacheBlock = VERBO_CACHE_BLOCK;

// cache_pages.cu
size_t cache_workspace_bytes(const verbo_cache& c);
cudaError_t launch_cache_reserve(const verbo_cache& c, const int* add, int* start, int* status, void* ws,
                                 cudaStream_t s);
cudaError_t launch_cache_fork(const verbo_cache& c, const int* parents, long long ld_parents, int beams,
                              cudaStream_t s);
cudaError_t launch_cache_free(const verbo_cache& c, const int* keep, cudaStream_t s);
cudaError_t launch_cache_compact(const verbo_cache& c, int* info, void* ws, cudaStream_t s);

struct CacheNew {  // the tokens of an append: token i, head h at x + i * ld + h * hd
  const void* k;
  const void* v;
  long long ld_k, hd_k, ld_v, hd_v;
  int tokens;
  const int* start;
  const long long* off;  // or null
};
cudaError_t launch_cache_append(const verbo_cache& c, int layer, const CacheNew& x, int dtype, cudaStream_t s);

// cache_attend.cu
struct CacheQuery {
  const void* q;
  long long ld_q, hd_q;
  void* out;
  long long ld_out, hd_out;
  int heads, steps;
  float scale;
  void* workspace;
};
size_t cache_attend_bytes(const verbo_cache& c, int heads, int steps, int q_type);
cudaError_t launch_cache_attend(const verbo_cache& c, int layer, const CacheQuery& x, int q_type, int out_type,
                                cudaStream_t s);

}  // namespace vb
