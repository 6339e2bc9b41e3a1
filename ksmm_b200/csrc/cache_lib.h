// Between libksmm_cu.so (entry points, checks, plans) and libksmm_cache.so (kernels).
#pragma once

#include <cuda.h>

#include "cache.cuh"

namespace ksmm {
namespace cache {

constexpr int kCacheLibrary = 1;  // of these structures

// what the kernels' library uses of the other
struct Host {
  int version;
  int (*fail)(int status, const char* text);
  void (*count_launch)();
  int (*encode_map)(CUtensorMap*, int, int, const void*, const uint64_t*, const uint64_t*, const uint32_t*, bool, bool);
  int (*num_sms)();
  bool (*pdl_enabled)();
};

// launches: each returns a status
struct Kernels {
  int (*append)(Append&, int dtype, int cache_dtype, cudaStream_t);
  int (*token)(const Attend&, int dtype, int cache_dtype, unsigned grid, cudaStream_t);
  int (*prompt)(const Attend&, int dtype, bool eight, unsigned grid, cudaStream_t);
  int (*floats)(const Attend&, unsigned grid, cudaStream_t);
  int (*rows)(const Attend&, unsigned grid, cudaStream_t);
  int (*plain)(const Attend&, int dtype, int cache_dtype, unsigned grid, cudaStream_t);
  int (*join)(const Attend&, int dtype, unsigned blocks, int rows, cudaStream_t);
};

}  // namespace cache
}  // namespace ksmm
