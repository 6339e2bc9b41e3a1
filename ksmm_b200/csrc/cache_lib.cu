// libksmm_cache.so: its one entry point, and what its kernels' launches use of libksmm_cu.so.
#include <cstdarg>
#include <cstdio>

#include "cache_lib.h"
#include "tc_host.h"

namespace ksmm {

static const cache::Host* g_host = nullptr;

int set_error(int status, const char* fmt, ...) {
  char text[512];
  va_list args;
  va_start(args, fmt);
  vsnprintf(text, sizeof(text), fmt, args);
  va_end(args);
  return g_host->fail(status, text);
}
void count_launch() { g_host->count_launch(); }

namespace tc {
int encode_map(CUtensorMap* tm, int dt, int rank, const void* base, const uint64_t* dims, const uint64_t* strides_elems, const uint32_t* box,
               bool swizzle128, bool atom32) {
  return g_host->encode_map(tm, dt, rank, base, dims, strides_elems, box, swizzle128, atom32);
}
int num_sms() { return g_host->num_sms(); }
bool pdl_enabled() { return g_host->pdl_enabled(); }
}  // namespace tc

}  // namespace ksmm

extern "C" __attribute__((visibility("default"))) const void* ksmm_cache_kernels(const void* host) {
  using namespace ksmm::cache;
  static const Kernels kernels = {&launch_append, &launch_token, &launch_prompt, &launch_float, &launch_rows, &launch_plain, &launch_join};
  const Host* h = static_cast<const Host*>(host);
  if (!h || h->version != kCacheLibrary) return nullptr;
  ksmm::g_host = h;  // (the same for every caller)
  return &kernels;
}
