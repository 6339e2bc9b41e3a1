// Attention over a paged cache: the C entry points, their checks and plans.  The kernels are in a library of their own,
// libksmm_cache.so beside this one, which the first call loads: a process that uses no cache does not load their images (with
// CUDA_MODULE_LOADING=EAGER all of a library's are loaded at its first call, 3 MB of them).
#include <dlfcn.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdio>

#include "cache_lib.h"
#include "tc_host.h"

namespace ksmm {
namespace cache {
namespace {

int fail_with(int status, const char* text) { return set_error(status, "%s", text); }

// The kernels, or nullptr with the error set.
const Kernels* kernels() {
  static std::atomic<const Kernels*> loaded{nullptr};
  if (const Kernels* k = loaded.load(std::memory_order_acquire)) return k;
  Dl_info self = {};
  char path[4096];
  const char* name = "libksmm_cache.so";
  if (dladdr(reinterpret_cast<const void*>(&ksmm_cu_cache_append), &self) && self.dli_fname) {
    const char* slash = nullptr;
    for (const char* c = self.dli_fname; *c; ++c)
      if (*c == '/') slash = c;
    const int n = slash ? static_cast<int>(slash + 1 - self.dli_fname) : 0;
    if (n + 32 < static_cast<int>(sizeof(path))) {
      snprintf(path, sizeof(path), "%.*slibksmm_cache.so", n, self.dli_fname);
      name = path;
    }
  }
  void* lib = dlopen(name, RTLD_NOW | RTLD_LOCAL);  // (counted: two threads get the same)
  using Attach = const Kernels* (*)(const Host*);
  const Attach attach = lib ? reinterpret_cast<Attach>(dlsym(lib, "ksmm_cache_kernels")) : nullptr;
  static const Host host = {kCacheLibrary, &fail_with, &count_launch, &tc::encode_map, &tc::num_sms, &tc::pdl_enabled};
  const Kernels* k = attach ? attach(&host) : nullptr;
  if (!k) {
    set_error(KSMM_ERR_CUDA, "the kernels of the paged cache are missing, or another version's: %s", lib ? name : dlerror());
    return nullptr;
  }
  loaded.store(k, std::memory_order_release);
  return k;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool plain_type(int t) { return t == KSMM_F32 || t == KSMM_F16 || t == KSMM_BF16; }

int check_cache(const ksmm_cache_t& c, int heads, int dtype) {
  if (!plain_type(dtype)) return set_error(KSMM_ERR_UNSUPPORTED, "caches take float32, float16 and bfloat16 models");
  if (c.cache_dtype != dtype && c.cache_dtype != KSMM_F8E4M3)
    return set_error(KSMM_ERR_UNSUPPORTED, "a cache holds the model's type or float8_e4m3fn");
  if (c.sequences < 0 || c.tokens < 0 || c.sequences >= INT_MAX - 65536 || c.tokens >= INT_MAX - 65536)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "sequences and tokens are between 0 and 2^31 - 65537");
  if (c.page_size <= 0 || c.kv_heads <= 0 || c.head_dim <= 0 || heads <= 0 || c.pages < 0 || c.table_width < 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "page_size, heads, kv_heads and head_dim are positive");
  if (c.head_dim > kMaxDim) return set_error(KSMM_ERR_UNSUPPORTED, "head_dim is at most %d, not %d", kMaxDim, c.head_dim);
  if (c.pages >= (1ll << 31)) return set_error(KSMM_ERR_BAD_ARGUMENT, "a pool has less than 2^31 pages");
  if (static_cast<int64_t>(c.table_width) * c.page_size > INT_MAX - 65536)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "a sequence has at most 2^31 - 65537 tokens: table_width * page_size is more");
  if (heads % c.kv_heads || heads > 65535)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "%d heads do not share %d key heads evenly", heads, c.kv_heads);
  if (c.tokens == 0) return KSMM_OK;
  if (c.sequences == 0) return set_error(KSMM_ERR_BAD_ARGUMENT, "tokens without sequences");
  if (!c.starts && c.tokens % c.sequences)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "%lld tokens do not divide into %lld sequences", static_cast<long long>(c.tokens),
                     static_cast<long long>(c.sequences));
  if (!c.lengths || (!c.table && c.table_width)) return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  if (c.pages && (!c.keys || !c.values)) return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  if (c.pages && c.cache_dtype == KSMM_F8E4M3 && (!c.key_scales || !c.value_scales))
    return set_error(KSMM_ERR_BAD_ARGUMENT, "an 8-bit cache has scales for keys and values");
  if (c.sequences * static_cast<int64_t>(c.kv_heads) >= INT_MAX)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "sequences * kv_heads is less than 2^31");
  return KSMM_OK;
}

Pool pool_of(const ksmm_cache_t& c) {
  Pool p = {};
  p.data[0] = static_cast<char*>(c.keys);
  p.data[1] = static_cast<char*>(c.values);
  p.scales[0] = c.key_scales;
  p.scales[1] = c.value_scales;
  const int64_t* strides[2] = {c.key_strides, c.value_strides};
  const int64_t* scales[2] = {c.key_scale_strides, c.value_scale_strides};
  for (int i = 0; i < 2; ++i) {
    p.page[i] = strides[i][0];
    p.head[i] = strides[i][1];
    p.token[i] = strides[i][2];
    p.spage[i] = scales[i][0];
    p.shead[i] = scales[i][1];
    p.stoken[i] = scales[i][2];
  }
  p.table = c.table;
  p.lengths = c.lengths;
  p.starts = c.starts;
  p.pages = c.pages;
  p.table_stride = c.table_stride;
  p.page_size = c.page_size;
  p.table_width = c.table_width;
  p.kv_heads = c.kv_heads;
  p.dim = c.head_dim;
  p.sequences = static_cast<int>(c.sequences);
  p.tokens = static_cast<int>(c.tokens);
  p.each = c.starts || !c.sequences ? 1 : static_cast<int>(c.tokens / c.sequences);
  return p;
}

// Whether TMA can address the pool and the rows of q and out are pairs on their boundary.
bool token_fits(const ksmm_cache_attention_desc_t& d) {
  const ksmm_cache_t& c = d.cache;
  const bool eight = c.cache_dtype == KSMM_F8E4M3;
  const int per16 = eight ? 16 : 8;
  if (d.dtype == KSMM_F32 || c.head_dim % per16 || c.page_size % 16 || c.pages == 0) return false;
  for (int i = 0; i < 2; ++i) {
    if (reinterpret_cast<uintptr_t>(i ? c.values : c.keys) % 16) return false;
    const int64_t* s = i ? c.value_strides : c.key_strides;
    for (int k = 0; k < 3; ++k)
      if (s[k] <= 0 || s[k] % per16 || s[k] >= (1ll << 38)) return false;
    if (eight) {
      const int64_t* f = i ? c.value_scale_strides : c.key_scale_strides;
      if (reinterpret_cast<uintptr_t>(i ? c.value_scales : c.key_scales) % 16 || f[0] % 4 || f[1] % 4 || f[2] != 1) return false;
    }
  }
  return reinterpret_cast<uintptr_t>(d.q) % 4 == 0 && reinterpret_cast<uintptr_t>(d.out) % 4 == 0 && d.q_strides[0] % 2 == 0 &&
         d.q_strides[1] % 2 == 0 && d.out_strides[0] % 2 == 0 && d.out_strides[1] % 2 == 0;
}

bool prompt_fits(const ksmm_cache_attention_desc_t& d) {
  const int group = d.heads / d.cache.kv_heads;
  if (!token_fits(d) || group > 128) return false;
  // (a negative scale would turn the maximum round)
  if (!(d.scale > 0.f) || d.scale > 1e30f) return false;
  return reinterpret_cast<uintptr_t>(d.q) % 16 == 0 && reinterpret_cast<uintptr_t>(d.out) % 16 == 0 && d.q_strides[0] > 0 &&
         d.q_strides[1] > 0 && d.q_strides[0] % 8 == 0 && d.q_strides[1] % 8 == 0 && d.q_strides[0] < (1ll << 38) &&
         d.q_strides[1] < (1ll << 38) && d.out_strides[0] % 8 == 0 && d.out_strides[1] % 8 == 0;
}

// Vectors of four everywhere.
bool float_fits(const ksmm_cache_attention_desc_t& d) {
  const ksmm_cache_t& c = d.cache;
  if (d.dtype != KSMM_F32 || c.cache_dtype != KSMM_F32 || c.head_dim % 4 || c.pages == 0) return false;
  auto whole = [](const void* p, const int64_t* s, int n) {
    bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int i = 0; i < n; ++i) ok = ok && s[i] % 4 == 0;
    return ok;
  };
  return whole(c.keys, c.key_strides, 3) && whole(c.values, c.value_strides, 3) && whole(d.q, d.q_strides, 2) && whole(d.out, d.out_strides, 2);
}

// Sequences of up to this many rows (new tokens x heads of a group), or of two new tokens, are the kernels' for few rows, which share a
// batch's keys evenly over the GPU but go through them once for every 4 to 16 rows.  The prompt kernels take 64 or 128 rows as fast as
// one, but an item of theirs (a tile of rows of one sequence and key head) is not split.  They gain with rows x sequences x key
// heads above about 2500: with enough items for every SM from 20 rows on, with fewer items later (64 sequences, 32/8 heads of 128, few
// rows / prompt: bf16, 4000 tokens, 16 rows 194 / 190 us, 32 rows 348 / 191, 64 rows 643 / 191; fp32, 1000 tokens, 16 rows 502 / 584, 32 rows
// 990 / 585; 8 sequences of 4000, 32 rows, bf16 63 / 70, 8 bits 74 / 118, 64 rows 99 / 70 and 134 / 119; one sequence, 64 rows, bf16 30 / 64).
// Lengths are on the device: where tables are long, one sequence of many may be too, and its items alone would be waited for (1 us per
// 64 tokens, in fp32 9); such batches stay shared evenly up to 64 rows.  The rule sees the table's width only: 64 sequences of 4000 in
// tables of 64000 take 346 us for 32 rows and 643 for 64 in bf16, 369 and 717 in 8 bits.  And an item is never split: one sequence of
// 131077 tokens takes 335 us for 64 rows (16 new tokens) and 1653 for 68, 346 and 3408 in 8 bits.
int64_t few_rows(bool floats, int64_t pairs, int64_t longest) {
  const int64_t even = std::max<int64_t>(20, 2500 / pairs);
  const int64_t rows = longest <= (floats ? 1024 : 4096) ? even : std::max<int64_t>(even, 64);
  return floats ? rows : std::min<int64_t>(rows, 64);  // (more for 16 bits: not measured to gain)
}

struct Plan {
  unsigned prompt;        // blocks of the prompt kernel; 0: none
  int prompt_tile;
  enum { kToken, kRows, kPlain } kind;  // the other kernel
  unsigned grid;          // its blocks; 0: none
  int tile;
  int unit;
  bool split;
  int most;               // rows of its sequences
  int rows;               // of its items, at most
  size_t bytes, partial_bytes;
};

int64_t items(const ksmm_cache_t& c, int64_t group, int tile) { return (c.sequences + c.tokens * group / tile) * c.kv_heads; }

// Few rows (decoding) are split over their length in units: as many blocks as run at the same time share all units evenly,
// however the lengths differ.  Many get a block for each item.
bool plan_of(const ksmm_cache_attention_desc_t& d, Plan* p) {
  const ksmm_cache_t& c = d.cache;
  *p = {};
  const int64_t group = d.heads / c.kv_heads;
  const int64_t sure = c.starts ? c.tokens : c.tokens / c.sequences;
  int64_t rows = (d.max_new > 0 && d.max_new < sure ? d.max_new : sure) * group;
  p->most = INT_MAX;
  const bool floats = float_fits(d);
  const int64_t few = std::max<int64_t>(
      few_rows(floats, c.sequences * c.kv_heads, static_cast<int64_t>(c.table_width) * c.page_size), 2 * group);
  if (rows > few && (floats || prompt_fits(d))) {
    p->prompt_tile = floats ? kFloatRows : prompt_rows(static_cast<int>(group));
    const int64_t n = items(c, group, p->prompt_tile);
    if (n >= INT_MAX) return false;
    p->prompt = static_cast<unsigned>(n);
    if (!c.starts) return true;
    rows = p->most = static_cast<int>(few);
  }
  p->kind = token_fits(d) ? Plan::kToken : floats ? Plan::kRows : Plan::kPlain;
  const bool eight = c.cache_dtype == KSMM_F8E4M3;
  p->tile = p->kind == Plan::kToken ? token_rows(rows, eight, c.head_dim) : p->kind == Plan::kRows ? rows_tile(c.head_dim, rows) : kPlainRows;
  const TokenShape shape = p->kind == Plan::kToken  ? token_shape(eight, padded_dim(c.head_dim))
                           : p->kind == Plan::kRows ? TokenShape{row_blocks(c.head_dim, p->tile), kRowsUnit}
                                                    : TokenShape{2, kRowsUnit};
  p->unit = shape.unit;
  p->split = rows <= few;
  p->rows = static_cast<int>(std::min<int64_t>(sure * group, p->tile));  // (max_new is the caller's word)
  if (!p->split) {
    const int64_t n = items(c, group, p->tile);
    if (n >= INT_MAX) return false;
    p->grid = static_cast<unsigned>(n);
    return true;
  }
  int sms = tc::num_sms();
  if (sms <= 0) sms = 148;
  // (no more than there can be units)
  const double units = static_cast<double>(static_cast<int64_t>(c.table_width) * c.page_size / p->unit + 2) *
                       static_cast<double>((rows + p->tile - 1) / p->tile) * c.kv_heads * static_cast<double>(c.sequences);
  int limit = sms * shape.blocks;
  // (where no table is longer than an item that stays whole, and each has its block, nothing will have to be joined)
  if (static_cast<int64_t>(c.table_width) * c.page_size <= static_cast<int64_t>(kWholeUnits) * p->unit && items(c, group, p->tile) <= limit) {
    p->split = false;
    p->grid = static_cast<unsigned>(items(c, group, p->tile));
    return true;
  }
  limit = limit < kMaxBlocks ? limit : kMaxBlocks;
  p->grid = units < limit ? static_cast<unsigned>(units) : static_cast<unsigned>(limit);
  p->partial_bytes = (2 * sizeof(float) * p->grid * p->tile * (c.head_dim + 2) + 255) / 256 * 256;
  p->bytes = p->partial_bytes + 2 * sizeof(int64_t) * p->grid;
  return true;
}

int check_attention(const ksmm_cache_attention_desc_t* d) {
  if (!d) return set_error(KSMM_ERR_BAD_ARGUMENT, "null descriptor");
  const int st = check_cache(d->cache, d->heads, d->dtype);
  if (st != KSMM_OK) return st;
  if (d->cache.tokens * (d->heads / d->cache.kv_heads) > INT_MAX - 65536)
    return set_error(KSMM_ERR_UNSUPPORTED, "too many rows for one call: tokens * heads / kv_heads is at most 2^31 - 65537");
  if (d->window < 0 || d->max_new < 0) return set_error(KSMM_ERR_BAD_ARGUMENT, "window and max_new are not negative");
  return KSMM_OK;
}

}  // namespace
}  // namespace cache
}  // namespace ksmm

using namespace ksmm;
using namespace ksmm::cache;

extern "C" {

int ksmm_cu_cache_append(const ksmm_cache_append_desc_t* d, void* stream) {
  if (!d) return set_error(KSMM_ERR_BAD_ARGUMENT, "null descriptor");
  const ksmm_cache_t& c = d->cache;
  const int st = check_cache(c, d->heads, d->dtype);
  if (st != KSMM_OK) return st;
  if (d->pairs < 0 || 2 * static_cast<int64_t>(d->pairs) > c.head_dim)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "%d rotated pairs do not fit a head of %d", d->pairs, c.head_dim);
  if (c.tokens == 0) return KSMM_OK;
  if (!d->k || !d->v || (d->pairs && !d->frequencies) || (d->q && !d->q_out)) return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  Append a = {};
  a.pool = pool_of(c);
  const void* in[3] = {d->q, d->k, d->v};
  const int64_t* strides[3] = {d->q_strides, d->k_strides, d->v_strides};
  for (int i = 0; i < 3; ++i) {
    a.in[i] = static_cast<const char*>(in[i]);
    a.token[i] = strides[i][0];
    a.head[i] = strides[i][1];
  }
  a.q_out = d->q ? static_cast<char*>(d->q_out) : nullptr;
  a.out_token = d->q_out_strides[0];
  a.out_head = d->q_out_strides[1];
  a.frequencies = d->frequencies;
  a.pairs = d->pairs;
  a.interleaved = d->interleaved != 0;
  a.heads = d->heads;
  a.clear_rest = d->clear_rest != 0;
  const Kernels* k = kernels();
  return k ? k->append(a, d->dtype, c.cache_dtype, static_cast<cudaStream_t>(stream)) : KSMM_ERR_CUDA;
}

size_t ksmm_cu_cache_attention_workspace_bytes(const ksmm_cache_attention_desc_t* d) {
  if (check_attention(d) != KSMM_OK || d->cache.tokens == 0) return 0;
  Plan plan;
  return plan_of(*d, &plan) ? plan.bytes : 0;
}

int ksmm_cu_cache_attention(const ksmm_cache_attention_desc_t* d, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_attention(d);
  if (st != KSMM_OK || d->cache.tokens == 0) return st;
  if (!d->q || !d->out) return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  const ksmm_cache_t& c = d->cache;
  Plan plan;
  if (!plan_of(*d, &plan)) return set_error(KSMM_ERR_UNSUPPORTED, "too many rows for one call");
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || reinterpret_cast<uintptr_t>(workspace) % 256))
    return set_error(KSMM_ERR_WORKSPACE, "cache attention needs a workspace of %zu bytes, aligned to 256", plan.bytes);
  Attend a = {};
  a.pool = pool_of(c);
  a.q = static_cast<const char*>(d->q);
  a.out = static_cast<char*>(d->out);
  a.q_token = d->q_strides[0];
  a.q_head = d->q_strides[1];
  a.out_token = d->out_strides[0];
  a.out_head = d->out_strides[1];
  a.window = d->window;
  a.heads = d->heads;
  a.group = d->heads / c.kv_heads;
  a.scale = d->scale * 1.4426950408889634f;
  a.clear_rest = d->clear_rest != 0;
  a.partial = static_cast<float*>(workspace);
  a.slots = reinterpret_cast<int64_t*>(static_cast<char*>(workspace) + plan.partial_bytes);
  a.status = tc::status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Kernels* k = kernels();
  if (!k) return KSMM_ERR_CUDA;
  if (plan.prompt) {
    a.tile_rows = plan.prompt_tile;
    a.unit_log2 = 6;  // (its items are whole, and their number is the grid's; the fp32 kernel goes by units of 64 keys)
    a.least = plan.grid ? plan.most + 1 : 1;
    a.most = INT_MAX;
    a.split = 0;
    st = d->dtype == KSMM_F32 ? k->floats(a, plan.prompt, s) : k->prompt(a, d->dtype, c.cache_dtype == KSMM_F8E4M3, plan.prompt, s);
    if (st != KSMM_OK || !plan.grid) return st;
    a.clear_rest = 0;
  }
  a.tile_rows = plan.tile;
  a.unit_log2 = 31 - __builtin_clz(plan.unit);
  a.least = 1;
  a.most = plan.most;
  a.split = plan.split;
  switch (plan.kind) {
    case Plan::kToken: st = k->token(a, d->dtype, c.cache_dtype, plan.grid, s); break;
    case Plan::kRows: st = k->rows(a, plan.grid, s); break;
    default: st = k->plain(a, d->dtype, c.cache_dtype, plan.grid, s);
  }
  if (st == KSMM_OK && plan.split) st = k->join(a, d->dtype, plan.grid, plan.rows, s);
  return st;
}

}  // extern "C"
