// Attention over a paged cache: the append kernel and the C entry points.
//
// Append: a block per token (and per 4 rounds of its rows) finds the token's sequence, position and page, forms the cosines and
// sines of its rotation once for all heads, and moves its rows of q, k and v.  The rows are loaded before all of that: their
// way from memory overlaps the chain starts -> length -> page.  An angle is position * frequency, formed and reduced to a
// part of a turn in 64 bits (a position of 10^6 leaves 32 bits four digits of the angle).
#include <climits>

#include "cache.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kRounds = 4;

struct Append {
  Pool pool;
  const char* in[3];     // q, k, v
  char* q_out;
  int64_t token[3], head[3], out_token, out_head;
  const double* frequencies;
  int pairs, interleaved, heads, clear_rest;
  int lanes;             // threads of a row, a power of two up to 32
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// Element of a row where piece `u` of VEC pairs starts, first and second half.  Pieces are rotated pairs first, then the rest.
template <int VEC>
__device__ __forceinline__ void piece(int u, int pairs, int interleaved, int* first, int* second) {
  const int d = u * VEC;
  if (d >= pairs) {
    *first = 2 * d;
    *second = 2 * d + VEC;
  } else if (interleaved) {
    *first = 2 * d;
    *second = 2 * d + VEC;
  } else {
    *first = d;
    *second = d + pairs;
  }
}

// T: the model's type, C: the cache's; VEC elements at a time, with PIECES pieces of a row per thread (VEC 1: pairs is any number
// and a row up to 4 * 32 * 2 elements).
template <typename T, typename C, int VEC>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ Append a) {
  constexpr bool kEight = sizeof(C) == 1;
  constexpr int PIECES = VEC == 1 ? 4 : 1;
  __shared__ float2 turn[kMaxDim / 2];
  tc::grid_dep_wait();
  tc::grid_dep_launch();
  const Pool& p = a.pool;
  const int t = blockIdx.x, tid = threadIdx.x;
  const int lane = tid % a.lanes, per_round = kAppendThreads / a.lanes;
  const int q_rows = a.in[0] ? a.heads : 0, rows = q_rows + 2 * p.kv_heads;
  const int first_row = blockIdx.y * kRounds * per_round + tid / a.lanes;

  Vec<T, VEC> x[kRounds][PIECES], y[kRounds][PIECES];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int row = first_row + i * per_round;
    if (row >= rows) break;
    const int what = row < q_rows ? 0 : row < q_rows + p.kv_heads ? 1 : 2;
    const int head = what == 0 ? row : row - q_rows - (what - 1) * p.kv_heads;
    const T* from = reinterpret_cast<const T*>(a.in[what]) + t * a.token[what] + head * a.head[what];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      int d, e;
      piece<VEC>(lane + k * 32, a.pairs, a.interleaved, &d, &e);
      if (d < p.dim) x[i][k] = *reinterpret_cast<const Vec<T, VEC>*>(from + d);
      if (e < p.dim) y[i][k] = *reinterpret_cast<const Vec<T, VEC>*>(from + e);
    }
  }

  // the token's sequence: as many as start at or before it
  int s;
  int64_t start, n;
  if (p.starts) {
    int count = 0;
    for (int i = 0; i <= p.sequences; i += kAppendThreads)
      count += __syncthreads_count(i + tid <= p.sequences && p.starts[i + tid] <= t);
    s = count - 1;
    const bool there = s >= 0 && s < p.sequences;
    start = there ? p.starts[s] : 0;
    n = there ? static_cast<int64_t>(p.starts[s + 1]) - start : 0;
    if (!there) {
      // a row of no sequence
      if (!a.clear_rest || !a.q_out) return;
#pragma unroll
      for (int i = 0; i < kRounds; ++i) {
        const int row = first_row + i * per_round;
        if (row >= q_rows) return;
        T* to = reinterpret_cast<T*>(a.q_out) + t * a.out_token + row * a.out_head;
        for (int d = lane; d < p.dim; d += a.lanes) to[d] = ElemTraits<T>::from_float(0.f);
      }
      return;
    }
  } else {
    s = t / p.each;
    start = static_cast<int64_t>(s) * p.each;
    n = p.each;
  }
  const int64_t position = static_cast<int64_t>(p.lengths[s]) - n + (t - start);
  int64_t page = -1;
  int slot = 0;
  if (position >= 0 && position < static_cast<int64_t>(p.table_width) * p.page_size) {
    const int at = static_cast<int>(position / p.page_size);
    slot = static_cast<int>(position - static_cast<int64_t>(at) * p.page_size);
    page = p.table[s * p.table_stride + at];
    if (page >= p.pages) page = -1;
  }
  for (int i = tid; i < a.pairs; i += kAppendThreads) {
    const double turns = static_cast<double>(position) * a.frequencies[i] * 0.15915494309189533577;
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &cs);
    turn[i] = make_float2(cs, sn);
  }
  __syncthreads();

#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    // (whole rows leave together, and a warp's shuffles below name its lanes: no break before them)
    const int row = first_row + i * per_round;
    const bool live = row < rows;
    const int what = row < q_rows ? 0 : row < q_rows + p.kv_heads ? 1 : 2;
    const int head = what == 0 ? row : row - q_rows - (what - 1) * p.kv_heads;
    float u[PIECES][VEC], v[PIECES][VEC], top = 0.f;
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int unit = lane + k * 32;
      int d, e;
      piece<VEC>(unit, a.pairs, a.interleaved, &d, &e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u[k][j] = live && d < p.dim ? ElemTraits<T>::to_float(x[i][k].v[j]) : 0.f;
        v[k][j] = live && e < p.dim ? ElemTraits<T>::to_float(y[i][k].v[j]) : 0.f;
      }
      if (what < 2 && unit * VEC < a.pairs) {
        if (a.interleaved && VEC > 1) {
          // the pairs are neighbours: VEC / 2 in each vector
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            const float2 c = turn[unit * VEC + j], f = turn[unit * VEC + VEC / 2 + j];
            const float u0 = u[k][2 * j], u1 = u[k][2 * j + 1], v0 = v[k][2 * j], v1 = v[k][2 * j + 1];
            u[k][2 * j] = u0 * c.x - u1 * c.y;
            u[k][2 * j + 1] = u0 * c.y + u1 * c.x;
            v[k][2 * j] = v0 * f.x - v1 * f.y;
            v[k][2 * j + 1] = v0 * f.y + v1 * f.x;
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float2 c = turn[unit * VEC + j];
            const float u0 = u[k][j], v0 = v[k][j];
            u[k][j] = u0 * c.x - v0 * c.y;
            v[k][j] = u0 * c.y + v0 * c.x;
          }
        }
      }
      if (kEight) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) top = fmaxf(top, fmaxf(fabsf(u[k][j]), fabsf(v[k][j])));
      }
    }
    float scale = 1.f;
    if (kEight) {
      for (int w = a.lanes / 2; w; w /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      scale = fmaxf(top / 448.f, 1.1754943508e-38f);
    }
    if (!live || (what > 0 && page < 0)) continue;
    char* to;
    if (what == 0) {
      to = a.q_out + sizeof(T) * (t * a.out_token + head * a.out_head);
    } else {
      to = p.data[what - 1] + sizeof(C) * (page * p.page[what - 1] + head * p.head[what - 1] + slot * p.token[what - 1]);
      if (kEight && lane == 0)
        p.scales[what - 1][page * p.spage[what - 1] + head * p.shead[what - 1] + slot * p.stoken[what - 1]] = scale;
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      int d, e;
      piece<VEC>(lane + k * 32, a.pairs, a.interleaved, &d, &e);
      if (kEight && what > 0) {
        Vec<uint8_t, VEC> first, second;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          first.v[j] = __nv_cvt_float_to_fp8(u[k][j] / scale, __NV_SATFINITE, __NV_E4M3);
          second.v[j] = __nv_cvt_float_to_fp8(v[k][j] / scale, __NV_SATFINITE, __NV_E4M3);
        }
        if (d < p.dim) *reinterpret_cast<Vec<uint8_t, VEC>*>(to + d) = first;
        if (e < p.dim) *reinterpret_cast<Vec<uint8_t, VEC>*>(to + e) = second;
      } else {
        Vec<T, VEC> first, second;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          first.v[j] = ElemTraits<T>::from_float(u[k][j]);
          second.v[j] = ElemTraits<T>::from_float(v[k][j]);
        }
        if (d < p.dim) *reinterpret_cast<Vec<T, VEC>*>(to + d * sizeof(T)) = first;
        if (e < p.dim) *reinterpret_cast<Vec<T, VEC>*>(to + e * sizeof(T)) = second;
      }
    }
  }
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

bool whole(const void* p, int64_t x, int64_t y, int64_t z, int vec, int size) {
  return reinterpret_cast<uintptr_t>(p) % (vec * size) == 0 && x % vec == 0 && y % vec == 0 && z % vec == 0;
}

template <typename T, typename C, int VEC>
int launch_append(const Append& a, cudaStream_t stream) {
  const int rows = (a.in[0] ? a.heads : 0) + 2 * a.pool.kv_heads, per_block = kAppendThreads / a.lanes * kRounds;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.pool.tokens, (rows + per_block - 1) / per_block);
  cfg.blockDim = dim3(kAppendThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = tc::pdl_enabled() ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, append_kernel<T, C, VEC>, a);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "cache append kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

template <typename T>
int launch_append_typed(Append& a, int cache_dtype, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const Pool& p = a.pool;
  const bool eight = cache_dtype == KSMM_F8E4M3;
  const int cs = eight ? 1 : static_cast<int>(sizeof(T));
  bool vec = p.dim % VEC == 0 && a.pairs % VEC == 0;
  for (int i = 0; i < 3; ++i) vec = vec && (!a.in[i] || whole(a.in[i], a.token[i], a.head[i], 0, VEC, sizeof(T)));
  for (int i = 0; i < 2; ++i) vec = vec && whole(p.data[i], p.page[i], p.head[i], p.token[i], VEC, cs);
  vec = vec && (!a.q_out || whole(a.q_out, a.out_token, a.out_head, 0, VEC, sizeof(T)));
  const int per = vec ? VEC : 1, pieces = (p.dim + 2 * per - 1) / (2 * per);
  a.lanes = 1;
  while (a.lanes < pieces && a.lanes < 32) a.lanes *= 2;
  if (eight) return vec ? launch_append<T, f8e4m3, VEC>(a, stream) : launch_append<T, f8e4m3, 1>(a, stream);
  return vec ? launch_append<T, T, VEC>(a, stream) : launch_append<T, T, 1>(a, stream);
}

// Sequences of up to kFewRows rows (new tokens x heads of a group) are the token kernel's, in up to four tiles that read the keys
// one after the other; with more the prompt kernel's tiles of 128 rows are at least half full.
constexpr int kFewRows = 64;

struct Plan {
  unsigned prompt;        // blocks of the prompt kernel; 0: none
  int prompt_tile;
  bool token;             // the other kernel: the token kernel or the CUDA cores'
  unsigned grid;          // its blocks; 0: none
  int tile;
  bool split;
  int most;               // rows of its sequences
  size_t bytes, partial_bytes;
};

int64_t items(const ksmm_cache_t& c, int64_t group, int tile) { return (c.sequences + c.tokens * group / tile) * c.kv_heads; }

// Few rows (decoding) are split over their length in units: as many blocks as run at the same time share all units evenly,
// however the lengths differ.  Many get a block for each item.
bool plan_of(const ksmm_cache_attention_desc_t& d, Plan* p) {
  const ksmm_cache_t& c = d.cache;
  *p = {};
  const int64_t group = d.heads / c.kv_heads;
  int64_t most = c.starts ? c.tokens : c.tokens / c.sequences;
  if (d.max_new > 0 && d.max_new < most) most = d.max_new;
  int64_t rows = most * group;
  p->most = INT_MAX;
  if (rows > kFewRows && prompt_fits(d)) {
    p->prompt_tile = prompt_rows(c.head_dim, static_cast<int>(group));
    const int64_t n = items(c, group, p->prompt_tile);
    if (n >= INT_MAX) return false;
    p->prompt = static_cast<unsigned>(n);
    if (!c.starts) return true;
    rows = p->most = kFewRows;
  }
  p->token = token_fits(d);
  p->tile = p->token ? kTokenRows : rows_tile(c.head_dim);
  p->split = rows <= kFewRows;
  if (!p->split) {
    const int64_t n = items(c, group, p->tile);
    if (n >= INT_MAX) return false;
    p->grid = static_cast<unsigned>(n);
    return true;
  }
  int sms = tc::num_sms();
  if (sms <= 0) sms = 148;
  // (no more than there can be units)
  const double units = static_cast<double>(static_cast<int64_t>(c.table_width) * c.page_size / kUnit + 2) *
                       static_cast<double>((rows + p->tile - 1) / p->tile) * c.kv_heads * static_cast<double>(c.sequences);
  int limit = sms * (p->token ? token_blocks_per_sm(c.cache_dtype, c.head_dim) : 1);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->dtype == KSMM_F32) return launch_append_typed<float>(a, c.cache_dtype, s);
  if (d->dtype == KSMM_F16) return launch_append_typed<__half>(a, c.cache_dtype, s);
  return launch_append_typed<__nv_bfloat16>(a, c.cache_dtype, s);
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
  if (plan.prompt) {
    a.tile_rows = plan.prompt_tile;
    a.least = plan.grid ? plan.most + 1 : 1;
    a.most = INT_MAX;
    a.split = 0;
    st = launch_prompt(a, d->dtype, plan.prompt, s);
    if (st != KSMM_OK || !plan.grid) return st;
    a.clear_rest = 0;
  }
  a.tile_rows = plan.tile;
  a.least = 1;
  a.most = plan.most;
  a.split = plan.split;
  st = plan.token ? launch_token(a, d->dtype, c.cache_dtype, plan.grid, s) : launch_rows(a, d->dtype, c.cache_dtype, plan.grid, s);
  if (st == KSMM_OK && plan.split) st = launch_join(a, d->dtype, plan.grid, s);
  return st;
}

}  // extern "C"
