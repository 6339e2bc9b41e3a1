// Attention over a paged cache: the append kernel and the C entry points.
//
// Append: a warp takes a token (or, where there are few, some of its rows).  It finds the token's sequence, position and page,
// forms the cosines and sines of its rotation once for all heads and keeps them in registers, and moves its rows of q, k and v, four
// rounds in flight; the next token's chain starts -> length -> page is on its way meanwhile, and no warp waits for another (blocks
// of 8 warps that met at barriers for each token: 366 us for 32768 tokens of 32 + 16 rows of 128 in bf16).  An angle is
// position * frequency, formed and reduced to a part of a turn in 64 bits (a position of 10^6 leaves 32 bits four digits of the
// angle).
#include <algorithm>
#include <climits>

#include "cache.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kFlight = 4;  // rounds of a warp in flight

struct Append {
  Pool pool;
  const char* in[3];     // q, k, v
  char* q_out;
  int64_t token[3], head[3], out_token, out_head;
  const double* frequencies;
  int pairs, interleaved, heads, clear_rest;
  int lanes;             // threads of a row, a power of two up to 32
  int chunks;            // of a token: chunk_rows rows each
  int chunk_rows;
};

// VEC elements of type T as they lie in memory.  (Words and shifts: packing through arrays of 16-bit elements put them into local
// memory, 84 of every 100 instructions.)
template <typename T, int VEC>
struct Packed {
  static constexpr int kWords = VEC * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
  __device__ void load(const T* p) {
    if constexpr (kWords == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    } else {
      static_assert(kWords == 4, "16 bytes");
    }
  }
  __device__ void unpack(float (&f)[VEC]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (ElemTraits<T>::kDtype == KSMM_BF16) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const uint32_t bits = w[i];
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&bits));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
};
template <typename T>
struct Packed<T, 1> {
  T v;
  __device__ void load(const T* p) { v = *p; }
  __device__ void unpack(float (&f)[1]) const { f[0] = ElemTraits<T>::to_float(v); }
};

template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = ElemTraits<T>::from_float(f[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    constexpr int kDt = ElemTraits<T>::kDtype;
    *reinterpret_cast<uint4*>(p) = make_uint4(tc::pack2(f[0], f[1], kDt), tc::pack2(f[2], f[3], kDt), tc::pack2(f[4], f[5], kDt), tc::pack2(f[6], f[7], kDt));
  }
}
// as e4m3; the quotient by the scale, not the product with its reciprocal: that is what the scale stands for
__device__ __forceinline__ uint32_t e4m3_pair(float x, float y, float scale) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x / scale, y / scale), __NV_SATFINITE, __NV_E4M3);
}
template <int VEC>
__device__ __forceinline__ void store_eight(char* p, const float (&f)[VEC], float scale) {
  if constexpr (VEC == 1) {
    *reinterpret_cast<uint8_t*>(p) = __nv_cvt_float_to_fp8(f[0] / scale, __NV_SATFINITE, __NV_E4M3);
  } else {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) w[i] = e4m3_pair(f[4 * i], f[4 * i + 1], scale) | e4m3_pair(f[4 * i + 2], f[4 * i + 3], scale) << 16;
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

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

// What a block knows of a token before it moves its rows.
struct Place {
  int64_t position;
  int64_t page;  // -1: not stored
  int slot;
  int there;     // whether it is a sequence's
};

__device__ __forceinline__ Place place_of(const Pool& p, int t) {
  Place r = {0, -1, 0, 0};
  int s;
  if (p.starts) {
    // the last sequence that starts at or before it
    int low = 0, high = p.sequences + 1;  // the first `low` do, those from `high` on do not
    while (low < high) {
      const int mid = low + (high - low) / 2;
      if (p.starts[mid] <= t) low = mid + 1;
      else high = mid;
    }
    s = low - 1;
  } else {
    s = t / p.each;
  }
  if (s < 0 || s >= p.sequences) return r;
  r.there = 1;
  const int64_t start = p.starts ? p.starts[s] : static_cast<int64_t>(s) * p.each;
  const int64_t n = p.starts ? p.starts[s + 1] - start : p.each;
  r.position = static_cast<int64_t>(p.lengths[s]) - n + (t - start);
  if (r.position >= 0 && r.position < static_cast<int64_t>(p.table_width) * p.page_size) {
    const int at = static_cast<int>(r.position) / p.page_size;
    r.slot = static_cast<int>(r.position) - at * p.page_size;
    r.page = p.table[s * p.table_stride + at];
    if (r.page >= p.pages || r.page < 0) r.page = -1;
  }
  return r;
}

// Rows of one kind (heads of q, k or v) of a token, [from, to), per_round at a time.
template <typename T, int VEC, int PIECES, bool EIGHT, bool INTER>
__device__ __forceinline__ void move_rows(const T* src, int64_t src_head, char* dst, int64_t dst_head, float* scales, int64_t scale_head,
                                          int from, int to, int dim, int lanes, int lane, int nth, bool turns, bool eight,
                                          const int (&first)[PIECES], const int (&second)[PIECES], const bool (&turned)[PIECES],
                                          const float2 (&turn)[PIECES][VEC]) {
  const int per_round = 32 / lanes;
  src += (from + nth) * src_head;
  const int64_t dst_step = dst_head * (EIGHT && eight ? 1 : static_cast<int64_t>(sizeof(T)));
  dst += (from + nth) * dst_step;
#pragma unroll 1
  for (int row0 = from; row0 < to; row0 += kFlight * per_round) {
    Packed<T, VEC> x[kFlight][PIECES], y[kFlight][PIECES];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (row0 + i * per_round + nth < to) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          if (first[k] < dim) x[i][k].load(src + first[k]);
          if (second[k] < dim) y[i][k].load(src + second[k]);
        }
      }
      src += per_round * src_head;
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      // (the rows of a round stay together: their lanes meet in shuffles)
      const int row = row0 + i * per_round + nth;
      if (row - nth >= to) break;
      float u[PIECES][VEC], v[PIECES][VEC], top = 0.f;
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        x[i][k].unpack(u[k]);
        y[i][k].unpack(v[k]);
        if (turns && turned[k]) {
          if constexpr (INTER && VEC > 1) {
            // the pairs are neighbours: VEC / 2 in each vector
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) {
              const float2 c = turn[k][j], d = turn[k][VEC / 2 + j];
              const float u0 = u[k][2 * j], u1 = u[k][2 * j + 1], v0 = v[k][2 * j], v1 = v[k][2 * j + 1];
              u[k][2 * j] = u0 * c.x - u1 * c.y;
              u[k][2 * j + 1] = u0 * c.y + u1 * c.x;
              v[k][2 * j] = v0 * d.x - v1 * d.y;
              v[k][2 * j + 1] = v0 * d.y + v1 * d.x;
            }
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const float u0 = u[k][j], v0 = v[k][j];
              u[k][j] = u0 * turn[k][j].x - v0 * turn[k][j].y;
              v[k][j] = u0 * turn[k][j].y + v0 * turn[k][j].x;
            }
          }
        }
        if (EIGHT && eight) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (first[k] < dim) top = fmaxf(top, fabsf(u[k][j]));
            if (second[k] < dim) top = fmaxf(top, fabsf(v[k][j]));
          }
        }
      }
      if (EIGHT && eight) {
        for (int w = lanes / 2; w; w /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float scale = fmaxf(top / 448.f, 1.1754943508e-38f);
        if (row < to) {
          if (lane == 0) scales[row * scale_head] = scale;
#pragma unroll
          for (int k = 0; k < PIECES; ++k) {
            if (first[k] < dim) store_eight<VEC>(dst + first[k], u[k], scale);
            if (second[k] < dim) store_eight<VEC>(dst + second[k], v[k], scale);
          }
        }
      } else if (row < to) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          if (first[k] < dim) store<T, VEC>(reinterpret_cast<T*>(dst) + first[k], u[k]);
          if (second[k] < dim) store<T, VEC>(reinterpret_cast<T*>(dst) + second[k], v[k]);
        }
      }
      dst += per_round * dst_step;
    }
  }
}

// T: the model's type, C: the cache's; VEC elements at a time, with PIECES pieces of a row per lane (VEC 1: pairs is any number
// and a row up to 4 * 32 * 2 elements).
template <typename T, typename C, int VEC, bool INTER>
__global__ void __launch_bounds__(kAppendThreads, 2) append_kernel(const __grid_constant__ Append a) {
  constexpr bool kEight = sizeof(C) == 1;
  constexpr int PIECES = VEC == 1 ? 4 : 1;
  constexpr int kWarps = kAppendThreads / 32;
  __shared__ __align__(16) float2 turns[VEC == 1 ? 1 : kWarps][kMaxDim / 2];
  touch_parameters(a);
  tc::grid_dep_wait();
  tc::grid_dep_launch();
  const Pool& p = a.pool;
  const int warp = threadIdx.x / 32, wl = threadIdx.x % 32;
  const int lane = wl % a.lanes, nth = wl / a.lanes;
  const int q_rows = a.in[0] ? a.heads : 0, rows = q_rows + 2 * p.kv_heads;
  const int64_t items = static_cast<int64_t>(p.tokens) * a.chunks, warps = static_cast<int64_t>(gridDim.x) * kWarps;
  int first[PIECES], second[PIECES];
  bool turned[PIECES];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    piece<VEC>(lane + k * 32, a.pairs, INTER, &first[k], &second[k]);
    turned[k] = (lane + k * 32) * VEC < a.pairs;
  }

  int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (item >= items) return;
  int t = static_cast<int>(item / a.chunks);
  Place next = place_of(p, t);
#pragma unroll 1
  for (; item < items; item += warps) {
    const Place place = next;
    const int this_t = t, row0 = static_cast<int>(item - static_cast<int64_t>(t) * a.chunks) * a.chunk_rows;
    const int end = min(rows, row0 + a.chunk_rows);
    if (item + warps < items) {
      t = static_cast<int>((item + warps) / a.chunks);
      next = place_of(p, t);
    }

    // cosines and sines of the lane's pairs
    float2 turn[PIECES][VEC];
    auto angle = [&](int pair) {
      const double part = static_cast<double>(place.position) * a.frequencies[pair] * 0.15915494309189533577;
      float sn, cs;
      sincospif(2.f * static_cast<float>(part - rint(part)), &sn, &cs);
      return make_float2(cs, sn);
    };
    if constexpr (VEC == 1) {
#pragma unroll
      for (int k = 0; k < PIECES; ++k) turn[k][0] = turned[k] ? angle(lane + k * 32) : make_float2(1.f, 0.f);
    } else {
      // (each lane forms some; a lane's VEC pairs then are VEC / 2 vectors, and lanes side by side read vectors side by side)
      __syncwarp();
      for (int i = wl; i < a.pairs; i += 32) turns[warp][((i % VEC / 2) * a.lanes + i / VEC) * 2 + i % 2] = angle(i);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float4 c = turned[0] ? reinterpret_cast<const float4*>(turns[warp])[j / 2 * a.lanes + lane] : make_float4(1.f, 0.f, 1.f, 0.f);
        turn[0][j] = make_float2(c.x, c.y);
        turn[0][j + 1] = make_float2(c.z, c.w);
      }
    }

    if (row0 < q_rows && !place.there && a.clear_rest) {
      // rows of no sequence
      T* to = reinterpret_cast<T*>(a.q_out) + this_t * a.out_token;
      for (int i = row0 * p.dim + wl; i < min(end, q_rows) * p.dim; i += 32) to[i / p.dim * a.out_head + i % p.dim] = ElemTraits<T>::from_float(0.f);
    }
    // (one copy of the code for the three kinds: with three the registers go to addresses)
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {
      const int kv = kind == 2, begin = kind == 0 ? 0 : q_rows + kv * p.kv_heads;
      const int from = max(row0 - begin, 0), to = min(end - begin, kind == 0 ? q_rows : p.kv_heads);
      if (from >= to || (kind == 0 ? !place.there : place.page < 0)) continue;
      char* dst;
      int64_t dst_head;
      float* scales = nullptr;
      if (kind == 0) {
        dst = a.q_out + this_t * a.out_token * static_cast<int64_t>(sizeof(T));
        dst_head = a.out_head;
      } else {
        dst = p.data[kv] + (place.page * p.page[kv] + place.slot * p.token[kv]) * static_cast<int64_t>(sizeof(C));
        dst_head = p.head[kv];
        if (kEight) scales = p.scales[kv] + place.page * p.spage[kv] + place.slot * p.stoken[kv];
      }
      move_rows<T, VEC, PIECES, kEight, INTER>(reinterpret_cast<const T*>(a.in[kind]) + this_t * a.token[kind], a.head[kind], dst, dst_head,
                                               scales, p.shead[kv], from, to, p.dim, a.lanes, lane, nth, kind < 2, kind > 0, first, second,
                                               turned, turn);
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

template <typename T, typename C, int VEC, bool INTER>
int launch_append(Append& a, cudaStream_t stream) {
  int sms = tc::num_sms();
  constexpr int kWarps = kAppendThreads / 32;
  const int64_t blocks = (sms > 0 ? sms : 148) * 2;
  const int rows = (a.in[0] ? a.heads : 0) + 2 * a.pool.kv_heads, rounds = (rows + 32 / a.lanes - 1) / (32 / a.lanes);
  // (where the tokens are fewer than the warps that run at a time, a token is several warps': each forms its rotation again)
  a.chunk_rows = (a.pool.tokens < blocks * kWarps ? kFlight : rounds) * (32 / a.lanes);
  a.chunks = (rows + a.chunk_rows - 1) / a.chunk_rows;
  const int64_t needed = (static_cast<int64_t>(a.pool.tokens) * a.chunks + kWarps - 1) / kWarps;
  const cudaError_t err =
      tc::launch_pdl(append_kernel<T, C, VEC, INTER>, static_cast<unsigned>(std::min(needed, blocks)), kAppendThreads, 0, stream, a);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "cache append kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

template <typename T, typename C>
int launch_append_order(Append& a, bool vec, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  if (a.interleaved) return vec ? launch_append<T, C, VEC, true>(a, stream) : launch_append<T, C, 1, true>(a, stream);
  return vec ? launch_append<T, C, VEC, false>(a, stream) : launch_append<T, C, 1, false>(a, stream);
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
  if (eight) return launch_append_order<T, f8e4m3>(a, vec, stream);
  return launch_append_order<T, T>(a, vec, stream);
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
  int unit;
  bool split, narrow;
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
  if (rows > kFewRows && (floats || prompt_fits(d))) {
    p->prompt_tile = floats ? kFloatRows : prompt_rows(static_cast<int>(group));
    const int64_t n = items(c, group, p->prompt_tile);
    if (n >= INT_MAX) return false;
    p->prompt = static_cast<unsigned>(n);
    if (!c.starts) return true;
    rows = p->most = kFewRows;
  }
  p->token = token_fits(d);
  p->tile = p->token ? token_rows(rows) : rows_tile(c.head_dim, rows);
  const TokenShape shape = p->token ? token_shape(c.cache_dtype, c.head_dim) : TokenShape{row_blocks(c.head_dim, p->tile), kRowsUnit};
  p->unit = shape.unit;
  p->split = rows <= kFewRows;
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
  // (rows are max_new's word; all tiles that there can be)
  p->narrow = units / static_cast<double>((rows + p->tile - 1) / p->tile) * static_cast<double>(sure * group / p->tile + 1) < 2e9;
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
    a.unit_log2 = 6;  // (its items are whole, and their number is the grid's; the fp32 kernel goes by units of 64 keys)
    a.narrow = 1;
    a.least = plan.grid ? plan.most + 1 : 1;
    a.most = INT_MAX;
    a.split = 0;
    st = d->dtype == KSMM_F32 ? launch_float(a, plan.prompt, s) : launch_prompt(a, d->dtype, plan.prompt, s);
    if (st != KSMM_OK || !plan.grid) return st;
    a.clear_rest = 0;
  }
  a.tile_rows = plan.tile;
  a.unit_log2 = 31 - __builtin_clz(plan.unit);
  a.narrow = plan.narrow || !plan.split;
  a.least = 1;
  a.most = plan.most;
  a.split = plan.split;
  st = plan.token ? launch_token(a, d->dtype, c.cache_dtype, plan.grid, s) : launch_rows(a, d->dtype, c.cache_dtype, plan.grid, s);
  if (st == KSMM_OK && plan.split) st = launch_join(a, d->dtype, plan.grid, plan.rows, s);
  return st;
}

}  // extern "C"
