// Appending to a paged cache.
//
// A warp takes a token (or, where there are few, some of its rows).  It finds the token's sequence, position and page,
// forms the cosines and sines of its rotation once for all heads and keeps them in registers, and moves its rows of q, k and v, four
// rounds in flight; the next token's chain starts -> length -> page is on its way meanwhile, and no warp waits for another (blocks
// of 8 warps that met at barriers for each token: 366 us for 32768 tokens of 32 + 16 rows of 128 in bf16; so: 135 us, 6.0 TB/s of
// the 6.4 that a copy reaches).  What it is bound by: memory; for a few tokens the chain of five waits, 4.5 us.  An angle is
// position * frequency, formed and reduced to a part of a turn in 64 bits (a position of 10^6 leaves 32 bits four digits of the
// angle).  That part, at most half a turn, is rounded to 32 bits for its sine and cosine: 2^-26 of a turn, 1e-7 radians, which
// shows beside the rounding of an fp32 result and of no 16-bit one (sines in 64 bits would take ten times the instructions).
#include <algorithm>

#include "cache.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

constexpr int kAppendThreads = 256;
// rounds of a warp in flight: one where elements go one by one
constexpr int flight(int vec) { return vec == 1 ? 1 : 4; }


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
  constexpr int kFlight = flight(VEC);
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
    piece<VEC>(lane + k * 32, a.pairs, VEC == 1 ? a.interleaved : INTER, &first[k], &second[k]);
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

bool whole(const void* p, int64_t x, int64_t y, int64_t z, int vec, int size) {
  return reinterpret_cast<uintptr_t>(p) % (vec * size) == 0 && x % vec == 0 && y % vec == 0 && z % vec == 0;
}

template <typename T, typename C, int VEC, bool INTER>
int launch_append_one(Append& a, cudaStream_t stream) {
  int sms = tc::num_sms();
  constexpr int kWarps = kAppendThreads / 32;
  const int64_t blocks = (sms > 0 ? sms : 148) * 2;
  const int rows = (a.in[0] ? a.heads : 0) + 2 * a.pool.kv_heads, rounds = (rows + 32 / a.lanes - 1) / (32 / a.lanes);
  // (where the tokens are fewer than the warps that run at a time, a token is several warps': each forms its rotation again)
  a.chunk_rows = (a.pool.tokens < blocks * kWarps ? 4 : rounds) * (32 / a.lanes);
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
  if (!vec) return launch_append_one<T, C, 1, false>(a, stream);  // (which asks at run time)
  return a.interleaved ? launch_append_one<T, C, VEC, true>(a, stream) : launch_append_one<T, C, VEC, false>(a, stream);
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

}  // namespace

int launch_append(Append& a, int dtype, int cache_dtype, cudaStream_t stream) {
  if (dtype == KSMM_F32) return launch_append_typed<float>(a, cache_dtype, stream);
  if (dtype == KSMM_F16) return launch_append_typed<__half>(a, cache_dtype, stream);
  return launch_append_typed<__nv_bfloat16>(a, cache_dtype, stream);
}

}  // namespace cache
}  // namespace ksmm
