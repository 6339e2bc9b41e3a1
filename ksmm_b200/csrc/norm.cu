// The passage from one block of a network to the next (ksmm_cu_norm_forward, ksmm_cu_norm_backward):
//
//   p = post(y) * post_weight + post_bias            post: none (p = y), layer norm, rms norm
//   z = alpha * x + gate * p                         (z = x without y)
//   h = (pre(z) * weight + bias) * (1 + scale) + shift      pre: none (no h), layer norm, rms norm
//
// over the channels of every token.  gate, scale and shift are one row for all tokens or one row per sample
// (a run of rows / samples consecutive tokens).  Backward, with G the whole gradient of z, n = pre's
// normalised value, m = post's (or y itself):
//
//   e = grad_h * weight * (1 + scale)
//   G = grad_z + r (e - n mean(e n) - mean(e))       (mean(e): layer norm only; r: the reciprocal deviation)
//   grad_x = alpha G,   f = G * gate * post_weight,   grad_y = r' (f - m mean(f m) - mean(f))
//
// and per sample and channel the sums A = sum grad_h, B = sum grad_h n, C = sum G, D = sum G m, from which
// every parameter's gradient follows without another look at the tensors:
//   shift: A, scale: weight B + bias A, weight: sum (1 + scale) B, bias: sum (1 + scale) A,
//   gate: post_weight D + post_bias C, post_weight: sum gate D, post_bias: sum gate C.
//
// All of it is bound by memory: each tensor is read once and written once.  Statistics, sums and the value
// h is made from stay in fp32; z and h are rounded once.  The backward pass of 16-bit tensors forms the unrounded
// z again from x and y, which takes no more bytes than reading the rounded one (that it reads if it is given z): 20
// deviations from 0 the rounding of z costs 2 % of a gradient in bf16.  It reads the statistics (16 bytes per token).
// Sums over tokens are formed in a fixed order: a CTA sums its own run of tokens, two small kernels add the runs up;
// no atomics.
//
// The stock form in the reference's models is a chain of separate PyTorch calls: LayerNorm and the sum around
// attention and feed-forward block (src/ksmm_py/model/vit.py:416-431, 770-800).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "backward.h"
#include "common.cuh"
#include "norm.h"
#include "tc_epilogue.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace {

enum { kNone = KSMM_NORM_NONE, kLayer = KSMM_NORM_LAYER, kRms = KSMM_NORM_RMS };
constexpr int kMaxChannels = 8192;

// a parameter: one row of the channels (ld = 0) or one per sample
struct Row {
  const void* p;
  int64_t ld;
};

struct Args {
  const void *x, *y, *z_in, *gz, *gh;
  void *z, *h, *gx, *gy;
  float4* stats;  // per token: mean and reciprocal deviation of pre, of post
  Row weight, bias, post_weight, post_bias, scale, shift, gate;
  float* part;    // backward: [chunk][4][channels]
  int64_t rows, per_sample;  // tokens, tokens of a sample
  int64_t samples;
  int chunks;     // chunks of tokens of one sample
  int C, pre, post, p32;  // p32: parameters are fp32
  int remake;     // backward, 16 bits: z_in is x, and z is formed from it and y
  float alpha, eps;
  int stages;     // rows in flight per group of threads
  int* status;    // where a wait that ran out leaves its code
};

// Arithmetic runs on pairs (the two-wide fp32 instructions: same roundings, half the issue slots), or on single
// values where rows start anywhere (V = 1).
__device__ __forceinline__ uint64_t e_fma(uint64_t a, uint64_t b, uint64_t c) { return tc::fma_f2(a, b, c); }
__device__ __forceinline__ uint64_t e_mul(uint64_t a, uint64_t b) { return tc::mul_f2(a, b); }
__device__ __forceinline__ uint64_t e_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float e_fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float e_mul(float a, float b) { return a * b; }
__device__ __forceinline__ float e_add(float a, float b) { return a + b; }
__device__ __forceinline__ float e_sum(uint64_t a) {
  float x, y;
  tc::unpack_f2(a, x, y);
  return x + y;
}
__device__ __forceinline__ float e_sum(float a) { return a; }

template <int V>
struct Elem {
  using E = uint64_t;
  static constexpr int N = V / 2;
  static __device__ __forceinline__ E all(float x) { return tc::pack_f2(x, x); }
};
template <>
struct Elem<1> {
  using E = float;
  static constexpr int N = 1;
  static __device__ __forceinline__ E all(float x) { return x; }
};

// V consecutive elements (16 bytes, or one element)
template <typename T, int V>
struct Raw {
  static_assert(V * sizeof(T) == 16, "a 16-byte piece");
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ uint64_t get(int i) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4) {
      return tc::pack_f2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (ElemTraits<T>::kDtype == KSMM_BF16) {
      return tc::pack_f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      return tc::pack_f2(f.x, f.y);
    }
  }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = ElemTraits<T>::from_float(0.f); }
  __device__ __forceinline__ float get(int) const { return ElemTraits<T>::to_float(v); }
};

template <typename T, int V>
__device__ __forceinline__ void store_piece(T* p, const typename Elem<V>::E (&f)[Elem<V>::N]) {
  if constexpr (V == 1) {
    *p = ElemTraits<T>::from_float(f[0]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float x, y;
      tc::unpack_f2(f[i], x, y);
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(x);
        w[2 * i + 1] = __float_as_uint(y);
      } else if constexpr (ElemTraits<T>::kDtype == KSMM_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(x, y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// V parameters from channel c of a sample's row; `other` where there is no such parameter.  (Pieces need aligned
// parameters; the host takes V = 1 otherwise.)
template <typename T, int V>
__device__ __forceinline__ void load_param(const Args& A, const Row& r, int64_t sample, int c, float other,
                                           typename Elem<V>::E (&f)[Elem<V>::N]) {
  if (r.p == nullptr) {
#pragma unroll
    for (int i = 0; i < Elem<V>::N; ++i) f[i] = Elem<V>::all(other);
    return;
  }
  const int64_t at = sample * r.ld + c;
  if (A.p32) {
    const float* p = static_cast<const float*>(r.p) + at;
    if constexpr (V == 1) {
      f[0] = __ldg(p);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; i += 2) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + 2 * i));
        f[i] = tc::pack_f2(q.x, q.y);
        f[i + 1] = tc::pack_f2(q.z, q.w);
      }
    }
  } else {
    Raw<T, V> q;
    q.load(static_cast<const T*>(r.p) + at);
#pragma unroll
    for (int i = 0; i < Elem<V>::N; ++i) f[i] = q.get(i);
  }
}

// one parameter as it lies in memory, and its value: loads first, conversions later, so that a thread's loads overlap
__device__ __forceinline__ uint32_t raw_param(const Args& A, const Row& r, int64_t sample, int c) {
  if (r.p == nullptr) return 0;
  const int64_t at = sample * r.ld + c;
  return A.p32 ? __ldg(static_cast<const uint32_t*>(r.p) + at) : __ldg(static_cast<const uint16_t*>(r.p) + at);
}
template <typename T>
__device__ __forceinline__ float param_value(const Args& A, const Row& r, uint32_t raw, float other) {
  if (r.p == nullptr) return other;
  if (A.p32) return __uint_as_float(raw);
  if constexpr (sizeof(T) == 4) return __uint_as_float(raw);
  else if constexpr (ElemTraits<T>::kDtype == KSMM_BF16) return __uint_as_float(raw << 16);
  else return __half2float(__ushort_as_half(static_cast<uint16_t>(raw)));
}

// V parameters from channel c as they lie in memory, and their values
template <typename T, int V>
__device__ __forceinline__ void raw_piece(const Args& A, const Row& r, int64_t sample, int c, uint4 (&q)[2]) {
  q[0] = q[1] = make_uint4(0, 0, 0, 0);
  if (r.p == nullptr) return;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(r.p) + (sample * r.ld + c) * (A.p32 ? 4 : static_cast<int>(sizeof(T))));
  q[0] = __ldg(p);
  if (V == 8 && A.p32) q[1] = __ldg(p + 1);
}
template <typename T, int V>
__device__ __forceinline__ float piece_value(const Args& A, const Row& r, const uint4 (&q)[2], int e, float other) {
  if (r.p == nullptr) return other;
  const uint32_t w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
  if (sizeof(T) == 4 || A.p32) return __uint_as_float(w[e]);
  const uint16_t h = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
  if constexpr (ElemTraits<T>::kDtype == KSMM_BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(__ushort_as_half(h));
}

// the parameters of channel c as z and h use them: gate * post_weight, gate * post_bias, weight (1 + scale),
// bias (1 + scale) + shift
template <typename T>
__device__ __forceinline__ float4 combined(const Args& A, int64_t sample, int c) {
  const uint32_t g = raw_param(A, A.gate, sample, c), pw = raw_param(A, A.post_weight, 0, c), pb = raw_param(A, A.post_bias, 0, c);
  const uint32_t w = raw_param(A, A.weight, 0, c), b = raw_param(A, A.bias, 0, c);
  const uint32_t sc = raw_param(A, A.scale, sample, c), sh = raw_param(A, A.shift, sample, c);
  const float gate = param_value<T>(A, A.gate, g, 1.f), by = 1.f + param_value<T>(A, A.scale, sc, 0.f);
  return make_float4(gate * param_value<T>(A, A.post_weight, pw, 1.f), gate * param_value<T>(A, A.post_bias, pb, 0.f),
                     by * param_value<T>(A, A.weight, w, 1.f),
                     fmaf(by, param_value<T>(A, A.bias, b, 0.f), param_value<T>(A, A.shift, sh, 0.f)));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The sums of N = 1, 2 or 4 values over the block, in a fixed order.  Within a warp the lanes share the values out
// (6 exchanges for four sums instead of 20), then every thread adds the warps' sums up.  `red` holds
// 2 * 32 * N floats; calls alternate between its halves (`turn`), so that one barrier per call is enough.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* red, int& turn) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = N; n > 1; n >>= 1, o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float keep = up ? v[i + n / 2] : v[i], send = up ? v[i] : v[i + n / 2];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  // lane bits 4, 3, ... pick the upper half of the values left: value i sits in lanes with those bits
  float* buf = red + (turn & 1) * 32 * N;
  ++turn;
  const int idx = N == 1 ? 0 : (N == 2 ? lane >> 4 : ((lane >> 4) & 1) * 2 + ((lane >> 3) & 1));
  if ((lane & (32 / N - 1)) == 0) buf[warp * N + idx] = v[0];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < N; ++q) v[q] = 0.f;
  for (int w = 0; w < warps; ++w) {
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] += buf[w * N + q];
  }
}

// ---------------------------------------------------------------------------
// batch-first: a token is a row
// ---------------------------------------------------------------------------
// A row of `bytes` from memory to shared memory; the barrier expects them
__device__ __forceinline__ void bulk_row(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}

// TPR threads hold a row in registers, K pieces each: a warp per row up to 1024 channels (no barrier), a group of
// threads beyond.
// RING: blocks that stay on their SM take equal runs of rows.  Rows come to shared memory by bulk copies, `stages` of
// them in flight per group of threads, and the parameters of the run's sample are combined there once, for every
// row of it; a run may pass on to the next sample.  Else every row reads its parameters (by groups of eight threads up to
// 128 channels of 16 bits, where most of a warp would lie idle: 62 x 4446 x 64 fp16 138 -> 85 us).  128 x 196 x 768 bf16 with
// gate, weight, bias, scale and shift (154 MB, 24 us at the copy's rate): 53 us with parameters read per row, 28 so;
// 32768 x 4096 bf16 (1.07 GB, 166 us): 217 with a block of 256 threads per row, 175 with four groups of 128 and two
// rows in flight for each.  (A block of 512 threads per row took 226: a row's waits and sums are paid per thread.)
constexpr int kRingBlock = 256, kRingWide = 512;

// the sum over a group of TPR threads
template <int TPR>
__device__ __forceinline__ float group_sum(float v, float* red, int& turn, int group) {
  if constexpr (TPR < 32) {  // a group's lanes only: other groups of the warp may have no row
    const unsigned mask = ((1u << (TPR & 31)) - 1u) << (threadIdx.x & 31 & ~(TPR - 1));
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
  }
  v = warp_sum(v);
  if constexpr (TPR <= 32) {
    return v;
  } else {
    constexpr int W = TPR / 32;
    float* buf = red + (group * 2 + (turn & 1)) * W;
    ++turn;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x % TPR / 32] = v;
    tc::bar_sync_named(1 + group, TPR);
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += buf[w];
    return v;
  }
}

template <typename T, int V, int K, int TPR, bool RING>
__global__ void __launch_bounds__(RING ? (TPR == 32 ? kRingBlock : kRingWide) : (TPR < 128 ? 128 : TPR),
                                  RING ? (TPR == 32 ? 2 : 1) : (TPR > 256 ? 1 : (TPR == 256 ? (K <= 2 ? 3 : 2) : 4)))
    norm_rows_kernel(const Args A) {
  using L = Elem<V>;
  using E = typename L::E;
  constexpr int kBlock = RING ? (TPR == 32 ? kRingBlock : kRingWide) : (TPR < 128 ? 128 : TPR);
  constexpr int kGroups = kBlock / TPR;
  constexpr int kMaxStages = 12;
  __shared__ float red[2 * kBlock / 32];
  __shared__ __align__(8) uint64_t bars[RING ? kGroups * kMaxStages : 1];
  __shared__ int abort_flag;
  extern __shared__ __align__(16) float4 coef[];  // RING: [4 kinds][V / 4 quarters of a piece][pieces], then the rows
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  int turn = 0;
  auto sum = [&](float v) { return group_sum<TPR>(v, red, turn, group); };
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group, end = row + 1;
  if (row >= A.rows) end = row;  // (whole warps, or the whole block)
  int64_t sample = 0;
  const int pieces = A.C / V;
  Raw<T, V> xr[K], yr[K];
  // RING: slot s of a group holds a row of x and one of y
  const uint32_t row_bytes = static_cast<uint32_t>(A.C * sizeof(T));
  uint8_t* const slots = reinterpret_cast<uint8_t*>(coef + A.C) + static_cast<size_t>(group) * A.stages * 2 * row_bytes;
  auto bar = [&](int slot) { return tc::smem_u32(&bars[group * kMaxStages + slot]); };
  auto fetch = [&](int slot, int64_t r) {
    tc::mbar_expect_tx(bar(slot), A.y ? 2 * row_bytes : row_bytes);
    const uint32_t dst = tc::smem_u32(slots + static_cast<size_t>(slot) * 2 * row_bytes);
    bulk_row(dst, static_cast<const T*>(A.x) + r * A.C, row_bytes, bar(slot));
    if (A.y) bulk_row(dst + row_bytes, static_cast<const T*>(A.y) + r * A.C, row_bytes, bar(slot));
  };
  int slot = 0;
  uint32_t phase = 0;
  int64_t run_end = end;
  if constexpr (RING) {
    if (threadIdx.x == 0) {
      for (int q = 0; q < kGroups * kMaxStages; ++q) tc::mbar_init(tc::smem_u32(&bars[q]), 1);
      abort_flag = 0;
      tc::fence_mbar_init();
    }
    __syncthreads();
    row = A.rows * blockIdx.x / gridDim.x;
    run_end = A.rows * (blockIdx.x + 1) / gridDim.x;
    sample = A.samples == 1 ? 0 : row / A.per_sample;
    row += group;
    if (t == 0)
      for (int q = 0; q < A.stages && row + q * kGroups < run_end; ++q) fetch(q, row + q * kGroups);
  } else {
    if (A.samples > 1 && row < end) sample = row / A.per_sample;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (t + k * TPR) * V;
      const bool ok = row < end && c < A.C;
      if (ok) xr[k].load(static_cast<const T*>(A.x) + row * A.C + c);
      else xr[k].zero();
      if (ok && A.y) yr[k].load(static_cast<const T*>(A.y) + row * A.C + c);
      else yr[k].zero();
    }
  }
  auto coefs = [&](int kind, int c, E (&f)[L::N]) {
    if constexpr (RING) {
#pragma unroll
      for (int i = 0; i < L::N; i += 2) {
        const float4 q = coef[(kind * (V / 4) + i / 2) * pieces + c / V];
        f[i] = tc::pack_f2(q.x, q.y);
        f[i + 1] = tc::pack_f2(q.z, q.w);
      }
    }
  };
  // sum of squares of (v - mean), of the channels that exist
  auto squares = [&](auto&& v, float mean) {
    E s = L::all(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((t + k * TPR) * V >= A.C) break;
#pragma unroll
      for (int i = 0; i < L::N; ++i) {
        const E d = e_add(v(k, i), L::all(-mean));
        s = e_fma(d, d, s);
      }
    }
    return e_sum(s);
  };
  auto total = [&](auto&& v) {
    E s = L::all(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < L::N; ++i) s = e_add(s, v(k, i));
    return e_sum(s);
  };
  const float inv = 1.f / static_cast<float>(A.C);
  // one round per sample of the block's run (RING), else one row
  for (bool more = true; more;) {
  more = false;
  if constexpr (RING) {
    end = min((sample + 1) * A.per_sample, run_end);
    more = end < run_end;
    float* flat = reinterpret_cast<float*>(coef);
    for (int pc = threadIdx.x; pc < pieces; pc += kBlock) {
      // every load before the first use
      uint4 g[2], pw[2], pb[2], w[2], b[2], sc[2], sh[2];
      const int c = pc * V;
      raw_piece<T, V>(A, A.gate, sample, c, g);
      raw_piece<T, V>(A, A.post_weight, 0, c, pw);
      raw_piece<T, V>(A, A.post_bias, 0, c, pb);
      raw_piece<T, V>(A, A.weight, 0, c, w);
      raw_piece<T, V>(A, A.bias, 0, c, b);
      raw_piece<T, V>(A, A.scale, sample, c, sc);
      raw_piece<T, V>(A, A.shift, sample, c, sh);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float gate = piece_value<T, V>(A, A.gate, g, e, 1.f), by = 1.f + piece_value<T, V>(A, A.scale, sc, e, 0.f);
        float* at = flat + ((e / 4) * pieces + pc) * 4 + e % 4;
        at[0] = gate * piece_value<T, V>(A, A.post_weight, pw, e, 1.f);
        at[A.C] = gate * piece_value<T, V>(A, A.post_bias, pb, e, 0.f);
        at[2 * A.C] = by * piece_value<T, V>(A, A.weight, w, e, 1.f);
        at[3 * A.C] = fmaf(by, piece_value<T, V>(A, A.bias, b, e, 0.f), piece_value<T, V>(A, A.shift, sh, e, 0.f));
      }
    }
    __syncthreads();
  }
  for (; row < end; row += kGroups) {
    if constexpr (RING) {
      // (a wait that ran out leaves its code; the rows of this block are then not to be used, and the slot takes no other
      // copy: its barrier still expects the last one)
      const bool arrived = tc::mbar_wait<0>(bar(slot), phase, &abort_flag, A.status, kNormWaits);
      const T* src = reinterpret_cast<const T*>(slots + static_cast<size_t>(slot) * 2 * row_bytes);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (t + k * TPR) * V;
        if (c < A.C) {
          xr[k].v = *reinterpret_cast<const uint4*>(src + c);
          if (A.y) yr[k].v = *reinterpret_cast<const uint4*>(src + A.C + c);
          else yr[k].zero();
        } else {
          xr[k].zero();
          yr[k].zero();
        }
      }
      // the row is in registers: its place takes the next one, once these loads are done
      tc::fence_proxy_async();
      if constexpr (TPR == 32) __syncwarp();
      else tc::bar_sync_named(1 + group, TPR);
      const int64_t ahead = row + static_cast<int64_t>(A.stages) * kGroups;
      if (t == 0 && arrived && ahead < run_end) fetch(slot, ahead);
      if (++slot == A.stages) {
        slot = 0;
        phase ^= 1u;
      }
    }
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
    if (A.y && A.post != kNone) {
      auto y = [&](int k, int i) { return yr[k].get(i); };
      if (A.post == kLayer) st.z = sum(total(y)) * inv;
      st.w = rsqrtf(sum(squares(y, st.z)) * inv + A.eps);
    }
    E z[K][L::N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (t + k * TPR) * V;
#pragma unroll
      for (int i = 0; i < L::N; ++i) z[k][i] = xr[k].get(i);
      if (A.y == nullptr || c >= A.C) continue;
      E g[L::N], p[L::N];
#pragma unroll
      for (int i = 0; i < L::N; ++i) p[i] = yr[k].get(i);
      if constexpr (RING) coefs(0, c, g);
      else load_param<T, V>(A, A.gate, sample, c, 1.f, g);
      if (A.post != kNone) {
        E b[L::N];
        const E r = L::all(st.w), m = L::all(-st.z);
        if constexpr (RING) {
          coefs(1, c, b);
#pragma unroll
          for (int i = 0; i < L::N; ++i) p[i] = e_fma(e_mul(e_add(p[i], m), r), g[i], b[i]);
        } else {
          E w[L::N];
          load_param<T, V>(A, A.post_weight, 0, c, 1.f, w);
          load_param<T, V>(A, A.post_bias, 0, c, 0.f, b);
#pragma unroll
          for (int i = 0; i < L::N; ++i) p[i] = e_mul(g[i], e_fma(e_mul(e_add(p[i], m), r), w[i], b[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < L::N; ++i) p[i] = e_mul(g[i], p[i]);
      }
      const E al = L::all(A.alpha);
#pragma unroll
      for (int i = 0; i < L::N; ++i) z[k][i] = e_fma(al, z[k][i], p[i]);
      store_piece<T, V>(static_cast<T*>(A.z) + row * A.C + c, z[k]);
    }
    if (A.pre != kNone) {
      auto zv = [&](int k, int i) { return z[k][i]; };
      if (A.pre == kLayer) st.x = sum(total(zv)) * inv;
      st.y = rsqrtf(sum(squares(zv, st.x)) * inv + A.eps);
      const E r = L::all(st.y), m = L::all(-st.x);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (t + k * TPR) * V;
        if (c >= A.C) break;
        E w[L::N], b[L::N], o[L::N];
        if constexpr (RING) {
          coefs(2, c, w);
          coefs(3, c, b);
        } else {
          load_param<T, V>(A, A.weight, 0, c, 1.f, w);
          load_param<T, V>(A, A.bias, 0, c, 0.f, b);
        }
#pragma unroll
        for (int i = 0; i < L::N; ++i) o[i] = e_fma(e_mul(e_add(z[k][i], m), r), w[i], b[i]);
        if constexpr (!RING) {
          if (A.scale.p || A.shift.p) {
            load_param<T, V>(A, A.scale, sample, c, 0.f, w);
            load_param<T, V>(A, A.shift, sample, c, 0.f, b);
#pragma unroll
            for (int i = 0; i < L::N; ++i) o[i] = e_fma(o[i], e_add(w[i], L::all(1.f)), b[i]);
          }
        }
        store_piece<T, V>(static_cast<T*>(A.h) + row * A.C + c, o);
      }
    }
    if (A.stats && t == 0) A.stats[row] = st;
  }
  if (RING && more) {
    __syncthreads();  // (the parameters have been read)
    ++sample;
  }
  }
  if (RING && abort_flag) __nanosleep(20000);  // rows in flight land before the shared memory is handed on
}

// A block walks a run of one sample's rows, R at a time; a thread keeps its channels, so that the sums over
// rows stay in its registers.  The next R rows are loaded while these are worked on.  Normalised values are
// (z - mean) r as in the forward pass: z r - mean r would round mean r, which costs a row whose mean is thousands of
// deviations as many of its digits.
template <typename T, int V, int K, int R, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 ? 3 : 1) norm_rows_backward_kernel(const Args A) {
  using L = Elem<V>;
  using E = typename L::E;
  constexpr int N = L::N;
  __shared__ float red[2 * 32 * 2 * R];
  extern __shared__ float4 coef[];  // remake with a post norm, wide rows: gate * post_bias of every thread's pieces
  int turn = 0;
  const int t = threadIdx.x, nt = blockDim.x;
  // (quarters of a piece apart: a warp's reads are whole lines)
  auto shift_at = [&](int k, int i) {
    const int c = (t + k * nt) * V;
    if constexpr (V == 1) return reinterpret_cast<float*>(coef) + c;
    else return reinterpret_cast<E*>(coef + (i / 2) * (A.C / V) + c / V) + i % 2;
  };
  const int64_t sample = blockIdx.x / A.chunks;
  const int chunk = static_cast<int>(blockIdx.x % A.chunks);
  const int64_t begin = sample * A.per_sample + A.per_sample * chunk / A.chunks;
  const int64_t end = sample * A.per_sample + A.per_sample * (chunk + 1) / A.chunks;
  const float inv = 1.f / static_cast<float>(A.C);
  const T* zp = static_cast<const T*>(A.z_in);
  const T* yp = static_cast<const T*>(A.y);
  const T* gzp = static_cast<const T*>(A.gz);
  const T* ghp = static_cast<const T*>(A.gh);
  struct Rows {
    Raw<T, V> z[R][K], y[R][K], gz[R][K], gh[R][K];
    float4 st[R];
  };
  auto load = [&](Rows& b, int64_t row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r;
      b.st[r] = row < end ? __ldg(A.stats + row) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (t + k * nt) * V;
        const bool live = row < end && c < A.C;
        const int64_t at = row * A.C + c;
        if (live && ghp) { b.gh[r][k].load(ghp + at); b.z[r][k].load(zp + at); }
        else { b.gh[r][k].zero(); b.z[r][k].zero(); }
        if (live && gzp) b.gz[r][k].load(gzp + at); else b.gz[r][k].zero();
        if (live && yp) b.y[r][k].load(yp + at); else b.y[r][k].zero();
      }
    }
  };
  Rows cur, next;
  load(cur, begin);
  E wp[K][N], wq[K][N];  // weight (1 + scale), gate * post_weight
  E sa[K][N], sb[K][N], sc[K][N], sd[K][N];
  E wb[K][N];                // gate * post_bias, narrow rows
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (t + k * nt) * V;
#pragma unroll
    for (int i = 0; i < N; ++i) wp[k][i] = wq[k][i] = wb[k][i] = sa[k][i] = sb[k][i] = sc[k][i] = sd[k][i] = L::all(0.f);
    if (c < A.C) {
      E q[N];
      load_param<T, V>(A, A.weight, 0, c, 1.f, wp[k]);
      load_param<T, V>(A, A.scale, sample, c, 0.f, q);
#pragma unroll
      for (int i = 0; i < N; ++i) wp[k][i] = e_fma(wp[k][i], q[i], wp[k][i]);
      load_param<T, V>(A, A.gate, sample, c, 1.f, wq[k]);
      if (A.post != kNone) {
        if (sizeof(T) == 2 && A.remake) {  // (a thread reads back what it writes)
          load_param<T, V>(A, A.post_bias, 0, c, 0.f, q);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if constexpr (MAXT == 128) wb[k][i] = e_mul(wq[k][i], q[i]);
            else *shift_at(k, i) = e_mul(wq[k][i], q[i]);
          }
        }
        load_param<T, V>(A, A.post_weight, 0, c, 1.f, q);
#pragma unroll
        for (int i = 0; i < N; ++i) wq[k][i] = e_mul(wq[k][i], q[i]);
      }
    }
  }
  // the normalised value of pre, 16 bits
  auto n_at = [&](int r, int k, int i) {
    E z = cur.z[r][k].get(i);
    if (A.remake) {
      E p = e_mul(e_add(cur.y[r][k].get(i), L::all(-cur.st[r].z)), L::all(cur.st[r].w));  // (y itself without a post norm)
      p = A.post != kNone && (t + k * nt) * V < A.C ? e_fma(p, wq[k][i], *shift_at(k, i)) : e_mul(p, wq[k][i]);
      z = e_fma(L::all(A.alpha), z, p);
    }
    return e_mul(e_add(z, L::all(-cur.st[r].x)), L::all(cur.st[r].y));
  };
  for (int64_t row0 = begin; row0 < end; row0 += R) {
    load(next, row0 + R);
    E G[R][K][N];
    if (ghp) {
      float s[2 * R];
      // z as it lies in memory (0), or from x and y without (1) and with (2) a post norm; 3 finds out value by value,
      // which is what wide rows want (32768 x 4096 bf16 without a post norm, forward and backward: 586 us with three
      // loops, 524 with one, 550 from the rounded z; 50432 x 768 with one: 224, 234, 216)
      auto pass = [&](auto way) {
        constexpr int kWay = decltype(way)::value;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const E by = L::all(cur.st[r].y), mean = L::all(-cur.st[r].x);
          const E by_y = L::all(cur.st[r].w), mean_y = L::all(-cur.st[r].z), al = L::all(A.alpha);
          E s1 = L::all(0.f), s2 = L::all(0.f);
#pragma unroll
          for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const E g = cur.gh[r][k].get(i);
              E z = cur.z[r][k].get(i);
              if constexpr (kWay == 1) z = e_fma(al, z, e_mul(cur.y[r][k].get(i), wq[k][i]));
              if constexpr (kWay == 2)
                z = e_fma(al, z, e_fma(e_mul(e_add(cur.y[r][k].get(i), mean_y), by_y), wq[k][i], wb[k][i]));
              E n;
              if constexpr (kWay == 3) n = n_at(r, k, i);
              else n = e_mul(e_add(z, mean), by);
              const E w = e_mul(g, wp[k][i]);
              G[r][k][i] = n;
              s1 = e_add(s1, w);
              s2 = e_fma(w, n, s2);
              sa[k][i] = e_add(sa[k][i], g);
              sb[k][i] = e_fma(g, n, sb[k][i]);
            }
          }
          s[2 * r] = e_sum(s1);
          s[2 * r + 1] = e_sum(s2);
        }
      };
      if constexpr (sizeof(T) == 4) {
        pass(std::integral_constant<int, 0>());
      } else if constexpr (MAXT > 128) {
        pass(std::integral_constant<int, 3>());
      } else {
        if (!A.remake) pass(std::integral_constant<int, 0>());
        else if (A.post == kNone) pass(std::integral_constant<int, 1>());
        else pass(std::integral_constant<int, 2>());
      }
      block_sum<2 * R>(s, red, turn);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const E m1 = L::all(A.pre == kLayer ? -s[2 * r] * inv : 0.f), m2 = L::all(-s[2 * r + 1] * inv);
        const E by = L::all(cur.st[r].y);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const E n = G[r][k][i];
            G[r][k][i] = e_fma(by, e_fma(n, m2, e_fma(cur.gh[r][k].get(i), wp[k][i], m1)), cur.gz[r][k].get(i));
          }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < N; ++i) G[r][k][i] = cur.gz[r][k].get(i);
    }
    if (A.gx) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (t + k * nt) * V;
          if (row0 + r >= end || c >= A.C) continue;
          E o[N];
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = e_mul(L::all(A.alpha), G[r][k][i]);
          store_piece<T, V>(static_cast<T*>(A.gx) + (row0 + r) * A.C + c, o);
        }
    }
    if (yp) {
      float s[2 * R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[2 * r] = s[2 * r + 1] = 0.f;
        if (row0 + r >= end) continue;  // (rows of the next run must not join the sums)
        const E by = L::all(cur.st[r].w), mean = L::all(-cur.st[r].z);
        E s1 = L::all(0.f), s2 = L::all(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if ((t + k * nt) * V >= A.C) continue;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const E m = e_mul(e_add(cur.y[r][k].get(i), mean), by), f = e_mul(G[r][k][i], wq[k][i]);
            s1 = e_add(s1, f);
            s2 = e_fma(f, m, s2);
            sc[k][i] = e_add(sc[k][i], G[r][k][i]);
            sd[k][i] = e_fma(G[r][k][i], m, sd[k][i]);
          }
        }
        s[2 * r] = e_sum(s1);
        s[2 * r + 1] = e_sum(s2);
      }
      if (A.post != kNone) block_sum<2 * R>(s, red, turn);
      if (A.gy) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const E m1 = L::all(A.post == kLayer ? -s[2 * r] * inv : 0.f), m2 = L::all(A.post != kNone ? -s[2 * r + 1] * inv : 0.f);
          const E by = L::all(cur.st[r].w), mean = L::all(-cur.st[r].z);
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const int c = (t + k * nt) * V;
            if (row0 + r >= end || c >= A.C) continue;
            E o[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const E m = e_mul(e_add(cur.y[r][k].get(i), mean), by);
              o[i] = e_mul(by, e_fma(m, m2, e_fma(G[r][k][i], wq[k][i], m1)));
            }
            store_piece<T, V>(static_cast<T*>(A.gy) + (row0 + r) * A.C + c, o);
          }
        }
      }
    }
    cur = next;
  }
  if (A.part) {
    float* part = A.part + static_cast<int64_t>(blockIdx.x) * 4 * A.C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (t + k * nt) * V;
      if (c >= A.C) break;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (V == 1) {
          part[c] = sa[k][0];
          part[A.C + c] = sb[k][0];
          part[2 * A.C + c] = sc[k][0];
          part[3 * A.C + c] = sd[k][0];
        } else {
          *reinterpret_cast<uint64_t*>(part + c + 2 * i) = sa[k][i];
          *reinterpret_cast<uint64_t*>(part + A.C + c + 2 * i) = sb[k][i];
          *reinterpret_cast<uint64_t*>(part + 2 * A.C + c + 2 * i) = sc[k][i];
          *reinterpret_cast<uint64_t*>(part + 3 * A.C + c + 2 * i) = sd[k][i];
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// batch-last: a token is a column
// ---------------------------------------------------------------------------
// A block takes 32 tokens of one sample, a lane per token; its W warps share the channels.
constexpr int kColWarps = 16;

// sum over the block's warps of a value per token
__device__ __forceinline__ float column_sum(float v, float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  red[warp * 32 + lane] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < kColWarps; ++w) s += red[w * 32 + lane];
  __syncthreads();
  return s;
}

// z stays in shared memory (128 bytes per channel, up to 1536 of them).  Every thread has 16 to 32 loads in flight:
// the block's latencies are what bounds it (768 x 6501 fp16, 40 MB: 93 us when every statistic read the tensors
// again and the loads waited for one another, 22.5 now; floor 6).
constexpr int kColStep = 16;  // channels that a warp loads at once
constexpr int kColumnChannels = 1536;

template <typename T>
__global__ void __launch_bounds__(kColWarps * 32) norm_columns_kernel(const Args A) {
  __shared__ float red[kColWarps * 32];
  extern __shared__ float4 coef[];  // combined parameters of the channels, then z
  float* const zc = reinterpret_cast<float*>(coef + A.C);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t sample = blockIdx.x / A.chunks;
  const int64_t in_sample = static_cast<int64_t>(blockIdx.x % A.chunks) * 32 + lane;
  const bool live = in_sample < A.per_sample;
  const int64_t tok = sample * A.per_sample + (live ? in_sample : 0);
  const T* x = static_cast<const T*>(A.x) + tok;
  const T* y = A.y ? static_cast<const T*>(A.y) + tok : nullptr;
  const float inv = 1.f / static_cast<float>(A.C);
  for (int c = threadIdx.x; c < A.C; c += kColWarps * 32) coef[c] = combined<T>(A, sample, c);
  __syncthreads();
  const int64_t step = kColWarps * A.rows;  // elements between a warp's channels
  // calls f(c, o, p[o], q[o]) for the warp's channels, o = c * rows, loads of a step ahead of their uses
  auto walk = [&](const T* p, const T* q, auto&& f) {
    int c = warp;
    int64_t o = c * A.rows;
    for (; c + (kColStep - 1) * kColWarps < A.C; c += kColStep * kColWarps, o += kColStep * step) {
      T a[kColStep], b[kColStep];
#pragma unroll
      for (int u = 0; u < kColStep; ++u) {
        a[u] = p[o + u * step];
        if (q) b[u] = q[o + u * step];
      }
#pragma unroll
      for (int u = 0; u < kColStep; ++u)
        f(c + u * kColWarps, o + u * step, ElemTraits<T>::to_float(a[u]), q ? ElemTraits<T>::to_float(b[u]) : 0.f);
    }
#pragma unroll 4
    for (; c < A.C; c += kColWarps, o += step) f(c, o, ElemTraits<T>::to_float(p[o]), q ? ElemTraits<T>::to_float(q[o]) : 0.f);
  };
  float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
  if (y && A.post != kNone) {
    float s = 0.f;
    if (A.post == kLayer) {
      walk(y, nullptr, [&](int, int64_t, float v, float) { s += v; });
      st.z = column_sum(s, red) * inv;
      s = 0.f;
    }
    walk(y, nullptr, [&](int, int64_t, float v, float) { s = fmaf(v - st.z, v - st.z, s); });
    st.w = rsqrtf(column_sum(s, red) * inv + A.eps);
  }
  auto join = [&](int c, float xv, float yv) {
    if (!y) return xv;
    const float4 q = coef[c];
    return fmaf(A.alpha, xv, A.post != kNone ? fmaf((yv - st.z) * st.w, q.x, q.y) : q.x * yv);
  };
  // z of every channel, to shared memory and (where there is a y) to memory, and its sum
  float s = 0.f;
  T* const zo = static_cast<T*>(A.z) + tok;
  T* const ho = static_cast<T*>(A.h) + tok;
  walk(x, y, [&](int c, int64_t o, float xv, float yv) {
    const float z = join(c, xv, yv);
    s += z;
    zc[c * 32 + lane] = z;
    if (y && live) zo[o] = ElemTraits<T>::from_float(z);
  });
  if (A.pre != kNone) {
    auto again = [&](auto&& f) {  // (a thread reads what it has written)
      int64_t o = warp * A.rows;
#pragma unroll 8
      for (int c = warp; c < A.C; c += kColWarps, o += step) f(c, o, zc[c * 32 + lane]);
    };
    if (A.pre == kLayer) st.x = column_sum(s, red) * inv;
    float v = 0.f;
    again([&](int, int64_t, float z) { v = fmaf(z - st.x, z - st.x, v); });
    st.y = rsqrtf(column_sum(v, red) * inv + A.eps);
    if (live)
      again([&](int c, int64_t o, float z) {
        const float4 q = coef[c];
        ho[o] = ElemTraits<T>::from_float(fmaf((z - st.x) * st.y, q.z, q.w));
      });
  }
  if (live && A.stats && warp == 0) A.stats[tok] = st;
}

// v[i] of all lanes summed into lane i (31 exchanges for 32 sums)
__device__ __forceinline__ float reduce_scatter(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], send = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// The normalised values of pre stay in shared memory between the passes (128 bytes per channel, as z in the forward pass):
// forward and backward of 768 x 6501 bf16 with both norms 158 us when every pass read z again, 148 so, with z formed
// from x and y on the way.
template <typename T>
__global__ void __launch_bounds__(kColWarps * 32) norm_columns_backward_kernel(const Args A) {
  __shared__ float red[kColWarps * 32];
  extern __shared__ float4 coef[];  // per channel: gate * post_weight, gate * post_bias, weight (1 + scale); then n
  float* const nc = reinterpret_cast<float*>(coef + A.C);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t sample = blockIdx.x / A.chunks;
  const int64_t in_sample = static_cast<int64_t>(blockIdx.x % A.chunks) * 32 + lane;
  const bool live = in_sample < A.per_sample;
  const int64_t tok = sample * A.per_sample + (live ? in_sample : 0);
  for (int c = threadIdx.x; c < A.C; c += kColWarps * 32) coef[c] = combined<T>(A, sample, c);
  __syncthreads();
  const T* zp = static_cast<const T*>(A.z_in) + tok;
  const T* yp = A.y ? static_cast<const T*>(A.y) + tok : nullptr;
  const T* gzp = A.gz ? static_cast<const T*>(A.gz) + tok : nullptr;
  const T* ghp = A.gh ? static_cast<const T*>(A.gh) + tok : nullptr;
  const float inv = 1.f / static_cast<float>(A.C);
  const float4 st = __ldg(A.stats + tok);
  // (a lane beyond the sample's end reads zeros for its gradients)
  auto at = [&](const T* p, int c) { return ElemTraits<T>::to_float(p[c * A.rows]); };
  float m1 = 0.f, m2 = 0.f, q1 = 0.f, q2 = 0.f;
  if (ghp) {
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 8
    for (int c = warp; c < A.C; c += kColWarps) {
      const float4 q = coef[c];
      const float w = (live ? at(ghp, c) : 0.f) * q.z;
      float z = at(zp, c);
      if (sizeof(T) == 2 && A.remake) z = fmaf(A.alpha, z, A.post != kNone ? fmaf((at(yp, c) - st.z) * st.w, q.x, q.y) : q.x * at(yp, c));
      const float n = (z - st.x) * st.y;
      nc[c * 32 + lane] = n;
      s1 += w;
      s2 = fmaf(w, n, s2);
    }
    if (A.pre == kLayer) m1 = column_sum(s1, red) * inv;
    m2 = column_sum(s2, red) * inv;
  }
  auto G_at = [&](int c, float gh, float n) {
    float g = live && gzp ? at(gzp, c) : 0.f;
    if (ghp) {
      const float w = gh * coef[c].z;
      g = fmaf(st.y, w - m1 - n * m2, g);
    }
    return live ? g : 0.f;
  };
  if (yp && A.post != kNone) {
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 8
    for (int c = warp; c < A.C; c += kColWarps) {
      const float gh = live && ghp ? at(ghp, c) : 0.f, n = ghp ? nc[c * 32 + lane] : 0.f;
      const float f = G_at(c, gh, n) * coef[c].x;
      s1 += f;
      s2 = fmaf(f, (at(yp, c) - st.z) * st.w, s2);
    }
    if (A.post == kLayer) q1 = column_sum(s1, red) * inv;
    q2 = column_sum(s2, red) * inv;
  }
  float* part = A.part ? A.part + static_cast<int64_t>(blockIdx.x) * 4 * A.C : nullptr;
  // eight channels at a time: their four sums over the 32 tokens are one reduction
  for (int c0 = warp * 8; c0 < A.C; c0 += kColWarps * 8) {
    float v[32];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int c = c0 + u;
      const bool ok = c < A.C;
      float gh = 0.f, n = 0.f, G = 0.f, m = 0.f;
      if (ok) {
        if (ghp) {
          gh = live ? at(ghp, c) : 0.f;
          n = nc[c * 32 + lane];
        }
        G = G_at(c, gh, n);
        if (live && A.gx) static_cast<T*>(A.gx)[c * A.rows + tok] = ElemTraits<T>::from_float(A.alpha * G);
        if (yp) {
          m = (at(yp, c) - st.z) * st.w;
          if (live && A.gy) {
            const float f = G * coef[c].x - q1 - m * q2;
            static_cast<T*>(A.gy)[c * A.rows + tok] = ElemTraits<T>::from_float(st.w * f);
          }
        }
      }
      v[u] = gh;
      v[8 + u] = live ? gh * n : 0.f;
      v[16 + u] = G;
      v[24 + u] = live ? G * m : 0.f;
    }
    if (part) {
      const float total = reduce_scatter(v);
      const int c = c0 + (lane & 7);
      if (c < A.C) part[(lane >> 3) * A.C + c] = total;
    }
  }
}

// ---------------------------------------------------------------------------
// parameters' gradients from the partial sums
// ---------------------------------------------------------------------------
struct Grads {
  void *weight, *bias, *post_weight, *post_bias, *scale, *shift, *gate;
  int scale_rows, shift_rows, gate_rows;  // per sample (1) or one row for all (0)
};

template <typename T>
__device__ __forceinline__ void put(const Args& A, void* p, int64_t at, float v) {
  if (!p) return;
  if (A.p32) static_cast<float*>(p)[at] = v;
  else static_cast<T*>(p)[at] = ElemTraits<T>::from_float(v);
}

// Slices of a sum of n: a column of partial sums is a thread's chain of loads (23598 x 143 fp32, 888 partial sums: 23 us
// in 8 slices, 13 in 32; 64 of 6464 channels: 4 and 8).
inline unsigned slices_of(int64_t n) { return n >= 256 ? 32 : 8; }

// the parameters of one channel and sample
struct Params {
  float w, b, pw, pb, sc, ga;
};
template <typename T>
__device__ __forceinline__ Params params_at(const Args& A, int64_t sample, int c) {
  const uint32_t w = raw_param(A, A.weight, 0, c), b = raw_param(A, A.bias, 0, c), pw = raw_param(A, A.post_weight, 0, c);
  const uint32_t pb = raw_param(A, A.post_bias, 0, c), sc = raw_param(A, A.scale, sample, c), ga = raw_param(A, A.gate, sample, c);
  return {param_value<T>(A, A.weight, w, 1.f), param_value<T>(A, A.bias, b, 0.f), param_value<T>(A, A.post_weight, pw, 1.f),
          param_value<T>(A, A.post_bias, pb, 0.f), 1.f + param_value<T>(A, A.scale, sc, 0.f), param_value<T>(A, A.gate, ga, 1.f)};
}

// 32 channels by 8 or 32 slices: first == 1 adds the chunks of sample blockIdx.y and writes the gradients of
// per-sample parameters and the sample's sums; first == 0 adds the samples.  With one sample the first does all.
template <typename T>
__global__ void __launch_bounds__(1024) norm_param_grads_kernel(const Args A, const Grads g, const float* part, float* sums,
                                                                        int first) {
  __shared__ float red[32][7][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, slices = blockDim.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const bool ok = c < A.C;
  const int at_c = ok ? c : 0;
  const int64_t sample = blockIdx.y;
  const Params own = params_at<T>(A, sample, at_c);  // (its loads are in flight with those of the sums)
  float t[7] = {};
  if (first) {
    const float* p = part + sample * A.chunks * 4 * A.C + at_c;
#pragma unroll 2
    for (int q = slice; q < A.chunks; q += slices)
#pragma unroll
      for (int s = 0; s < 4; ++s) t[s] += p[(static_cast<int64_t>(q) * 4 + s) * A.C];
  } else {
#pragma unroll 2
    for (int64_t s = slice; s < A.samples; s += slices) {
      const float* p = part + s * 4 * A.C + at_c;
      const float a = p[0], bb = p[A.C], cc = p[2 * A.C], d = p[3 * A.C];
      const uint32_t sr = raw_param(A, A.scale, s, at_c), gr = raw_param(A, A.gate, s, at_c);
      const float sc = 1.f + param_value<T>(A, A.scale, sr, 0.f), ga = param_value<T>(A, A.gate, gr, 1.f);
      t[0] = fmaf(sc, bb, t[0]);
      t[1] = fmaf(sc, a, t[1]);
      t[2] = fmaf(ga, d, t[2]);
      t[3] = fmaf(ga, cc, t[3]);
      t[4] += fmaf(own.w, bb, own.b * a);
      t[5] += a;
      t[6] += fmaf(own.pw, d, own.pb * cc);
    }
  }
#pragma unroll
  for (int s = 0; s < 7; ++s) red[slice][s][lane] = t[s];
  __syncthreads();
  if (slice != 0 || !ok) return;
#pragma unroll
  for (int s = 0; s < 7; ++s) {
    t[s] = 0.f;
#pragma unroll 8
    for (int q = 0; q < slices; ++q) t[s] += red[q][s][lane];
  }
  if (first) {
    const bool one = A.samples == 1;
    const int64_t at = sample * A.C + c;
    if (one || g.scale_rows) put<T>(A, g.scale, at, fmaf(own.w, t[1], own.b * t[0]));
    if (one || g.shift_rows) put<T>(A, g.shift, at, t[0]);
    if (one || g.gate_rows) put<T>(A, g.gate, at, fmaf(own.pw, t[3], own.pb * t[2]));
    if (one) {
      put<T>(A, g.weight, c, own.sc * t[1]);
      put<T>(A, g.bias, c, own.sc * t[0]);
      put<T>(A, g.post_weight, c, own.ga * t[3]);
      put<T>(A, g.post_bias, c, own.ga * t[2]);
    } else if (sums) {
#pragma unroll
      for (int s = 0; s < 4; ++s) sums[(sample * 4 + s) * A.C + c] = t[s];
    }
  } else {
    put<T>(A, g.weight, c, t[0]);
    put<T>(A, g.bias, c, t[1]);
    put<T>(A, g.post_weight, c, t[2]);
    put<T>(A, g.post_bias, c, t[3]);
    if (!g.scale_rows) put<T>(A, g.scale, c, t[4]);
    if (!g.shift_rows) put<T>(A, g.shift, c, t[5]);
    if (!g.gate_rows) put<T>(A, g.gate, c, t[6]);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int launched(const char* what) {
  count_launch();
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(err));
  return KSMM_OK;
}

bool whole_pieces(const void* p, int64_t ld, int es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * es) % 16 == 0;
}

// can tokens and parameters be read in 16-byte pieces?
bool vector_rows(const ksmm_norm_desc_t& d) {
  const int es = dtype_size(d.dtype), ps = dtype_size(d.param_dtype);
  const struct { const void* p; int64_t ld; } params[7] = {{d.weight, 0}, {d.bias, 0}, {d.post_weight, 0}, {d.post_bias, 0},
                                                          {d.scale, d.scale_stride}, {d.shift, d.shift_stride}, {d.gate, d.gate_stride}};
  for (const auto& q : params)
    if (!whole_pieces(q.p, q.ld, ps)) return false;
  for (const void* p : {d.x, d.y, static_cast<const void*>(d.z), static_cast<const void*>(d.h), d.grad_z, d.grad_h,
                        static_cast<const void*>(d.grad_x), static_cast<const void*>(d.grad_y)})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return (static_cast<int64_t>(d.channels) * es) % 16 == 0;
}

// does the backward pass form z from x and y?
bool remakes_z(const ksmm_norm_desc_t& d) { return d.y && !d.z && d.grad_h && d.dtype != KSMM_F32; }

Args args_of(const ksmm_norm_desc_t& d) {
  Args A = {};
  A.x = d.x; A.y = d.y; A.z = d.z; A.h = d.h;
  A.remake = remakes_z(d);
  A.z_in = d.y && !A.remake ? d.z : d.x;
  A.gz = d.grad_z; A.gh = d.grad_h; A.gx = d.grad_x; A.gy = d.grad_y;
  A.stats = reinterpret_cast<float4*>(d.stats);
  A.weight = {d.weight, 0}; A.bias = {d.bias, 0};
  A.post_weight = {d.post_weight, 0}; A.post_bias = {d.post_bias, 0};
  A.scale = {d.scale, d.scale_stride}; A.shift = {d.shift, d.shift_stride}; A.gate = {d.gate, d.gate_stride};
  A.rows = d.rows;
  A.samples = d.samples;
  A.per_sample = d.samples > 0 ? d.rows / d.samples : 0;
  A.C = d.channels; A.pre = d.norm; A.post = d.post_norm;
  A.p32 = d.param_dtype == KSMM_F32;
  A.alpha = d.y ? d.alpha : 1.f;
  A.eps = d.eps;
  return A;
}

// Dynamic shared memory beyond 48 KB needs a word with the driver, once per kernel and device, for `most`: what any call of
// the kernel may ask for.  (The driver keeps the last value, so that a limit of a call's own size could be lowered
// by another thread's call between this one's word and its launch.  A repeated set of one value is harmless.)
using Granted = std::atomic<bool>[64];
int allow_smem(const void* kern, size_t bytes, size_t most, Granted& granted) {
  if (bytes <= 40 * 1024) return KSMM_OK;  // (what a kernel declares itself, up to 2 KB here, counts as well)
  if (bytes > most) return set_error(KSMM_ERR_UNSUPPORTED, "norm: %zu bytes of shared memory", bytes);
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < 64;
  if (known && granted[dev].load(std::memory_order_relaxed)) return KSMM_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
  if (e != cudaSuccess) return set_error(KSMM_ERR_CUDA, "cannot reserve %zu bytes of shared memory: %s", most, cudaGetErrorString(e));
  if (known) granted[dev].store(true, std::memory_order_relaxed);
  return KSMM_OK;
}

template <typename T, int V, int K, int TPR, bool RING = false>
int go_rows(Args A, cudaStream_t stream) {
  constexpr int kBlock = RING ? (TPR == 32 ? kRingBlock : kRingWide) : (TPR < 128 ? 128 : TPR);
  int64_t grid = (A.rows + kBlock / TPR - 1) / (kBlock / TPR);
  constexpr size_t room = TPR == 32 ? 110 * 1024 : 224 * 1024;  // of a ring
  size_t smem = 0;
  if (RING) {
    A.status = tc::status_word();
    if (!A.status) return set_error(KSMM_ERR_CUDA, "cannot resolve the device status word");
    grid = tc::num_sms() * (TPR == 32 ? 2 : 1);
    const size_t coefs = static_cast<size_t>(A.C) * sizeof(float4), slot = static_cast<size_t>(A.C) * 2 * sizeof(T) * (kBlock / TPR);
    A.stages = static_cast<int>(std::min<size_t>(TPR == 32 ? 6 : 12, (room - coefs) / slot));
    smem = coefs + A.stages * slot;
  }
  if (grid > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "norm: too many rows");
  static Granted granted;
  const int st = allow_smem(reinterpret_cast<const void*>(norm_rows_kernel<T, V, K, TPR, RING>), smem, room, granted);
  if (st != KSMM_OK) return st;
  norm_rows_kernel<T, V, K, TPR, RING><<<static_cast<unsigned>(grid), kBlock, smem, stream>>>(A);
  return launched("norm");
}

template <typename T, int V>
int launch_rows(const Args& A, cudaStream_t stream) {
  const int pieces = (A.C + V - 1) / V;
  if constexpr (V > 1) {
    // Resident blocks against rows one by one, bf16, with gate, scale and shift for 32 to 600 tokens each and without: 768
    // channels, 2368 rows 7.3 and 8.3 us, 6.3 and 6.2; 4800 rows 11.7 and 16.5, 10.3 and 10.3; 12544 rows 22.6 and 40,
    // 18 and 22.6.  4096 channels, 600 rows 10.3 and 12.4, 9.3 and 10.3; 1184 rows 14.4 and 20.4, 10.3 and 14.4.  256
    // channels, 2368 rows 6.2 and 6.2, 6.2 and 4.7.  (Samples of 16 tokens gain as well, 24 and 40 for 12544 x 768, and
    // go one by one still.)
    if (pieces <= 8) return go_rows<T, V, 1, 8>(A, stream);
    if (pieces <= 16) return go_rows<T, V, 2, 8>(A, stream);
    if (pieces <= 128 && A.per_sample >= 32 && A.rows >= 148 * 16) {
      if (pieces <= 32) return go_rows<T, V, 1, 32, true>(A, stream);
      if (pieces <= 64) return go_rows<T, V, 2, 32, true>(A, stream);
      if (pieces <= 96) return go_rows<T, V, 3, 32, true>(A, stream);
      return go_rows<T, V, 4, 32, true>(A, stream);
    }
    if (pieces > 128 && pieces <= 1024 && A.per_sample >= 24 && A.rows >= 148 * 8) {
      if (pieces <= 256) return go_rows<T, V, 2, 128, true>(A, stream);
      return pieces <= 512 ? go_rows<T, V, 4, 128, true>(A, stream) : go_rows<T, V, 4, 256, true>(A, stream);
    }
    if (pieces <= 128) return go_rows<T, V, 4, 32>(A, stream);
    if constexpr (V == 4) {
      if (pieces > 1024) return go_rows<T, V, 4, 512>(A, stream);
    }
    return go_rows<T, V, 4, 256>(A, stream);
  } else {
    if (pieces <= 256) return go_rows<T, 1, 8, 32>(A, stream);
    // (10000 x 1303 bf16: 417 us with 1024 threads per row, one block on an SM; 101 with 256)
    if (pieces <= 2048) return go_rows<T, 1, 8, 256>(A, stream);
    return go_rows<T, 1, 8, 1024>(A, stream);
  }
}

template <typename T, int V>
int launch_rows_backward(const Args& A, cudaStream_t stream) {
  const int pieces = (A.C + V - 1) / V;
  const int64_t grid = A.samples * A.chunks;
  if (grid > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "norm: too many rows");
  const int k = (pieces + 511) / 512;
  auto go = [&](auto kern, int kk) {
    const int n = ((pieces + kk - 1) / kk + 31) / 32 * 32;
    kern<<<static_cast<unsigned>(grid), n, A.remake && A.post != kNone ? A.C * sizeof(float) : 0, stream>>>(A);
    return launched("norm backward");
  };
  if constexpr (V > 1) {
    if (pieces <= 128) return go(norm_rows_backward_kernel<T, V, 1, 2, 128>, 1);
    if (k <= 1) return go(norm_rows_backward_kernel<T, V, 1, 1, 512>, 1);
    if constexpr (V == 4) {
      if (k > 2) return go(norm_rows_backward_kernel<T, V, 4, 1, 512>, 4);
    }
    return go(norm_rows_backward_kernel<T, V, 2, 1, 512>, 2);
  } else {
    if (k <= 1) return go(norm_rows_backward_kernel<T, 1, 1, 2, 512>, 1);
    if (k <= 4) return go(norm_rows_backward_kernel<T, 1, 4, 1, 512>, 4);
    return go(norm_rows_backward_kernel<T, 1, 8, 1, 1024>, 8);
  }
}

template <typename T>
int forward_typed(const ksmm_norm_desc_t& d, cudaStream_t stream) {
  Args A = args_of(d);
  if (!d.bs_last)
    return vector_rows(d) ? launch_rows<T, 16 / sizeof(T)>(A, stream) : launch_rows<T, 1>(A, stream);
  const int64_t chunks = (A.per_sample + 31) / 32;
  if (chunks * A.samples > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "norm: too many tokens");
  A.chunks = static_cast<int>(chunks);
  constexpr size_t per_channel = sizeof(float4) + 32 * sizeof(float);
  const size_t smem = A.C * per_channel;
  static Granted granted;
  const int st = allow_smem(reinterpret_cast<const void*>(norm_columns_kernel<T>), smem, kColumnChannels * per_channel, granted);
  if (st != KSMM_OK) return st;
  norm_columns_kernel<T><<<static_cast<unsigned>(chunks * A.samples), kColWarps * 32, smem, stream>>>(A);
  return launched("norm");
}

// Batch-last tensors of more channels than a block keeps: transposed copies, the kernels for rows, transposes back.
// (4 x 305 tokens of 6950 channels fp32: 229 us by columns that were read again for every statistic, 179 so.)
bool turned(const ksmm_norm_desc_t& d) { return d.bs_last && d.channels > kColumnChannels; }

size_t tensor_bytes(const ksmm_norm_desc_t& d) {
  return (static_cast<size_t>(d.rows) * d.channels * dtype_size(d.dtype) + 255) / 256 * 256;
}

// copies of up to four inputs and two outputs
size_t turned_bytes(const ksmm_norm_desc_t& d, bool backward) {
  if (!turned(d)) return 0;
  int n = backward ? (d.grad_h ? 2 : 0) + (d.grad_z ? 1 : 0) + (d.y ? 1 : 0) + (d.grad_x ? 1 : 0) + (d.grad_y ? 1 : 0)
                   : 1 + (d.y ? 2 : 0) + (d.norm != kNone ? 1 : 0);
  return n * tensor_bytes(d);
}

// `t` with its tensors replaced by transposed copies in `ws`; outputs to turn back in out[]
struct Turn {
  ksmm_norm_desc_t t;
  struct { const void* from; void* to; } out[2];
  int outs = 0;
};

int turn_in(const ksmm_norm_desc_t& d, bool backward, char* ws, cudaStream_t stream, Turn* r) {
  r->t = d;
  r->t.bs_last = 0;
  const int es = dtype_size(d.dtype);
  auto take = [&]() {
    char* p = ws;
    ws += tensor_bytes(d);
    return p;
  };
  auto in = [&](const void* src, int* st) -> void* {
    if (!src || *st != KSMM_OK) return nullptr;
    void* p = take();
    *st = launch_transpose(src, p, d.channels, d.rows, es, stream);
    return p;
  };
  auto out = [&](void* dst) -> void* {
    if (!dst) return nullptr;
    void* p = take();
    r->out[r->outs++] = {p, dst};
    return p;
  };
  int st = KSMM_OK;
  if (!backward) {
    r->t.x = in(d.x, &st);
    r->t.y = in(d.y, &st);
    r->t.z = out(d.y ? d.z : nullptr);
    r->t.h = out(d.norm != kNone ? d.h : nullptr);
    return st;
  }
  if (d.grad_h) {  // the value that pre normalised, or x to form it from
    void* z = in(d.y && !remakes_z(d) ? d.z : d.x, &st);
    if (d.y && !remakes_z(d)) r->t.z = z;
    else r->t.x = z;
    r->t.grad_h = in(d.grad_h, &st);
  }
  r->t.grad_z = in(d.grad_z, &st);
  r->t.y = in(d.y, &st);
  r->t.grad_x = out(d.grad_x);
  r->t.grad_y = out(d.grad_y);
  return st;
}

int turn_out(const ksmm_norm_desc_t& d, const Turn& r, cudaStream_t stream) {
  for (int q = 0; q < r.outs; ++q) {
    const int st = launch_transpose(r.out[q].from, r.out[q].to, d.rows, d.channels, dtype_size(d.dtype), stream);
    if (st != KSMM_OK) return st;
  }
  return KSMM_OK;
}

int forward_any(const ksmm_norm_desc_t& d, cudaStream_t s) {
  if (d.dtype == KSMM_F32) return forward_typed<float>(d, s);
  if (d.dtype == KSMM_F16) return forward_typed<__half>(d, s);
  return forward_typed<__nv_bfloat16>(d, s);
}

// Tokens of a sample are cut into runs, one block each: 32 columns, or as many runs of rows as blocks fit the SMs
// at once (168 registers a thread up to 128 threads, 128 beyond).
int64_t chunks_of(const ksmm_norm_desc_t& d) {
  const int64_t per = d.samples > 0 ? d.rows / d.samples : 0;
  if (per <= 0) return 1;
  if (d.bs_last && !turned(d)) return (per + 31) / 32;
  const int64_t pieces = (d.channels * dtype_size(d.dtype) + 15) / 16, threads = std::min<int64_t>(512, (pieces + 31) / 32 * 32);
  const int64_t blocks = std::min<int64_t>(8, 65536 / ((threads <= 128 ? 168 : 128) * threads));
  const int64_t want = std::max<int64_t>(1, 148 * blocks / d.samples);
  // (eight rows or more share a block's sums where there are rows enough; 64 rows of 6464 fp32 channels: 56 us with
  // eight blocks, 17 with 64)
  const int64_t least = std::max<int64_t>(1, std::min<int64_t>(8, d.rows / 148));
  return std::max<int64_t>(1, std::min(want, (per + least - 1) / least));
}

bool wants_sums(const ksmm_norm_desc_t& d) {
  return d.grad_weight || d.grad_bias || d.grad_post_weight || d.grad_post_bias || d.grad_scale || d.grad_shift || d.grad_gate;
}

template <typename T>
int backward_typed(const ksmm_norm_desc_t& d, void* workspace, cudaStream_t stream) {
  Args A = args_of(d);
  const int64_t chunks = chunks_of(d);
  if (chunks * d.samples > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "norm: too many tokens");
  A.chunks = static_cast<int>(chunks);
  const bool sums = wants_sums(d);
  A.part = sums ? static_cast<float*>(workspace) : nullptr;
  int st;
  if (d.bs_last) {
    constexpr size_t per_channel = sizeof(float4) + 32 * sizeof(float);
    const size_t smem = A.C * per_channel;
    static Granted granted;
    st = allow_smem(reinterpret_cast<const void*>(norm_columns_backward_kernel<T>), smem, kColumnChannels * per_channel, granted);
    if (st != KSMM_OK) return st;
    norm_columns_backward_kernel<T><<<static_cast<unsigned>(chunks * d.samples), kColWarps * 32, smem, stream>>>(A);
    st = launched("norm backward");
  } else {
    st = vector_rows(d) ? launch_rows_backward<T, 16 / sizeof(T)>(A, stream) : launch_rows_backward<T, 1>(A, stream);
  }
  if (st != KSMM_OK || !sums) return st;
  const Grads g = {d.grad_weight, d.grad_bias, d.grad_post_weight, d.grad_post_bias, d.grad_scale, d.grad_shift, d.grad_gate,
                   d.scale_stride != 0, d.shift_stride != 0, d.gate_stride != 0};
  const bool totals = d.grad_weight || d.grad_bias || d.grad_post_weight || d.grad_post_bias ||
                      (d.grad_scale && !g.scale_rows) || (d.grad_shift && !g.shift_rows) || (d.grad_gate && !g.gate_rows);
  float* per_sample = A.part + chunks * d.samples * 4 * A.C;
  const unsigned cx = static_cast<unsigned>((A.C + 31) / 32);
  for (int64_t s0 = 0; s0 < d.samples; s0 += 65535) {  // (grid.y)
    Args B = A;
    const unsigned ns = static_cast<unsigned>(std::min<int64_t>(65535, d.samples - s0));
    Grads gs = g;
    const int ps = dtype_size(d.param_dtype);
    auto skip = [&](void* p, int rows) { return p && rows ? static_cast<char*>(p) + s0 * A.C * ps : static_cast<char*>(p); };
    gs.scale = skip(g.scale, g.scale_rows); gs.shift = skip(g.shift, g.shift_rows); gs.gate = skip(g.gate, g.gate_rows);
    auto row = [&](Row r) { return Row{r.p ? static_cast<const char*>(r.p) + s0 * r.ld * ps : nullptr, r.ld}; };
    B.scale = row(A.scale); B.shift = row(A.shift); B.gate = row(A.gate);
    norm_param_grads_kernel<T><<<dim3(cx, ns), 32 * slices_of(chunks), 0, stream>>>(B, gs, A.part + s0 * chunks * 4 * A.C,
                                                                  totals ? per_sample + s0 * 4 * A.C : nullptr, 1);
    if ((st = launched("norm gradients")) != KSMM_OK) return st;
  }
  if (d.samples > 1 && totals) {
    norm_param_grads_kernel<T><<<cx, 32 * slices_of(d.samples), 0, stream>>>(A, g, per_sample, nullptr, 0);
    st = launched("norm gradients");
  }
  return st;
}

int check_norm(const ksmm_norm_desc_t* d) {
  if (!d) return set_error(KSMM_ERR_BAD_ARGUMENT, "null descriptor");
  if (d->dtype != KSMM_F32 && d->dtype != KSMM_F16 && d->dtype != KSMM_BF16)
    return set_error(d->dtype == KSMM_F8E4M3 ? KSMM_ERR_UNSUPPORTED : KSMM_ERR_BAD_ARGUMENT,
                     "norms run in fp32, fp16 or bf16, not type %d", d->dtype);
  if (d->param_dtype != d->dtype && d->param_dtype != KSMM_F32)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "parameters have the tensors' type or fp32");
  if (d->norm < kNone || d->norm > kRms || d->post_norm < kNone || d->post_norm > kRms)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "unknown norm %d / %d", d->norm, d->post_norm);
  if (d->bs_last != 0 && d->bs_last != 1) return set_error(KSMM_ERR_BAD_ARGUMENT, "bs_last must be 0 or 1");
  if (d->rows < 0 || d->channels <= 0 || d->samples <= 0 || (d->rows % d->samples) != 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "%lld tokens of %d channels in %lld samples", static_cast<long long>(d->rows),
                     d->channels, static_cast<long long>(d->samples));
  if (d->channels > kMaxChannels)
    return set_error(KSMM_ERR_UNSUPPORTED, "norms take up to %d channels, not %d", kMaxChannels, d->channels);
  if (d->norm == kNone && !d->y) return set_error(KSMM_ERR_BAD_ARGUMENT, "neither a norm nor a second tensor");
  if (d->post_norm != kNone && !d->y) return set_error(KSMM_ERR_BAD_ARGUMENT, "a norm of y without y");
  if (d->post_norm == kNone && (d->post_weight || d->post_bias || d->grad_post_weight || d->grad_post_bias))
    return set_error(KSMM_ERR_BAD_ARGUMENT, "post_weight and post_bias belong to a post_norm");
  if (d->scale_stride < 0 || d->shift_stride < 0 || d->gate_stride < 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "negative stride");
  if (!(d->eps >= 0.f)) return set_error(KSMM_ERR_BAD_ARGUMENT, "eps must not be negative");
  return KSMM_OK;
}

size_t sums_bytes(const ksmm_norm_desc_t& d) {
  if (!wants_sums(d)) return 0;
  return (static_cast<size_t>(chunks_of(d) + 1) * d.samples * 4 * d.channels * sizeof(float) + 255) / 256 * 256;
}

int backward_any(const ksmm_norm_desc_t& d, void* workspace, cudaStream_t s) {
  if (d.dtype == KSMM_F32) return backward_typed<float>(d, workspace, s);
  if (d.dtype == KSMM_F16) return backward_typed<__half>(d, workspace, s);
  return backward_typed<__nv_bfloat16>(d, workspace, s);
}

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return set_error(KSMM_ERR_WORKSPACE, "norm: need %zu bytes of workspace aligned to 16, got %zu", need, bytes);
  return KSMM_OK;
}

}  // namespace
}  // namespace ksmm

using namespace ksmm;

extern "C" {

size_t ksmm_cu_norm_forward_workspace_bytes(const ksmm_norm_desc_t* d) {
  return check_norm(d) != KSMM_OK || d->rows == 0 ? 0 : turned_bytes(*d, false);
}

int ksmm_cu_norm_forward(const ksmm_norm_desc_t* d, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_norm(d);
  if (st != KSMM_OK || d->rows == 0) return st;
  if (!d->x || (d->y && !d->z) || (d->norm != kNone && !d->h)) return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  if (d->stats && reinterpret_cast<uintptr_t>(d->stats) % 16 != 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "the statistics are aligned to 16 bytes");
  if ((st = check_workspace(workspace, workspace_bytes, turned_bytes(*d, false))) != KSMM_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!turned(*d)) return forward_any(*d, s);
  Turn r;
  st = turn_in(*d, false, static_cast<char*>(workspace), s, &r);
  if (st == KSMM_OK) st = forward_any(r.t, s);
  return st == KSMM_OK ? turn_out(*d, r, s) : st;
}

size_t ksmm_cu_norm_backward_workspace_bytes(const ksmm_norm_desc_t* d) {
  if (check_norm(d) != KSMM_OK || d->rows == 0) return 0;
  return sums_bytes(*d) + turned_bytes(*d, true);
}

int ksmm_cu_norm_backward(const ksmm_norm_desc_t* d, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_norm(d);
  if (st != KSMM_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->rows == 0) {
    // sums over nothing
    const size_t row = static_cast<size_t>(d->channels) * dtype_size(d->param_dtype);
    const struct { void* p; int64_t rows; } all[7] = {
        {d->grad_weight, 1}, {d->grad_bias, 1}, {d->grad_post_weight, 1}, {d->grad_post_bias, 1},
        {d->grad_scale, d->scale_stride ? d->samples : 1}, {d->grad_shift, d->shift_stride ? d->samples : 1},
        {d->grad_gate, d->gate_stride ? d->samples : 1}};
    for (const auto& q : all) {
      if (!q.p) continue;
      const cudaError_t e = cudaMemsetAsync(q.p, 0, row * q.rows, s);
      if (e != cudaSuccess) return set_error(KSMM_ERR_CUDA, "memset failed: %s", cudaGetErrorString(e));
    }
    return KSMM_OK;
  }
  if (!d->stats || (d->norm != kNone && d->grad_h && !(d->y && !remakes_z(*d) ? d->z : d->x)) || (!d->grad_z && !d->grad_h))
    return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  if (d->grad_h && d->norm == kNone) return set_error(KSMM_ERR_BAD_ARGUMENT, "a gradient of h without a norm");
  if (d->grad_z && !d->y) return set_error(KSMM_ERR_BAD_ARGUMENT, "a gradient of z without y");
  if (reinterpret_cast<uintptr_t>(d->stats) % 16 != 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "the statistics are aligned to 16 bytes");
  if ((st = check_workspace(workspace, workspace_bytes, sums_bytes(*d) + turned_bytes(*d, true))) != KSMM_OK) return st;
  if (!turned(*d)) return backward_any(*d, workspace, s);
  Turn r;
  st = turn_in(*d, true, static_cast<char*>(workspace) + sums_bytes(*d), s, &r);
  if (st == KSMM_OK) st = backward_any(r.t, workspace, s);
  return st == KSMM_OK ? turn_out(*d, r, s) : st;
}

}  // extern "C"
