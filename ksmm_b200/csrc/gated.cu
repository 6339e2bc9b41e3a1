// The product of a gated layer, h = act(g) * u, and its backward, dg = dh u act'(g) and du = dh act(g), as passes
// over whole tensors: for types and shapes whose last factor does not form the product in its epilogue, and
// for every backward pass.  Memory is what bounds them: three tensors move forward, five backward.
// Arithmetic is fp32.  dg and du are rounded to the layer's type, once, as the gradient of any intermediate is: the
// multiplications that read them take no other.  (16-bit training, 12544 rows 768 -> 2048 bf16: every gradient within 0.0039 of
// the definition's in the 2-norm, one rounding is 0.0017.)
#include <algorithm>
#include <type_traits>

#include "gated.cuh"
#include "gated.h"

namespace ksmm {
namespace {

template <typename T, int V>
__device__ __forceinline__ void get(const T* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = ElemTraits<T>::to_float(*p);
  } else {
    __align__(16) T t[V];
    *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = ElemTraits<T>::to_float(t[e]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const float (&f)[V]) {
  __align__(16) T t[V];
#pragma unroll
  for (int e = 0; e < V; ++e) t[e] = ElemTraits<T>::from_float(f[e]);
  if constexpr (V == 1) *p = t[0];
  else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
}

// `pieces` pieces of V elements per line; `half`: elements between g and u, `out_half`: between dg and du
template <typename T, int V, bool BACKWARD>
__global__ void __launch_bounds__(256)
    gate_kernel(const T* __restrict__ gu, int64_t ld, const T* __restrict__ dh, int64_t h_ld, T* __restrict__ out,
                int64_t half, int64_t out_half, int64_t lines, uint32_t pieces, int act) {
  const int64_t total = lines * pieces;
#pragma unroll 1
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total; t += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t line = total <= 0xffffffffLL ? static_cast<uint32_t>(t) / pieces : t / pieces;
    const int64_t x = (t - line * pieces) * V;
    const T* at = gu + line * ld + x;
    float g[V], u[V];
    get<T, V>(at, g);
    get<T, V>(at + half, u);
    if constexpr (BACKWARD) {
      float d[V], a[V], b[V];
      get<T, V>(dh + line * h_ld + x, d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float value, slope;
        gate_slope<sizeof(T) == 2>(g[e], act, value, slope);
        a[e] = d[e] * u[e] * slope;
        b[e] = d[e] * value;
      }
      put<T, V>(out + line * ld + x, a);
      put<T, V>(out + out_half + line * ld + x, b);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = gate_value<sizeof(T) == 2>(g[e], act) * u[e];
      put<T, V>(out + line * h_ld + x, g);
    }
  }
}

// The product in the other layout, out[x, y] = h[y, x], by tiles of 64 x 64: 4096 rows of 2816 fp32 features (138 MB,
// 21 us at the copy's rate) take 23 us, the product and a transpose after it 34.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    gate_turn_kernel(const T* __restrict__ gu, int64_t ld, T* __restrict__ out, int64_t half, int64_t lines, int64_t len,
                     uint32_t tiles_x, int act) {
  __shared__ float tile[64][65];
  constexpr int P = 64 / V, AHEAD = V > 1 ? 4 : 1;
  const int64_t y0 = static_cast<int64_t>(blockIdx.x / tiles_x) * 64, x0 = static_cast<int64_t>(blockIdx.x % tiles_x) * 64;
#pragma unroll AHEAD
  for (int s = threadIdx.x; s < 64 * P; s += 256) {
    const int y = s / P, x = s % P * V;
    if (y0 + y >= lines || x0 + x >= len) continue;
    const T* at = gu + (y0 + y) * ld + x0 + x;  // (the last piece of a padded line may reach into its padding)
    float g[V], u[V];
    get<T, V>(at, g);
    get<T, V>(at + half, u);
#pragma unroll
    for (int e = 0; e < V; ++e) tile[x + e][y] = gate_value<sizeof(T) == 2>(g[e], act) * u[e];
  }
  __syncthreads();
#pragma unroll AHEAD
  for (int s = threadIdx.x; s < 64 * P; s += 256) {
    const int x = s / P, y = s % P * V;
    if (x0 + x >= len || y0 + y >= lines) continue;
    float h[V];
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = tile[x][y + e];
    put<T, V>(out + (x0 + x) * lines + y0 + y, h);
  }
}

template <typename T>
int gate_turn_typed(const void* gu, int64_t ld, void* out, int64_t lines, int64_t len, int act, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int64_t half = lines * ld, tiles_x = (len + 63) / 64, blocks = (lines + 63) / 64 * tiles_x;
  if (blocks > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "gated layer: too many elements");
  const bool vec = reinterpret_cast<uintptr_t>(gu) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 && ld % V == 0 &&
                   half % V == 0 && lines % V == 0;
  auto go = [&](auto kern) {
    kern<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<const T*>(gu), ld, static_cast<T*>(out), half, lines, len,
                                                            static_cast<uint32_t>(tiles_x), act);
  };
  if (vec) go(gate_turn_kernel<T, V>);
  else go(gate_turn_kernel<T, 1>);
  count_launch();
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "gate kernel launch failed: %s", cudaGetErrorString(err));
  return KSMM_OK;
}

// The backward with the sums of its lines (features of a batch-last tensor), which are the gradients of the biases:
// a block per line.  Against a pass of its own over dg and du, 2 x 2048 x 12544 bf16: 21 us saved.
template <typename T, int V>
__global__ void __launch_bounds__(256, 6)
    gate_lines_kernel(const T* __restrict__ gu, int64_t ld, const T* __restrict__ dh, int64_t h_ld, T* __restrict__ out,
                      int64_t half, int64_t out_half, int64_t len, int act, T* __restrict__ bias_grad) {
  using Sum = typename std::conditional<sizeof(T) == 4, double, float>::type;  // (a thread's share of a long line)
  const int64_t line = blockIdx.x;
  const T* at = gu + line * ld;
  const T* dp = dh + line * h_ld;
  T* op = out + line * ld;
  Sum sg = 0, su = 0;
  for (int64_t x = threadIdx.x * V; x < len; x += 256 * V) {
    float g[V], u[V], d[V], a[V], b[V];
    get<T, V>(at + x, g);
    get<T, V>(at + half + x, u);
    get<T, V>(dp + x, d);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float value, slope;
      gate_slope<sizeof(T) == 2>(g[e], act, value, slope);
      a[e] = d[e] * u[e] * slope;
      b[e] = d[e] * value;
      s1 += a[e];
      s2 += b[e];
    }
    put<T, V>(op + x, a);
    put<T, V>(op + out_half + x, b);
    sg += s1;
    su += s2;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sg += __shfl_xor_sync(0xffffffffu, sg, o);
    su += __shfl_xor_sync(0xffffffffu, su, o);
  }
  __shared__ Sum part[2][8];
  if ((threadIdx.x & 31) == 0) {
    part[0][threadIdx.x >> 5] = sg;
    part[1][threadIdx.x >> 5] = su;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    Sum t = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += part[threadIdx.x][w];
    bias_grad[threadIdx.x * gridDim.x + line] = ElemTraits<T>::from_float(static_cast<float>(t));
  }
}

template <typename T>
int gate_lines_typed(const void* gu, int64_t ld, const void* dh, int64_t dh_ld, void* out, int64_t out_half, int64_t lines,
                     int64_t len, int act, void* bias_grad, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (lines > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "gated layer: too many features");
  const int64_t half = lines * ld;
  const bool vec = reinterpret_cast<uintptr_t>(gu) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(dh) % 16 == 0 && ld % V == 0 && dh_ld % V == 0 && len % V == 0 && out_half % V == 0;
  auto go = [&](auto kern) {
    kern<<<static_cast<unsigned>(lines), 256, 0, stream>>>(static_cast<const T*>(gu), ld, static_cast<const T*>(dh), dh_ld,
                                                           static_cast<T*>(out), half, out_half, len, act, static_cast<T*>(bias_grad));
  };
  if (vec) go(gate_lines_kernel<T, V>);
  else go(gate_lines_kernel<T, 1>);
  count_launch();
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "gate kernel launch failed: %s", cudaGetErrorString(err));
  return KSMM_OK;
}

template <typename T, bool BACKWARD>
int gate_typed(const void* gu, int64_t ld, const void* dh, int64_t h_ld, void* out, int64_t out_half, int64_t lines, int64_t len,
               int act, cudaStream_t stream) {
  if (lines <= 0 || len <= 0) return KSMM_OK;
  constexpr int V = 16 / sizeof(T);
  const int64_t half = lines * ld;
  const void* narrow = BACKWARD ? dh : out;
  const bool aligned = reinterpret_cast<uintptr_t>(gu) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(narrow) % 16 == 0 && half % V == 0 && out_half % V == 0;
  if (ld == len && h_ld == len) {  // lines that follow one another are one line
    len *= lines;
    ld = h_ld = len;
    lines = 1;
  }
  const bool vec = aligned && len % V == 0 && (lines == 1 || (ld % V == 0 && h_ld % V == 0));
  const int64_t pieces = vec ? len / V : len;
  if (pieces > 0xffffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "gated layer: too many elements");
  const int64_t blocks = std::min<int64_t>((lines * pieces + 255) / 256, 148 * 64);
  auto go = [&](auto kern) {
    kern<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<const T*>(gu), ld, static_cast<const T*>(dh), h_ld,
                                                             static_cast<T*>(out), half, out_half, lines, static_cast<uint32_t>(pieces), act);
  };
  if (vec) go(gate_kernel<T, V, BACKWARD>);
  else go(gate_kernel<T, 1, BACKWARD>);
  count_launch();
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "gate kernel launch failed: %s", cudaGetErrorString(err));
  return KSMM_OK;
}

}  // namespace

int launch_gate(const void* gu, int64_t ld, void* h, int64_t h_ld, int64_t lines, int64_t len, int dtype, int act,
                cudaStream_t stream) {
  if (dtype == KSMM_F32) return gate_typed<float, false>(gu, ld, nullptr, h_ld, h, 0, lines, len, act, stream);
  if (dtype == KSMM_F16) return gate_typed<__half, false>(gu, ld, nullptr, h_ld, h, 0, lines, len, act, stream);
  return gate_typed<__nv_bfloat16, false>(gu, ld, nullptr, h_ld, h, 0, lines, len, act, stream);
}

int launch_gate_turn(const void* gu, int64_t ld, void* h, int64_t lines, int64_t len, int dtype, int act, cudaStream_t stream) {
  if (dtype == KSMM_F32) return gate_turn_typed<float>(gu, ld, h, lines, len, act, stream);
  if (dtype == KSMM_F16) return gate_turn_typed<__half>(gu, ld, h, lines, len, act, stream);
  return gate_turn_typed<__nv_bfloat16>(gu, ld, h, lines, len, act, stream);
}

int launch_gate_backward(const void* gu, int64_t ld, const void* dh, int64_t dh_ld, void* out, int64_t out_half, int64_t lines,
                         int64_t len, int dtype, int act, void* bias_grad, cudaStream_t stream) {
  if (bias_grad) {
    if (dtype == KSMM_F32) return gate_lines_typed<float>(gu, ld, dh, dh_ld, out, out_half, lines, len, act, bias_grad, stream);
    if (dtype == KSMM_F16) return gate_lines_typed<__half>(gu, ld, dh, dh_ld, out, out_half, lines, len, act, bias_grad, stream);
    return gate_lines_typed<__nv_bfloat16>(gu, ld, dh, dh_ld, out, out_half, lines, len, act, bias_grad, stream);
  }
  if (dtype == KSMM_F32) return gate_typed<float, true>(gu, ld, dh, dh_ld, out, out_half, lines, len, act, stream);
  if (dtype == KSMM_F16) return gate_typed<__half, true>(gu, ld, dh, dh_ld, out, out_half, lines, len, act, stream);
  return gate_typed<__nv_bfloat16, true>(gu, ld, dh, dh_ld, out, out_half, lines, len, act, stream);
}

}  // namespace ksmm
