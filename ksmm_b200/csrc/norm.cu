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
// h is made from stay in fp32; z and h are rounded once.  The backward pass reads the rounded z and the
// statistics of the unrounded one (16 bytes per token).  Sums over tokens are formed in a fixed order: a
// CTA sums its own run of tokens, two small kernels add the runs up; no atomics.
//
// The stock form in the reference's models is a chain of separate PyTorch calls: LayerNorm and the sum around
// attention and feed-forward block (src/ksmm_py/model/vit.py:416-431, 770-800).
#include <algorithm>

#include "common.cuh"

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
  int C, pre, post, p32, pvec;  // p32: parameters are fp32; pvec: they can be read in pieces of V
  float alpha, eps;
};

template <typename T>
__device__ __forceinline__ float bits_to_float(uint16_t b) {
  if constexpr (sizeof(T) == 2 && ElemTraits<T>::kDtype == KSMM_BF16) return __uint_as_float(static_cast<uint32_t>(b) << 16);
  else return __half2float(__ushort_as_half(b));
}

// V consecutive elements (16 bytes, or one element)
template <typename T, int V>
struct Raw {
  static_assert(V == 1 || V * sizeof(T) == 16, "a 16-byte piece or an element");
  uint4 v;
  T one;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) one = *p;
    else v = __ldg(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void zero() {
    if constexpr (V == 1) one = ElemTraits<T>::from_float(0.f);
    else v = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (V == 1) {
      return ElemTraits<T>::to_float(one);
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
      else return bits_to_float<T>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ void store_piece(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    *p = ElemTraits<T>::from_float(f[0]);
  } else {
    __align__(16) T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = ElemTraits<T>::from_float(f[e]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
  }
}

// V parameters from channel c of a sample's row; `other` where there is no such parameter
template <typename T, int V>
__device__ __forceinline__ void load_param(const Args& A, const Row& r, int64_t sample, int c, float other, float (&f)[V]) {
  if (r.p == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = other;
    return;
  }
  const int64_t at = sample * r.ld + c;
  if (A.p32) {
    const float* p = static_cast<const float*>(r.p) + at;
    if (V >= 4 && A.pvec) {
#pragma unroll
      for (int e = 0; e + 3 < V; e += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + e));
        f[e] = q.x; f[e + 1] = q.y; f[e + 2] = q.z; f[e + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = __ldg(p + e);
    }
  } else {
    const T* p = static_cast<const T*>(r.p) + at;
    if (V > 1 && A.pvec) {
      Raw<T, V> q;
      q.load(p);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = q.at(e);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = ElemTraits<T>::to_float(p[e]);
    }
  }
}
template <typename T>
__device__ __forceinline__ float param_at(const Args& A, const Row& r, int64_t sample, int c, float other) {
  float f[1];
  load_param<T, 1>(A, r, sample, c, other, f);
  return f[0];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// the sums of N values over all threads of the block; `red` holds 32 * N floats and is free again after it
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* red) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < N; ++q) v[q] = warp_sum(v[q]);
  if (warps == 1) return;
  if (lane == 0) {
#pragma unroll
    for (int q = 0; q < N; ++q) red[warp * N + q] = v[q];
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < N; ++q) v[q] = warp_sum(lane < warps ? red[lane * N + q] : 0.f);
  __syncthreads();
}

// ---------------------------------------------------------------------------
// batch-first: a token is a row
// ---------------------------------------------------------------------------
// TPR threads hold a row in registers, K pieces each: a warp per row up to 1024 channels (no barrier),
// a block per row beyond.
template <typename T, int V, int K, int TPR>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_rows_kernel(const Args A) {
  constexpr int kBlock = TPR < 128 ? 128 : TPR;
  __shared__ float red[32];
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / TPR) + threadIdx.x / TPR;
  if (row >= A.rows) return;  // (whole warps, or the whole block)
  auto sum = [&](float v) {
    if constexpr (TPR == 32) {
      return warp_sum(v);
    } else {
      float q[1] = {v};
      block_sum<1>(q, red);
      return q[0];
    }
  };
  const int64_t sample = A.samples == 1 ? 0 : row / A.per_sample;
  const T* x = static_cast<const T*>(A.x) + row * A.C;
  const float inv = 1.f / static_cast<float>(A.C);
  float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
  Raw<T, V> xr[K], yr[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (t + k * TPR) * V;
    if (c < A.C) xr[k].load(x + c);
    else xr[k].zero();
  }
  if (A.y) {
    const T* y = static_cast<const T*>(A.y) + row * A.C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (t + k * TPR) * V;
      if (c < A.C) yr[k].load(y + c);
      else yr[k].zero();
    }
    if (A.post != kNone) {
      float s = 0.f;
      if (A.post == kLayer) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) s += yr[k].at(e);
        st.z = sum(s) * inv;
      }
      s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if ((t + k * TPR) * V >= A.C) break;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = yr[k].at(e) - st.z;
          s = fmaf(d, d, s);
        }
      }
      st.w = rsqrtf(sum(s) * inv + A.eps);
    }
  }
  float z[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (t + k * TPR) * V;
    if (A.y == nullptr) {
#pragma unroll
      for (int e = 0; e < V; ++e) z[k][e] = xr[k].at(e);
    } else if (c < A.C) {
      float g[V], p[V];
#pragma unroll
      for (int e = 0; e < V; ++e) p[e] = yr[k].at(e);
      if (A.post != kNone) {
        float w[V], b[V];
        load_param<T, V>(A, A.post_weight, 0, c, 1.f, w);
        load_param<T, V>(A, A.post_bias, 0, c, 0.f, b);
#pragma unroll
        for (int e = 0; e < V; ++e) p[e] = fmaf((p[e] - st.z) * st.w, w[e], b[e]);
      }
      load_param<T, V>(A, A.gate, sample, c, 1.f, g);
#pragma unroll
      for (int e = 0; e < V; ++e) z[k][e] = fmaf(A.alpha, xr[k].at(e), g[e] * p[e]);
      store_piece<T, V>(static_cast<T*>(A.z) + row * A.C + c, z[k]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) z[k][e] = 0.f;
    }
  }
  if (A.pre != kNone) {
    float s = 0.f;
    if (A.pre == kLayer) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) s += z[k][e];
      st.x = sum(s) * inv;
    }
    s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((t + k * TPR) * V >= A.C) break;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = z[k][e] - st.x;
        s = fmaf(d, d, s);
      }
    }
    st.y = rsqrtf(sum(s) * inv + A.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (t + k * TPR) * V;
      if (c >= A.C) break;
      float w[V], b[V], o[V];
      load_param<T, V>(A, A.weight, 0, c, 1.f, w);
      load_param<T, V>(A, A.bias, 0, c, 0.f, b);
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf((z[k][e] - st.x) * st.y, w[e], b[e]);
      if (A.scale.p || A.shift.p) {
        load_param<T, V>(A, A.scale, sample, c, 0.f, w);
        load_param<T, V>(A, A.shift, sample, c, 0.f, b);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(o[e], 1.f + w[e], b[e]);
      }
      store_piece<T, V>(static_cast<T*>(A.h) + row * A.C + c, o);
    }
  }
  if (A.stats && t == 0) A.stats[row] = st;
}

// A block walks a run of one sample's rows, R at a time; a thread keeps its channels, so that the sums over
// rows stay in its registers.
template <typename T, int V, int K, int R>
__global__ void __launch_bounds__(512) norm_rows_backward_kernel(const Args A) {
  __shared__ float red[32 * 2 * R];
  const int t = threadIdx.x, nt = blockDim.x;
  const int64_t sample = blockIdx.x / A.chunks;
  const int chunk = static_cast<int>(blockIdx.x % A.chunks);
  const int64_t begin = sample * A.per_sample + A.per_sample * chunk / A.chunks;
  const int64_t end = sample * A.per_sample + A.per_sample * (chunk + 1) / A.chunks;
  const float inv = 1.f / static_cast<float>(A.C);
  const T* zp = static_cast<const T*>(A.z_in);
  const T* yp = static_cast<const T*>(A.y);
  const T* gzp = static_cast<const T*>(A.gz);
  const T* ghp = static_cast<const T*>(A.gh);
  float wp[K][V], wq[K][V];  // weight (1 + scale), gate * post_weight
  float sa[K][V], sb[K][V], sc[K][V], sd[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (t + k * nt) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) wp[k][e] = wq[k][e] = sa[k][e] = sb[k][e] = sc[k][e] = sd[k][e] = 0.f;
    if (c < A.C) {
      float q[V];
      load_param<T, V>(A, A.weight, 0, c, 1.f, wp[k]);
      load_param<T, V>(A, A.scale, sample, c, 0.f, q);
#pragma unroll
      for (int e = 0; e < V; ++e) wp[k][e] *= 1.f + q[e];
      load_param<T, V>(A, A.gate, sample, c, 1.f, wq[k]);
      if (A.post != kNone) {
        load_param<T, V>(A, A.post_weight, 0, c, 1.f, q);
#pragma unroll
        for (int e = 0; e < V; ++e) wq[k][e] *= q[e];
      }
    }
  }
  for (int64_t row0 = begin; row0 < end; row0 += R) {
    Raw<T, V> zr[R][K], yr[R][K], gz[R][K], gh[R][K];
    float4 st[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r;
      st[r] = row < end ? __ldg(A.stats + row) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (t + k * nt) * V;
        const bool live = row < end && c < A.C;
        const int64_t at = row * A.C + c;
        if (live && ghp) { gh[r][k].load(ghp + at); zr[r][k].load(zp + at); }
        else { gh[r][k].zero(); zr[r][k].zero(); }
        if (live && gzp) gz[r][k].load(gzp + at); else gz[r][k].zero();
        if (live && yp) yr[r][k].load(yp + at); else yr[r][k].zero();
      }
    }
    float G[R][K][V];
    if (ghp) {
      float s[2 * R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float g = gh[r][k].at(e), n = (zr[r][k].at(e) - st[r].x) * st[r].y;
            const float w = g * wp[k][e];
            s[2 * r] += w;
            s[2 * r + 1] = fmaf(w, n, s[2 * r + 1]);
            sa[k][e] += g;
            sb[k][e] = fmaf(g, n, sb[k][e]);
          }
      }
      block_sum<2 * R>(s, red);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m1 = A.pre == kLayer ? s[2 * r] * inv : 0.f, m2 = s[2 * r + 1] * inv;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float n = (zr[r][k].at(e) - st[r].x) * st[r].y;
            G[r][k][e] = fmaf(st[r].y, gh[r][k].at(e) * wp[k][e] - m1 - n * m2, gz[r][k].at(e));
          }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) G[r][k][e] = gz[r][k].at(e);
    }
    if (A.gx) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (t + k * nt) * V;
          if (row0 + r >= end || c >= A.C) continue;
          float o[V];
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] = A.alpha * G[r][k][e];
          store_piece<T, V>(static_cast<T*>(A.gx) + (row0 + r) * A.C + c, o);
        }
    }
    if (yp) {
      float s[2 * R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[2 * r] = s[2 * r + 1] = 0.f;
        if (row0 + r >= end) continue;  // (rows of the next run must not join the sums)
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if ((t + k * nt) * V >= A.C) continue;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float m = (yr[r][k].at(e) - st[r].z) * st[r].w;
            const float f = G[r][k][e] * wq[k][e];
            s[2 * r] += f;
            s[2 * r + 1] = fmaf(f, m, s[2 * r + 1]);
            sc[k][e] += G[r][k][e];
            sd[k][e] = fmaf(G[r][k][e], m, sd[k][e]);
          }
        }
      }
      if (A.post != kNone) block_sum<2 * R>(s, red);
      if (A.gy) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float m1 = A.post == kLayer ? s[2 * r] * inv : 0.f, m2 = A.post != kNone ? s[2 * r + 1] * inv : 0.f;
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const int c = (t + k * nt) * V;
            if (row0 + r >= end || c >= A.C) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float m = (yr[r][k].at(e) - st[r].z) * st[r].w;
              o[e] = st[r].w * (G[r][k][e] * wq[k][e] - m1 - m * m2);
            }
            store_piece<T, V>(static_cast<T*>(A.gy) + (row0 + r) * A.C + c, o);
          }
        }
      }
    }
  }
  if (A.part) {
    float* part = A.part + static_cast<int64_t>(blockIdx.x) * 4 * A.C;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (t + k * nt) * V;
      if (c >= A.C) break;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        part[c + e] = sa[k][e];
        part[A.C + c + e] = sb[k][e];
        part[2 * A.C + c + e] = sc[k][e];
        part[3 * A.C + c + e] = sd[k][e];
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

template <typename T>
__global__ void __launch_bounds__(kColWarps * 32) norm_columns_kernel(const Args A) {
  __shared__ float red[kColWarps * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t sample = blockIdx.x / A.chunks;
  const int64_t in_sample = static_cast<int64_t>(blockIdx.x % A.chunks) * 32 + lane;
  const bool live = in_sample < A.per_sample;
  const int64_t tok = sample * A.per_sample + (live ? in_sample : 0);
  const T* x = static_cast<const T*>(A.x) + tok;
  const T* y = A.y ? static_cast<const T*>(A.y) + tok : nullptr;
  const float inv = 1.f / static_cast<float>(A.C);
  auto at = [&](const T* p, int c) { return ElemTraits<T>::to_float(p[c * A.rows]); };
  float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
  if (y && A.post != kNone) {
    float s = 0.f;
    if (A.post == kLayer) {
#pragma unroll 8
      for (int c = warp; c < A.C; c += kColWarps) s += at(y, c);
      st.z = column_sum(s, red) * inv;
      s = 0.f;
    }
#pragma unroll 8
    for (int c = warp; c < A.C; c += kColWarps) {
      const float d = at(y, c) - st.z;
      s = fmaf(d, d, s);
    }
    st.w = rsqrtf(column_sum(s, red) * inv + A.eps);
  }
  auto z_at = [&](int c) {
    const float xv = at(x, c);
    if (!y) return xv;
    float p = at(y, c);
    if (A.post != kNone)
      p = fmaf((p - st.z) * st.w, param_at<T>(A, A.post_weight, 0, c, 1.f), param_at<T>(A, A.post_bias, 0, c, 0.f));
    return fmaf(A.alpha, xv, param_at<T>(A, A.gate, sample, c, 1.f) * p);
  };
  if (A.pre != kNone) {
    float s = 0.f;
    if (A.pre == kLayer) {
#pragma unroll 8
      for (int c = warp; c < A.C; c += kColWarps) s += z_at(c);
      st.x = column_sum(s, red) * inv;
      s = 0.f;
    }
#pragma unroll 8
    for (int c = warp; c < A.C; c += kColWarps) {
      const float d = z_at(c) - st.x;
      s = fmaf(d, d, s);
    }
    st.y = rsqrtf(column_sum(s, red) * inv + A.eps);
  }
  if (live) {
#pragma unroll 4
    for (int c = warp; c < A.C; c += kColWarps) {
      const float z = z_at(c);
      if (y) static_cast<T*>(A.z)[c * A.rows + tok] = ElemTraits<T>::from_float(z);
      if (A.pre != kNone) {
        float o = fmaf((z - st.x) * st.y, param_at<T>(A, A.weight, 0, c, 1.f), param_at<T>(A, A.bias, 0, c, 0.f));
        o = fmaf(o, 1.f + param_at<T>(A, A.scale, sample, c, 0.f), param_at<T>(A, A.shift, sample, c, 0.f));
        static_cast<T*>(A.h)[c * A.rows + tok] = ElemTraits<T>::from_float(o);
      }
    }
    if (A.stats && warp == 0) A.stats[tok] = st;
  }
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

template <typename T>
__global__ void __launch_bounds__(kColWarps * 32) norm_columns_backward_kernel(const Args A) {
  __shared__ float red[kColWarps * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t sample = blockIdx.x / A.chunks;
  const int64_t in_sample = static_cast<int64_t>(blockIdx.x % A.chunks) * 32 + lane;
  const bool live = in_sample < A.per_sample;
  const int64_t tok = sample * A.per_sample + (live ? in_sample : 0);
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
      const float w = (live ? at(ghp, c) : 0.f) * param_at<T>(A, A.weight, 0, c, 1.f) * (1.f + param_at<T>(A, A.scale, sample, c, 0.f));
      s1 += w;
      s2 = fmaf(w, (at(zp, c) - st.x) * st.y, s2);
    }
    if (A.pre == kLayer) m1 = column_sum(s1, red) * inv;
    m2 = column_sum(s2, red) * inv;
  }
  auto G_at = [&](int c, float gh, float n) {
    float g = live && gzp ? at(gzp, c) : 0.f;
    if (ghp) {
      const float w = gh * param_at<T>(A, A.weight, 0, c, 1.f) * (1.f + param_at<T>(A, A.scale, sample, c, 0.f));
      g = fmaf(st.y, w - m1 - n * m2, g);
    }
    return live ? g : 0.f;
  };
  if (yp && A.post != kNone) {
    float s1 = 0.f, s2 = 0.f;
#pragma unroll 8
    for (int c = warp; c < A.C; c += kColWarps) {
      const float gh = live && ghp ? at(ghp, c) : 0.f, n = ghp ? (at(zp, c) - st.x) * st.y : 0.f;
      const float f = G_at(c, gh, n) * param_at<T>(A, A.gate, sample, c, 1.f) * param_at<T>(A, A.post_weight, 0, c, 1.f);
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
          n = (at(zp, c) - st.x) * st.y;
        }
        G = G_at(c, gh, n);
        if (live && A.gx) static_cast<T*>(A.gx)[c * A.rows + tok] = ElemTraits<T>::from_float(A.alpha * G);
        if (yp) {
          m = (at(yp, c) - st.z) * st.w;
          if (live && A.gy) {
            float f = G * param_at<T>(A, A.gate, sample, c, 1.f);
            if (A.post != kNone) f = f * param_at<T>(A, A.post_weight, 0, c, 1.f) - q1 - m * q2;
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

// 32 channels x 32 slices: first == 1 adds the chunks of sample blockIdx.y and writes the gradients of
// per-sample parameters and the sample's sums; first == 0 adds the samples.  With one sample the first does all.
template <typename T>
__global__ void __launch_bounds__(1024) norm_param_grads_kernel(const Args A, const Grads g, const float* part, float* sums,
                                                                int first) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const bool ok = c < A.C;
  const int64_t sample = blockIdx.y;
  // the totals that the last stage needs: A, B, C, D weighted for weight, bias, post_weight, post_bias, plus plain ones
  float t[7] = {};
  if (first) {
    const float* p = part + sample * A.chunks * 4 * A.C + c;
    if (ok)
      for (int q = slice; q < A.chunks; q += 32)
#pragma unroll
        for (int s = 0; s < 4; ++s) t[s] += p[(static_cast<int64_t>(q) * 4 + s) * A.C];
  } else if (ok) {
    const float pw = param_at<T>(A, A.post_weight, 0, c, 1.f), pb = param_at<T>(A, A.post_bias, 0, c, 0.f);
    const float w = param_at<T>(A, A.weight, 0, c, 1.f), b = param_at<T>(A, A.bias, 0, c, 0.f);
    for (int64_t s = slice; s < A.samples; s += 32) {
      const float* p = part + s * 4 * A.C + c;
      const float a = p[0], bb = p[A.C], cc = p[2 * A.C], d = p[3 * A.C];
      const float sc = 1.f + param_at<T>(A, A.scale, s, c, 0.f), ga = param_at<T>(A, A.gate, s, c, 1.f);
      t[0] = fmaf(sc, bb, t[0]);
      t[1] = fmaf(sc, a, t[1]);
      t[2] = fmaf(ga, d, t[2]);
      t[3] = fmaf(ga, cc, t[3]);
      t[4] += fmaf(w, bb, b * a);
      t[5] += a;
      t[6] += fmaf(pw, d, pb * cc);
    }
  }
#pragma unroll
  for (int s = 0; s < 7; ++s) {
    if (first && s >= 4) break;
    red[slice][lane] = t[s];
    __syncthreads();
    if (slice == 0) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < 32; ++q) v += red[q][lane];
      t[s] = v;
    }
    __syncthreads();
  }
  if (slice != 0 || !ok) return;
  if (first) {
    const float pw = param_at<T>(A, A.post_weight, 0, c, 1.f), pb = param_at<T>(A, A.post_bias, 0, c, 0.f);
    const float w = param_at<T>(A, A.weight, 0, c, 1.f), b = param_at<T>(A, A.bias, 0, c, 0.f);
    const float sc = 1.f + param_at<T>(A, A.scale, sample, c, 0.f), ga = param_at<T>(A, A.gate, sample, c, 1.f);
    const bool one = A.samples == 1;
    const int64_t at = sample * A.C + c;
    if (one || g.scale_rows) put<T>(A, g.scale, at, fmaf(w, t[1], b * t[0]));
    if (one || g.shift_rows) put<T>(A, g.shift, at, t[0]);
    if (one || g.gate_rows) put<T>(A, g.gate, at, fmaf(pw, t[3], pb * t[2]));
    if (one) {
      put<T>(A, g.weight, c, sc * t[1]);
      put<T>(A, g.bias, c, sc * t[0]);
      put<T>(A, g.post_weight, c, ga * t[3]);
      put<T>(A, g.post_bias, c, ga * t[2]);
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

// can tokens be read in 16-byte pieces?
bool vector_rows(const ksmm_norm_desc_t& d) {
  const int es = dtype_size(d.dtype);
  for (const void* p : {d.x, d.y, static_cast<const void*>(d.z), static_cast<const void*>(d.h), d.grad_z, d.grad_h,
                        static_cast<const void*>(d.grad_x), static_cast<const void*>(d.grad_y)})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return (static_cast<int64_t>(d.channels) * es) % 16 == 0;
}

Args args_of(const ksmm_norm_desc_t& d) {
  Args A = {};
  A.x = d.x; A.y = d.y; A.z = d.z; A.h = d.h;
  A.z_in = d.y ? d.z : d.x;
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
  const int ps = dtype_size(d.param_dtype);
  A.pvec = 1;
  for (const Row& r : {A.weight, A.bias, A.post_weight, A.post_bias, A.scale, A.shift, A.gate})
    A.pvec &= whole_pieces(r.p, r.ld, ps) ? 1 : 0;
  A.alpha = d.y ? d.alpha : 1.f;
  A.eps = d.eps;
  return A;
}

template <typename T, int V>
int launch_rows(const Args& A, cudaStream_t stream) {
  const int pieces = (A.C + V - 1) / V;
  auto go = [&](auto kern, int tpr) {
    const int block = tpr < 128 ? 128 : tpr;
    const int64_t grid = (A.rows + block / tpr - 1) / (block / tpr);
    if (grid > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "norm: too many rows");
    kern<<<static_cast<unsigned>(grid), block, 0, stream>>>(A);
    return launched("norm");
  };
  if constexpr (V > 1) {
    if (pieces <= 32) return go(norm_rows_kernel<T, V, 1, 32>, 32);
    if (pieces <= 64) return go(norm_rows_kernel<T, V, 2, 32>, 32);
    if (pieces <= 96) return go(norm_rows_kernel<T, V, 3, 32>, 32);
    if (pieces <= 128) return go(norm_rows_kernel<T, V, 4, 32>, 32);
    if (pieces <= 256) return go(norm_rows_kernel<T, V, 2, 128>, 128);
    if (pieces <= 512) return go(norm_rows_kernel<T, V, 4, 128>, 128);
    if constexpr (V == 4) {
      if (pieces > 1024) return go(norm_rows_kernel<T, V, 4, 512>, 512);
    }
    return go(norm_rows_kernel<T, V, 4, 256>, 256);
  } else {
    if (pieces <= 256) return go(norm_rows_kernel<T, 1, 8, 32>, 32);
    if (pieces <= 1024) return go(norm_rows_kernel<T, 1, 8, 128>, 128);
    return go(norm_rows_kernel<T, 1, 16, 512>, 512);
  }
}

template <typename T, int V>
int launch_rows_backward(const Args& A, cudaStream_t stream) {
  const int pieces = (A.C + V - 1) / V;
  const int64_t grid = A.samples * A.chunks;
  if (grid > 0x7fffffffLL) return set_error(KSMM_ERR_UNSUPPORTED, "norm: too many rows");
  const int k = (pieces + 511) / 512, per = (pieces + k - 1) / k, block = (per + 31) / 32 * 32;
  auto go = [&](auto kern, int kk) {
    const int n = kk == k ? block : ((pieces + kk - 1) / kk + 31) / 32 * 32;
    kern<<<static_cast<unsigned>(grid), n, 0, stream>>>(A);
    return launched("norm backward");
  };
  if constexpr (V > 1) {
    if (k <= 1) return go(norm_rows_backward_kernel<T, V, 1, 2>, 1);
    if constexpr (V == 4) {
      if (k > 2) return go(norm_rows_backward_kernel<T, V, 4, 1>, 4);
    }
    return go(norm_rows_backward_kernel<T, V, 2, 1>, 2);
  } else {
    if (k <= 1) return go(norm_rows_backward_kernel<T, 1, 1, 4>, 1);
    if (k <= 4) return go(norm_rows_backward_kernel<T, 1, 4, 2>, 4);
    return go(norm_rows_backward_kernel<T, 1, 16, 1>, 16);
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
  norm_columns_kernel<T><<<static_cast<unsigned>(chunks * A.samples), kColWarps * 32, 0, stream>>>(A);
  return launched("norm");
}

// Tokens of a sample are cut into runs, one block each: 32 columns, or enough runs of rows to give every SM
// several blocks.
int64_t chunks_of(const ksmm_norm_desc_t& d) {
  const int64_t per = d.samples > 0 ? d.rows / d.samples : 0;
  if (per <= 0) return 1;
  if (d.bs_last) return (per + 31) / 32;
  const int64_t want = std::max<int64_t>(1, 148 * 8 / d.samples);
  return std::max<int64_t>(1, std::min(want, (per + 7) / 8));
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
    norm_columns_backward_kernel<T><<<static_cast<unsigned>(chunks * d.samples), kColWarps * 32, 0, stream>>>(A);
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
    norm_param_grads_kernel<T><<<dim3(cx, ns), 1024, 0, stream>>>(B, gs, A.part + s0 * chunks * 4 * A.C,
                                                                  totals ? per_sample + s0 * 4 * A.C : nullptr, 1);
    if ((st = launched("norm gradients")) != KSMM_OK) return st;
  }
  if (d.samples > 1 && totals) {
    norm_param_grads_kernel<T><<<cx, 1024, 0, stream>>>(A, g, per_sample, nullptr, 0);
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
  if (d->scale_stride < 0 || d->shift_stride < 0 || d->gate_stride < 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "negative stride");
  if (!(d->eps >= 0.f)) return set_error(KSMM_ERR_BAD_ARGUMENT, "eps must not be negative");
  return KSMM_OK;
}

size_t norm_workspace(const ksmm_norm_desc_t& d) {
  return static_cast<size_t>(chunks_of(d) + 1) * d.samples * 4 * d.channels * sizeof(float);
}

}  // namespace
}  // namespace ksmm

using namespace ksmm;

extern "C" {

int ksmm_cu_norm_forward(const ksmm_norm_desc_t* d, void* stream) {
  int st = check_norm(d);
  if (st != KSMM_OK || d->rows == 0) return st;
  if (!d->x || (d->y && !d->z) || (d->norm != kNone && !d->h)) return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->dtype == KSMM_F32) return forward_typed<float>(*d, s);
  if (d->dtype == KSMM_F16) return forward_typed<__half>(*d, s);
  return forward_typed<__nv_bfloat16>(*d, s);
}

size_t ksmm_cu_norm_backward_workspace_bytes(const ksmm_norm_desc_t* d) {
  if (check_norm(d) != KSMM_OK || d->rows == 0 || !wants_sums(*d)) return 0;
  return norm_workspace(*d);
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
  if (!d->stats || (d->norm != kNone && d->grad_h && !(d->y ? d->z : d->x)) || (!d->grad_z && !d->grad_h))
    return set_error(KSMM_ERR_BAD_ARGUMENT, "null pointer");
  if (d->grad_h && d->norm == kNone) return set_error(KSMM_ERR_BAD_ARGUMENT, "a gradient of h without a norm");
  if (d->grad_z && !d->y) return set_error(KSMM_ERR_BAD_ARGUMENT, "a gradient of z without y");
  if (reinterpret_cast<uintptr_t>(d->stats) % 16 != 0)
    return set_error(KSMM_ERR_BAD_ARGUMENT, "the statistics are aligned to 16 bytes");
  const size_t need = wants_sums(*d) ? norm_workspace(*d) : 0;
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return set_error(KSMM_ERR_WORKSPACE, "norm backward: need %zu bytes aligned to 16, got %zu", need, workspace_bytes);
  if (d->dtype == KSMM_F32) return backward_typed<float>(*d, workspace, s);
  if (d->dtype == KSMM_F16) return backward_typed<__half>(*d, workspace, s);
  return backward_typed<__nv_bfloat16>(*d, workspace, s);
}

}  // extern "C"
