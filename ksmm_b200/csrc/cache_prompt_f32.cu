// Attention of many new tokens (prompts) over a paged cache in fp32, on the CUDA cores.
//
// A block has one key head and a tile of 64 rows (token, head of the group); 256 threads as 16 x 16.  Per 64 keys: each thread forms 4
// x 4 scores from q and K in shared memory, 16 threads find their rows' maxima and sums by shuffles, the weights go to
// shared memory, and each thread adds 4 rows x (columns / 16) of the output.  Every value that a thread reads meets four others, so
// the FMA pipes wait for neither loads nor shared memory (the kernel for few rows, a token per eight lanes, met each key with four
// rows only: 6.6 ms against 4.1 ms for the same formula as library products).  V's rows are on their way while the scores are formed, the
// next K's while the output is; blocks side by side on an SM fill the rest.  28 to 35 TFLOP/s of the pairs that are seen, of 72 that
// the FMA pipes have (2000 tokens of 32/8 heads of 128: 1.0 ms).  What bounds it: the FMA pipes are busy for 50 % of the cycles (tiles on
// the diagonal form twice the pairs that are seen) and 63 % issue, with two warps on a scheduler that wait for shared memory.  The tensor
// cores are not used: three tf32 products per term keep 21 bits, six of bf16 parts would keep 24 and are not built.
#include <atomic>

#include "cache.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

constexpr int kTile = 64;  // rows, and keys
constexpr int kFloatThreads = 256;

template <int DP>
struct Float {
  static constexpr int kRow = DP + 4;  // floats of a row in shared memory: 8 rows' vectors are on different banks
  static constexpr int kQAt = 0, kKAt = kTile * kRow, kVAt = 2 * kTile * kRow, kPAt = 3 * kTile * kRow;
  static constexpr int kPRow = kTile + 4;
  static constexpr int kOffsetsAt = kPAt + kTile * kPRow;  // two tiles' int64: where a key starts, -1: nothing, -2: a page that is not there
  static constexpr int kBytes = kOffsetsAt * 4 + 2 * 2 * kTile * 8 + static_cast<int>(sizeof(Segment));
  static constexpr int kBlocks = 228 * 1024 / (kBytes + 1024) < 3 ? 228 * 1024 / (kBytes + 1024) : 3;  // on an SM
};

__device__ __forceinline__ void copy16(uint32_t dst, const float* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int DP>
__global__ void __launch_bounds__(kFloatThreads, Float<DP>::kBlocks) float_kernel(const __grid_constant__ Attend a) {
  using C = Float<DP>;
  constexpr int kCols = DP / 64;  // vectors of four columns of a thread
  extern __shared__ __align__(16) float smem_f[];
  float *qs = smem_f + C::kQAt, *ks = smem_f + C::kKAt, *vs = smem_f + C::kVAt, *ps = smem_f + C::kPAt;
  int64_t* offsets = reinterpret_cast<int64_t*>(smem_f + C::kOffsetsAt);  // [tile % 2][key, value][token]
  Segment* segment = reinterpret_cast<Segment*>(offsets + 2 * 2 * kTile);
  const uint32_t base = tc::smem_u32(smem_f);
  touch_parameters(a);
  tc::grid_dep_wait();
  tc::grid_dep_launch();
  clear_rest<float>(a);
  const Pool& p = a.pool;
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  if (tid < 32) {
    Walker walker;
    Segment next;
    next.s = -1;
    if (walker.start(a)) walker.next(a, &next);
    if (tid == 0) *segment = next;
  }
  __syncthreads();
  const Segment g = *segment;
  if (g.s < 0) return;
  const int rows = min(kTile, g.n * a.group - g.tile * kTile);
  const int32_t* table = p.table + g.s * p.table_stride;
  const float* data[2] = {reinterpret_cast<const float*>(p.data[0]), reinterpret_cast<const float*>(p.data[1])};

  auto look = [&](int tile) {
    // where a tile's keys and values are
    if (tid >= 2 * kTile) return;
    const int kv = tid / kTile, token = tile * kTile + tid % kTile;
    int64_t at = -1;
    if (tile < g.to && token >= g.lo && token < g.hi) {
      const int nth = token / p.page_size, page = table[nth];
      at = page < 0 || page >= p.pages ? -2 : page * p.page[kv] + g.head * p.head[kv] + static_cast<int64_t>(token - nth * p.page_size) * p.token[kv];
    }
    offsets[(tile & 1) * 2 * kTile + tid] = at;
  };
  auto fetch = [&](int tile, int kv) {
    const int64_t* from = offsets + (tile & 1) * 2 * kTile + kv * kTile;
    const uint32_t to = base + 4 * (kv ? C::kVAt : C::kKAt);
#pragma unroll 4
    for (int e = tid; e < kTile * (DP / 4); e += kFloatThreads) {
      const int r = e / (DP / 4), d = e % (DP / 4) * 4;
      const int64_t at = from[r];
      const bool there = at >= 0 && d < p.dim;  // (zeros else: what the rows do not see stays out of the sums)
      copy16(to + 4 * (r * C::kRow + d), there ? data[kv] + at + d : reinterpret_cast<const float*>(a.q), there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  look(g.from);
  for (int e = tid; e < kTile * (DP / 4); e += kFloatThreads) {
    const int r = e / (DP / 4), d = e % (DP / 4) * 4, row = g.tile * kTile + r, t = row / a.group;
    const bool there = r < rows && d < p.dim;
    const float* from = reinterpret_cast<const float*>(a.q) +
                        (there ? (g.start + t) * a.q_token + (g.head * a.group + row - t * a.group) * a.q_head + d : 0);
    copy16(base + 4 * (C::kQAt + r * C::kRow + d), from, there);
  }
  __syncthreads();
  fetch(g.from, 0);  // (with q)

  float o[4][kCols][4], m[4], sum[4];
  int position[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = kNone;
    sum[i] = 0.f;
    position[i] = g.length - g.n + (g.tile * kTile + ty * 4 + i) / a.group;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
  }
#pragma unroll 1
  for (int tile = g.from; tile < g.to; ++tile) {
    fetch(tile, 1);
    look(tile + 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    // ---- scores: rows 4 ty + i, keys tx + 16 j ----
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 q[4], k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * C::kRow + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * C::kRow + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(q[i].w, k[j].w, fmaf(q[i].z, k[j].z, fmaf(q[i].y, k[j].y, fmaf(q[i].x, k[j].x, s[i][j]))));
    }
    const int64_t* at = offsets + (tile & 1) * 2 * kTile;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = tile * kTile + tx + 16 * j;
      const bool in = key >= g.lo && key < g.hi, gone = at[tx + 16 * j] == -2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool sees = in && key <= position[i] && (!a.window || key > position[i] - a.window);
        s[i][j] = sees ? (gone ? __int_as_float(0x7fffffff) : s[i][j] * a.scale) : -INFINITY;
      }
    }
    // ---- maximum and sum over a row's 16 threads ----
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(top, m[i]);
      const float f = exp2f(m[i] - top);
      m[i] = top;
      sum[i] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - top);
        sum[i] += s[i][j];  // (of this thread's keys)
        ps[(ty * 4 + i) * C::kPRow + tx + 16 * j] = s[i][j];
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][c][e] *= f;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (tile + 1 < g.to) fetch(tile + 1, 0);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    // ---- output: rows 4 ty + i, columns 64 c + 4 tx .. ----
#pragma unroll 2
    for (int k = 0; k < kTile; k += 4) {
      float4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4*>(ps + (ty * 4 + i) * C::kPRow + k);
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const float4 v = *reinterpret_cast<const float4*>(vs + (k + q) * C::kRow + 64 * c + 4 * tx);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = q == 0 ? w[i].x : q == 1 ? w[i].y : q == 2 ? w[i].z : w[i].w;
            o[i][c][0] = fmaf(x, v.x, o[i][c][0]);
            o[i][c][1] = fmaf(x, v.y, o[i][c][1]);
            o[i][c][2] = fmaf(x, v.z, o[i][c][2]);
            o[i][c][3] = fmaf(x, v.w, o[i][c][3]);
          }
        }
    }
    __syncthreads();  // (V and the weights are written again)
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int x = 1; x < 16; x *= 2) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], x);
    if (g.bad) sum[i] = __int_as_float(0x7fffffff);
    const int r = ty * 4 + i, row = g.tile * kTile + r, t = row / a.group;
    if (r >= rows) continue;
    float* to = reinterpret_cast<float*>(a.out) + (g.start + t) * a.out_token + (g.head * a.group + row - t * a.group) * a.out_head;
    const float back = sum[i] == 0.f ? 0.f : 1.f / sum[i];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int d = 64 * c + 4 * tx;
      if (d < p.dim)
        *reinterpret_cast<float4*>(to + d) = make_float4(o[i][c][0] * back, o[i][c][1] * back, o[i][c][2] * back, o[i][c][3] * back);
    }
  }
}

template <int DP>
int launch_one(const Attend& a, unsigned grid, cudaStream_t stream) {
  auto kern = float_kernel<DP>;
  static std::atomic<uint64_t> ready{0};  // a bit per device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(ready.load(std::memory_order_acquire) & bit)) {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Float<DP>::kBytes);
    if (err == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  }
  if (err == cudaSuccess) err = tc::launch_pdl(kern, grid, kFloatThreads, Float<DP>::kBytes, stream, a);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "attention float kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

}  // namespace

int launch_float(const Attend& a, unsigned grid, cudaStream_t stream) {
  if (a.pool.dim <= 64) return launch_one<64>(a, grid, stream);
  if (a.pool.dim <= 128) return launch_one<128>(a, grid, stream);
  return launch_one<256>(a, grid, stream);
}

}  // namespace cache
}  // namespace ksmm
