// Attention of few new tokens over a paged cache on the CUDA cores: rows_kernel for fp32 rows of whole 16-byte vectors, plain_kernel for
// what no other kernel takes (pages that are no multiple of 16 tokens, other alignments and orders, fp32 models on 8-bit caches), and
// the kernel that joins the parts of items which blocks shared.
//
// rows_kernel: eight lanes hold a token's key: with q in registers each lane multiplies its dims, three shuffles join them.  A warp
// has four such groups and a block eight warps, and every group keeps a running maximum, sum and output row of its own over its
// tokens, two at a time; they are joined once, at the end of a segment.
#include <atomic>

#include "cache.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

constexpr int kRowThreads = 256;
// Keys and values on their way: each thread copies its own pieces asynchronously into shared memory, kSlots units deep, and reads
// them back itself, without a barrier.  Wider rows would fill it with one unit.
constexpr int kSlots = 3;
constexpr bool row_ring(int dpl) { return dpl <= 16; }

// Dims (j * 8 + l) * 4 .. of a row, for lane l of eight.  (Plain loads: the append before this kernel may still be writing when its
// blocks start, and nothing is read before the wait.)
template <int DPL>
__device__ __forceinline__ void load_row(const float* row, int l, int dim, bool there, float* out) {
#pragma unroll
  for (int j = 0; j < DPL / 4; ++j) {
    const int d = (j * 8 + l) * 4;
    if (there && d < dim) {
      const float4 v = *reinterpret_cast<const float4*>(row + d);
      out[4 * j] = v.x;
      out[4 * j + 1] = v.y;
      out[4 * j + 2] = v.z;
      out[4 * j + 3] = v.w;
    } else {
      out[4 * j] = out[4 * j + 1] = out[4 * j + 2] = out[4 * j + 3] = 0.f;
    }
  }
}

// R: rows of an item.  Where a key head has one or two, registers for no more let several blocks share an SM, which is what keeps
// enough loads in flight (32 sequences of 12 heads of 64, fp32: 123 us with one block of eight rows, 67 with two of two rows, 74 with three).
template <int DPL, int R>
__global__ void __launch_bounds__(kRowThreads, row_blocks(8 * DPL, R)) rows_kernel(const __grid_constant__ Attend a) {
  constexpr bool kRing = row_ring(DPL);
  __shared__ Segment segment;
  __shared__ float stats[2][kRowThreads / 32][R];
  extern __shared__ __align__(16) char smem[];
  float* sums = reinterpret_cast<float*>(smem);  // [warp][R][8 DPL]
  const uint32_t smem_base = tc::smem_u32(smem), ring = smem_base + kRowThreads / 32 * R * 8 * DPL * sizeof(float);
  touch_parameters(a);
  tc::grid_dep_wait();
  tc::grid_dep_launch();
  clear_rest<float>(a);
  Walker walker;  // the first warp's
  bool some = true;
  if (threadIdx.x < 32) some = walker.start(a);
  if (!__syncthreads_or(threadIdx.x < 32 && some)) return;
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, l = lane % 8, at = warp * 4 + lane / 8;
  const float* q_rows = reinterpret_cast<const float*>(a.q);
  const float* data[2] = {reinterpret_cast<const float*>(p.data[0]), reinterpret_cast<const float*>(p.data[1])};

  bool slot_used[2] = {false, false};
  while (true) {
    if (warp == 0) {
      Segment next;
      walker.next(a, &next);
      if (lane == 0) segment = next;
    }
    __syncthreads();
    const Segment g = segment;
    if (g.s < 0) break;
    const int rows = min(R, g.n * a.group - g.tile * R);
    float q[R][DPL], o[R][DPL], m[R], sum[R];
    int position[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = g.tile * R + r, t = row / a.group;
      position[r] = r < rows ? g.length - g.n + t : -1;
      const int64_t from = (g.start + t) * a.q_token + (g.head * a.group + row - t * a.group) * a.q_head;
      load_row<DPL>(q_rows + from, l, p.dim, r < rows, q[r]);
      m[r] = kNone;
      sum[r] = 0.f;
#pragma unroll
      for (int e = 0; e < DPL; ++e) o[r][e] = 0.f;
    }
    const int32_t* table = p.table + g.s * p.table_stride;
    int page_next[2], row_next[2];  // of the next unit to be fetched: looked up a unit ahead
    bool want_next[2];              // whether the token is the sequence's (an entry outside the pool says nothing of it)
    auto look = [&](int unit) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int token = unit * kRowsUnit + h * 32 + at, nth = token / p.page_size;
        row_next[h] = token - nth * p.page_size;
        want_next[h] = unit < g.to && token >= g.lo && token < g.hi;
        page_next[h] = want_next[h] ? table[nth] : -1;
      }
    };
    // a thread's own bytes of the ring: nobody else reads them
    auto mine_at = [&](int slot, int h, int kv, int j) {
      return ring + static_cast<uint32_t>(((((slot * 2 + h) * 2 + kv) * (DPL / 4) + j) * kRowThreads + tid) * 16);
    };
    const float* nowhere = reinterpret_cast<const float*>(a.q);  // (a copy of no bytes still names an address)
    uint32_t gone = 0;  // a bit per token fetched, the last ones lowest: its page is not there
    int fetched = g.from, slot_in = 0, slot_out = 0;
    auto fetch = [&]() {
      gone <<= 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool get = page_next[h] >= 0 && page_next[h] < p.pages;
        if (!get && want_next[h]) gone |= 1u << h;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const float* row = data[kv] + static_cast<int64_t>(get ? page_next[h] : 0) * p.page[kv] + g.head * p.head[kv] + row_next[h] * p.token[kv];
#pragma unroll
          for (int j = 0; j < DPL / 4; ++j) {
            const int d = (j * 8 + l) * 4;
            const bool take = get && d < p.dim;
            // (zeros where there is nothing)
            if constexpr (kRing)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mine_at(slot_in, h, kv, j)), "l"(take ? row + d : nowhere), "r"(take ? 16 : 0) : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      slot_in = slot_in + 1 == kSlots ? 0 : slot_in + 1;
      look(++fetched);
    };
    look(g.from);
    if constexpr (kRing) {
#pragma unroll 1
      for (int i = 0; i < kSlots - 1; ++i) fetch();
    }
#pragma unroll 1
    for (int unit = g.from; unit < g.to; ++unit) {
      float k[2][DPL], v[2][DPL];
      int j[2];
      bool there[2], bad[2];
      if constexpr (kRing) {
        fetch();
        asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        j[h] = unit * kRowsUnit + h * 32 + at;
        there[h] = j[h] >= g.lo && j[h] < g.hi;
        if constexpr (kRing) {
          bad[h] = gone >> (2 * (kSlots - 1) + h) & 1;
#pragma unroll
          for (int c = 0; c < DPL / 4; ++c) {
            const float4 x = *reinterpret_cast<const float4*>(smem + (mine_at(slot_out, h, 0, c) - smem_base));
            const float4 y = *reinterpret_cast<const float4*>(smem + (mine_at(slot_out, h, 1, c) - smem_base));
            k[h][4 * c] = x.x;
            k[h][4 * c + 1] = x.y;
            k[h][4 * c + 2] = x.z;
            k[h][4 * c + 3] = x.w;
            v[h][4 * c] = y.x;
            v[h][4 * c + 1] = y.y;
            v[h][4 * c + 2] = y.z;
            v[h][4 * c + 3] = y.w;
          }
        } else {
          const int64_t page = page_next[h];
          const int nth = row_next[h];
          bad[h] = there[h] && (page < 0 || page >= p.pages);
          const bool get = there[h] && !bad[h];
          load_row<DPL>(data[0] + page * p.page[0] + g.head * p.head[0] + nth * p.token[0], l, p.dim, get, k[h]);
          load_row<DPL>(data[1] + page * p.page[1] + g.head * p.head[1] + nth * p.token[1], l, p.dim, get, v[h]);
        }
      }
      if constexpr (kRing) slot_out = slot_out + 1 == kSlots ? 0 : slot_out + 1;
      else look(unit + 1);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= rows) continue;
        float s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < DPL; ++e) d = fmaf(q[r][e], k[h][e], d);
          d += __shfl_xor_sync(0xffffffffu, d, 1);
          d += __shfl_xor_sync(0xffffffffu, d, 2);
          d += __shfl_xor_sync(0xffffffffu, d, 4);
          s[h] = bad[h] ? __int_as_float(0x7fffffff) : d * a.scale;
        }
        bool sees[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          sees[h] = there[h] && j[h] <= position[r] && (!a.window || j[h] > position[r] - a.window);
        float top = m[r];
        if (sees[0]) top = fmaxf(top, s[0]);
        if (sees[1]) top = fmaxf(top, s[1]);
        if (top != m[r]) {
          const float f = exp2f(m[r] - top);
          sum[r] *= f;
#pragma unroll
          for (int e = 0; e < DPL; ++e) o[r][e] *= f;
          m[r] = top;
        }
        // (a token that the row does not see is left out, whatever it holds)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!sees[h]) continue;
          const float w = exp2f(s[h] - top);
          sum[r] += w;
#pragma unroll
          for (int e = 0; e < DPL; ++e) o[r][e] = fmaf(w, v[h][e], o[r][e]);
        }
      }
    }

    if constexpr (kRing) asm volatile("cp.async.wait_group 0;" ::: "memory");  // (what was fetched beyond the end: zeros)
    // the four groups of a warp, then the warps
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int x = 8; x < 32; x *= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, m[r], x), top = fmaxf(m[r], other);
        const float f = exp2f(m[r] - top);
        sum[r] *= f;
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], x);
#pragma unroll
        for (int e = 0; e < DPL; ++e) {
          o[r][e] *= f;
          o[r][e] += __shfl_xor_sync(0xffffffffu, o[r][e], x);
        }
        m[r] = top;
      }
      if (lane < 8) {
#pragma unroll
        for (int e = 0; e < DPL; ++e) sums[(warp * R + r) * 8 * DPL + (e / 4 * 8 + l) * 4 + e % 4] = o[r][e];
        if (lane == 0) {
          stats[0][warp][r] = m[r];
          stats[1][warp][r] = sum[r];
        }
      }
    }
    __syncthreads();
    const int slot = g.slot;
    if (slot && tid == 0) a.slots[2 * blockIdx.x + slot - 1] = g.item;
    if (slot) slot_used[slot - 1] = true;
    float* part = a.partial + (2 * static_cast<int64_t>(blockIdx.x) + slot - 1) * a.tile_rows * (p.dim + 2);
    for (int i = tid; i < rows * p.dim; i += kRowThreads) {
      const int r = i / p.dim, d = i - r * p.dim;
      float top = stats[0][0][r];
#pragma unroll
      for (int w = 1; w < kRowThreads / 32; ++w) top = fmaxf(top, stats[0][w][r]);
      float total = 0.f, out = 0.f;
#pragma unroll
      for (int w = 0; w < kRowThreads / 32; ++w) {
        const float f = exp2f(stats[0][w][r] - top);
        total = fmaf(f, stats[1][w][r], total);
        out = fmaf(f, sums[(w * R + r) * 8 * DPL + d], out);
      }
      if (g.bad) total = __int_as_float(0x7fffffff);
      if (slot) {
        part[i] = out;
        if (d == 0) {
          part[a.tile_rows * p.dim + r] = top;
          part[a.tile_rows * (p.dim + 1) + r] = total;
        }
      } else {
        const int row = g.tile * R + r, t = row / a.group;
        reinterpret_cast<float*>(a.out)[(g.start + t) * a.out_token + (g.head * a.group + row - t * a.group) * a.out_head + d] =
            total == 0.f ? 0.f : out / total;
      }
    }
    __syncthreads();
  }
  if (a.split && tid < 2 && !slot_used[tid]) a.slots[2 * blockIdx.x + tid] = -1;
}

// Any type, alignment and page size, one element at a time: a warp for each row, a lane for each of 32 keys while the scores are
// formed and for every 32nd column while the values are added.  (Rows of eight lanes in all these variants were 4 MB of code.)
constexpr int kPlainThreads = 32 * kPlainRows;

template <typename T, typename C>
__global__ void __launch_bounds__(kPlainThreads) plain_kernel(const __grid_constant__ Attend a) {
  constexpr bool kEight = sizeof(C) == 1;
  __shared__ Segment segment;
  __shared__ float q[kPlainRows][kMaxDim];
  touch_parameters(a);
  tc::grid_dep_wait();
  tc::grid_dep_launch();
  clear_rest<T>(a);
  const Pool& p = a.pool;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  Walker walker;  // the first warp's
  bool some = true;
  if (warp == 0) some = walker.start(a);
  if (!__syncthreads_or(warp == 0 && some)) return;
  bool slot_used[2] = {false, false};
  while (true) {
    if (warp == 0) {
      Segment next;
      walker.next(a, &next);
      if (lane == 0) segment = next;
    }
    __syncthreads();
    const Segment g = segment;
    if (g.s < 0) break;
    if (g.slot) slot_used[g.slot - 1] = true;
    const int rows = min(kPlainRows, g.n * a.group - g.tile * kPlainRows);
    const int row = g.tile * kPlainRows + warp, t = row / a.group, position = g.length - g.n + t;
    if (warp < rows) {
      const T* from = reinterpret_cast<const T*>(a.q) + (g.start + t) * a.q_token + (g.head * a.group + row - t * a.group) * a.q_head;
      for (int d = lane; d < p.dim; d += 32) q[warp][d] = ElemTraits<T>::to_float(from[d]);
      __syncwarp();
      float m = kNone, sum = 0.f, o[kMaxDim / 32];
#pragma unroll
      for (int c = 0; c < kMaxDim / 32; ++c) o[c] = 0.f;
      const int last = min(g.to << a.unit_log2, g.hi);
#pragma unroll 1
      for (int key0 = max(g.from << a.unit_log2, g.lo); key0 < last; key0 += 32) {
        const int key = key0 + lane;
        const bool sees = key < last && key <= position && (!a.window || key > position - a.window);
        int64_t page = -1, nth = 0;
        float s = -INFINITY;
        if (sees) {
          const int at = key / p.page_size;
          nth = key - at * p.page_size;
          page = p.table[g.s * p.table_stride + at];
          if (page < 0 || page >= p.pages) {
            page = -1;
            s = __int_as_float(0x7fffffff);
          } else {
            const C* k = reinterpret_cast<const C*>(p.data[0]) + page * p.page[0] + g.head * p.head[0] + nth * p.token[0];
            float dot = 0.f;
#pragma unroll 4
            for (int d = 0; d < p.dim; ++d) dot = fmaf(q[warp][d], ElemTraits<C>::to_float(k[d]), dot);
            if (kEight) dot *= p.scales[0][page * p.spage[0] + g.head * p.shead[0] + nth * p.stoken[0]];
            s = dot * a.scale;
          }
        }
        float top = s;
#pragma unroll
        for (int x = 16; x; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top, m);
        const float f = exp2f(m - top), w = exp2f(s - top);
        m = top;
        sum = sum * f + w;  // (of this lane's keys)
#pragma unroll
        for (int c = 0; c < kMaxDim / 32; ++c) o[c] *= f;
        const int64_t at = page * p.page[1] + g.head * p.head[1] + nth * p.token[1];
        const float scale = kEight && page >= 0 ? p.scales[1][page * p.spage[1] + g.head * p.shead[1] + nth * p.stoken[1]] : 1.f;
        const int n = min(32, last - key0);
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          // (keys that the row does not see, or that are not there, add nothing)
          if (__shfl_sync(0xffffffffu, page, j) < 0) continue;
          const C* v = reinterpret_cast<const C*>(p.data[1]) + __shfl_sync(0xffffffffu, at, j);
          const float x = __shfl_sync(0xffffffffu, w * scale, j);
#pragma unroll
          for (int c = 0; c < kMaxDim / 32; ++c)
            if (lane + 32 * c < p.dim) o[c] = fmaf(x, ElemTraits<C>::to_float(v[lane + 32 * c]), o[c]);
        }
      }
#pragma unroll
      for (int x = 16; x; x /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if (g.bad) sum = __int_as_float(0x7fffffff);
      if (g.slot) {
        float* part = a.partial + (2 * static_cast<int64_t>(blockIdx.x) + g.slot - 1) * kPlainRows * (p.dim + 2);
        if (tid == 0) a.slots[2 * blockIdx.x + g.slot - 1] = g.item;
#pragma unroll
        for (int c = 0; c < kMaxDim / 32; ++c)
          if (lane + 32 * c < p.dim) part[warp * p.dim + lane + 32 * c] = o[c];
        if (lane == 0) {
          part[kPlainRows * p.dim + warp] = m;
          part[kPlainRows * (p.dim + 1) + warp] = sum;
        }
      } else {
        T* to = reinterpret_cast<T*>(a.out) + (g.start + t) * a.out_token + (g.head * a.group + row - t * a.group) * a.out_head;
        const float back = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int c = 0; c < kMaxDim / 32; ++c)
          if (lane + 32 * c < p.dim) to[lane + 32 * c] = ElemTraits<T>::from_float(o[c] * back);
      }
    }
    __syncthreads();
  }
  if (a.split && tid < 2 && !slot_used[tid]) a.slots[2 * blockIdx.x + tid] = -1;
}

// Joins the parts of items that several blocks shared.  Block (c, r): row r of the item that begins in block c and goes on; its
// further parts are in slot 0 of the blocks after c, as long as they name the item.  They are summed in the order of the blocks,
// eight runs side by side, whoever was first.  A chain of reads is all the time that it takes: what may turn out not to be a
// part (maxima and sums of the first blocks after c) is read before that is known.
constexpr int kJoinThreads = 256;
constexpr int kAhead = 8;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Attend a, int blocks) {
  constexpr int kWarps = kJoinThreads / 32, kReads = kMaxBlocks / kJoinThreads;
  __shared__ float weight[kMaxBlocks];
  __shared__ float reduce[2][kWarps];
  __shared__ float sums[kWarps][kMaxDim];
  touch_parameters(a);
  tc::grid_dep_wait();
  tc::grid_dep_launch();
  const Pool& p = a.pool;
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t size = static_cast<int64_t>(a.tile_rows) * (p.dim + 2);
  auto part = [&](int i) { return a.partial + (i == 0 ? 2 * c + 1 : 2 * static_cast<int64_t>(c + i)) * size; };
  const int64_t item = a.slots[2 * c + 1];
  if (item < 0) return;
  int64_t named[kReads];
  float m[kReads], l[kReads];
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    const int i = tid + k * kJoinThreads;
    const bool there = c + i < blocks;
    named[k] = !there ? -1 : i == 0 ? item : a.slots[2 * static_cast<int64_t>(c + i)];
    m[k] = l[k] = 0.f;
    // (few items have more parts than this; reading all blocks' values took 4 us more than the second wait)
    if (there && i < kAhead) {
      m[k] = part(i)[a.tile_rows * p.dim + r];
      l[k] = part(i)[a.tile_rows * (p.dim + 1) + r];
    }
  }
  const int s = static_cast<int>((item >> 32) / p.kv_heads), head = static_cast<int>((item >> 32) % p.kv_heads);
  const int tile = static_cast<int>(item & 0xffffffff);
  const Sequence q = sequence(p, s);
  if (tile * a.tile_rows + r >= q.n * a.group) return;
  int parts = 0;
  float top = kNone;
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    // (an item's blocks follow one another)
    parts += __syncthreads_count(named[k] == item);
    if (named[k] != item) continue;
    const int i = tid + k * kJoinThreads;
    if (i >= kAhead) {
      m[k] = part(i)[a.tile_rows * p.dim + r];
      l[k] = part(i)[a.tile_rows * (p.dim + 1) + r];
    }
    top = fmaxf(top, m[k]);
  }
#pragma unroll
  for (int x = 16; x; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  if (lane == 0) reduce[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, reduce[0][w]);
  float total = 0.f;
#pragma unroll
  for (int k = 0; k < kReads; ++k) {
    if (named[k] != item) continue;
    const float f = exp2f(m[k] - top);
    weight[tid + k * kJoinThreads] = f;
    total = fmaf(f, l[k], total);
  }
#pragma unroll
  for (int x = 16; x; x /= 2) total += __shfl_xor_sync(0xffffffffu, total, x);
  if (lane == 0) reduce[1][warp] = total;
  __syncthreads();
  total = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += reduce[1][w];
  constexpr int kPer = kMaxDim / 32;
  float sum[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) sum[k] = 0.f;
#pragma unroll 4
  for (int i = warp; i < parts; i += kWarps) {
    const float* from = part(i) + r * p.dim + lane;
    const float f = weight[i];
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (lane + 32 * k < p.dim) sum[k] = fmaf(f, from[32 * k], sum[k]);
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) sums[warp][lane + 32 * k] = sum[k];
  __syncthreads();
  const int row = tile * a.tile_rows + r, t = row / a.group;
  T* out = reinterpret_cast<T*>(a.out) + (q.start + t) * a.out_token + (head * a.group + row - t * a.group) * a.out_head;
  if (tid >= p.dim) return;
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += sums[w][tid];
  out[tid] = ElemTraits<T>::from_float(total == 0.f ? 0.f : all / total);
}

template <int DPL, int R>
int launch_one(const Attend& a, unsigned grid, cudaStream_t stream) {
  constexpr size_t smem = kRowThreads / 32 * R * DPL * 8 * sizeof(float) + (row_ring(DPL) ? kSlots * 4 * DPL * sizeof(float) * kRowThreads : 0);
  static std::atomic<uint64_t> ready{0};  // a bit per device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(ready.load(std::memory_order_acquire) & bit)) {
    err = cudaFuncSetAttribute(rows_kernel<DPL, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  }
  if (err == cudaSuccess) err = tc::launch_pdl(rows_kernel<DPL, R>, grid, kRowThreads, smem, stream, a);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "attention rows kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

template <typename T, typename C>
int launch_plain_one(const Attend& a, unsigned grid, cudaStream_t stream) {
  const cudaError_t err = tc::launch_pdl(plain_kernel<T, C>, grid, kPlainThreads, 0, stream, a);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "attention plain kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

template <typename T>
int launch_plain_cached(const Attend& a, int cache_dtype, unsigned grid, cudaStream_t stream) {
  return cache_dtype == KSMM_F8E4M3 ? launch_plain_one<T, f8e4m3>(a, grid, stream) : launch_plain_one<T, T>(a, grid, stream);
}

}  // namespace

int launch_rows(const Attend& a, unsigned grid, cudaStream_t stream) {
  const bool few = a.tile_rows == kFewRowsTile;
  if (a.pool.dim <= 64) return few ? launch_one<8, kFewRowsTile>(a, grid, stream) : launch_one<8, 8>(a, grid, stream);
  if (a.pool.dim <= 128) return few ? launch_one<16, kFewRowsTile>(a, grid, stream) : launch_one<16, 4>(a, grid, stream);
  return launch_one<32, kFewRowsTile>(a, grid, stream);
}

int launch_plain(const Attend& a, int dtype, int cache_dtype, unsigned grid, cudaStream_t stream) {
  if (dtype == KSMM_F32) return launch_plain_cached<float>(a, cache_dtype, grid, stream);
  if (dtype == KSMM_F16) return launch_plain_cached<__half>(a, cache_dtype, grid, stream);
  return launch_plain_cached<__nv_bfloat16>(a, cache_dtype, grid, stream);
}

template <typename T>
static int launch_join_typed(const Attend& a, unsigned blocks, int rows, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, rows);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = tc::pdl_enabled() ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, join_kernel<T>, a, static_cast<int>(blocks));
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "attention join kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

int launch_join(const Attend& a, int dtype, unsigned blocks, int rows, cudaStream_t stream) {
  if (dtype == KSMM_F32) return launch_join_typed<float>(a, blocks, rows, stream);
  if (dtype == KSMM_F16) return launch_join_typed<__half>(a, blocks, rows, stream);
  return launch_join_typed<__nv_bfloat16>(a, blocks, rows, stream);
}

}  // namespace cache
}  // namespace ksmm
