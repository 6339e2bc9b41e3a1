// Attention of few new tokens over a paged cache in 16 or 8 bits.
//
// Each key and value is read once and met by the few rows of q that share its head, so the kernel is a stream of memory.  Its blocks,
// as many as fit the SMs, share all sequences' units evenly however their lengths differ (cache.cuh).  One warp of a block walks its
// share, hands each segment with its rows of q on, and keeps a ring of 3 to 6 units in flight through TMA (96 KB a block, 190 KB on
// an SM; 43 GB/s per SM times 1.5 us of latency need 65).  Four warps (eight for 256 columns) take 16 or 32 tokens of a unit each,
// with a running maximum, sum and output of their own, and meet only at the end of a segment: warps that each wait for their unit
// alone hide the latency that a block-wide step for each unit would show.  Parts of an item that several blocks shared are joined by
// join_kernel (cache_rows.cu).
//
// Measured (one B200, kernel and join): 64 sequences of 1 to 8192 tokens, 32/8 heads of 128, bf16: 184 us, 5.9 TB/s of the 6.4 that a
// copy reaches; 131077 tokens of one sequence 93 us (86 the kernel, 7 the join); 128 sequences in 8 bits 213 us, 5.6 TB/s; a window
// of 4096 tokens on heads of 256: 76 us, 4.6 TB/s.  Short sequences are bound by a block's start and a segment's chain: 64 of up to 512
// tokens take 33 us for 71 MB.
//
// mma.sync, not tcgen05: an item has 8 or 16 rows (heads that share a key head, new tokens), a sixteenth of tcgen05's
// smallest tile, and the scores have to come back to registers at once.  Its rate is what a step costs (two warps on a
// scheduler took 1800 cycles for 48 products each of 16 tokens x 128), so the tokens are the 16 rows of a product and the rows of q its
// 8 columns: S^T = K q^T with K as the A operand as it lies in shared memory, o^T = V^T w^T with V through transposing loads and w^T
// transposed in registers; with the rows of q as A half of a tile's 16 rows stood idle.  Of 16-bit caches the weights enter the
// second product as two 16-bit parts (w = hi + lo, each rounded): one part would add an error as large as the result's final
// rounding.  fp16 parts are subnormal below 2^-14 and end at 2^-24, so weights of fp16 products are raised by 2^15 (a row's reference m
// is its maximum less 15; the sum has the same factor): they lose digits from 2^-29 of the row's largest on.
//
// 8-bit caches: the products run in fp16, which holds e4m3 exactly.  q is scaled by a power of two per row so that bf16's
// range fits; a token's key scale multiplies its scores; its value scale f, of any sign, multiplies its weight.  What has to fit
// fp16 is that product, so a row's reference is the maximum of score + log2 |f|, less 15: a token of a large scale and hardly any weight
// does not take the others' digits, nor one of a large weight and values near zero.  Weights alone then reach 2^95, which fp32
// holds 2^31 of (log2 |f| counts as -80 at least).  A bf16 model's products go in as one fp16 number, off by 2^-11 at most, an eighth
// of the result's own rounding.  One 16-byte chunk of a key row is a k step: its elements are taken in the order 4 q, 4 q + 1 | 4 q +
// 2, 4 q + 3 that the load gives, by q as well.
#include <atomic>
#include <climits>
#include <type_traits>

#include "cache.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

using namespace tc;


template <bool EIGHT, int DP, int NT>
struct Layout {
  static constexpr int kRows = 8 * NT;                                  // of an item
  // Warps that meet different tokens; rows of 256 have two for the same tokens, each with half of the output's columns (one alone has
  // 96 products and 32 loads in a step, and nothing else on its scheduler)
  static constexpr int kRuns = 4, kHalves = DP == 256 ? 2 : 1, kConsumers = kRuns * kHalves;
  static constexpr int kThreads = (kConsumers + 1) * 32;
  static constexpr int kCols = DP / kHalves;                            // of a warp's output
  static constexpr int kStep = token_shape(EIGHT, DP).unit / kRuns;
  static constexpr int kTokens = kRuns * kStep;                         // a unit, a stage of the ring
  static constexpr int kBoxes = EIGHT ? (DP + 127) / 128 : DP / 64;     // 128-byte columns of a row
  static constexpr int kOperand = kBoxes * kTokens * 128;               // a unit's keys
  static constexpr int kScales = EIGHT ? 2 * kTokens * 4 : 0;
  static constexpr int kStageBytes = 2 * kOperand;
  static constexpr int kBlocks = token_shape(EIGHT, DP).blocks;         // on an SM
  static constexpr int kStages = 196608 / kBlocks / (kStageBytes + kScales);
  static constexpr int kMerge = kRuns * 4 * kCols * 4;                  // the runs' output for 4 rows, or part of it for more
  static constexpr int kMergeAt = kStages * kStageBytes;
  static constexpr int kScalesAt = kMergeAt + kHalves * kMerge;
  static constexpr int kQRow = DP * 2 + 16;                             // bytes of a row of q (and no two rows on the same banks)
  static constexpr int kQAt = kScalesAt + kStages * kScales;
  static constexpr int kStatsAt = kQAt + kRows * kQRow;             // of the runs: maxima and sums of 16 rows, a half
  static constexpr int kBarsAt = kStatsAt + kHalves * kRuns * 2 * kRows * 4;    // full, empty | a segment full, empty
  static constexpr int kSegmentAt = kBarsAt + (2 * kStages + 2) * 8;
  static constexpr int kFlagsAt = kSegmentAt + static_cast<int>(sizeof(Segment));
  static constexpr int kBytes = kFlagsAt + kStages * 4 + 4;
  static_assert(kBlocks * (kBytes + 1024) <= 228 * 1024, "the blocks of an SM fit its shared memory");
  static_assert(kStages >= 2, "a ring");
};

struct Maps {
  CUtensorMap keys, values;
};

template <typename H>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(H) == 2 && ElemTraits<H>::kDtype == KSMM_F16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 8 x 8 values of 16 bits, a row of four pairs in the lanes 4 r .. 4 r + 3: transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename H>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  return pack2(lo, hi, ElemTraits<H>::kDtype);
}
template <typename H>
__device__ __forceinline__ float2 unpack(uint32_t v) {
  if constexpr (ElemTraits<H>::kDtype == KSMM_F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  else return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float log2_fast(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// a barrier of the consumers that tells all whether one says so
template <int THREADS>
__device__ __forceinline__ bool any_of(bool v) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r)
               : "r"(v ? 1u : 0u), "n"(THREADS)
               : "memory");
  return r != 0;
}

// A place in the ring.
template <int STAGES>
struct Turn {
  int stage = 0;
  uint32_t parity = 0;
  __device__ void next() {
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
  }
};

// T: q and the output.  Tokens of a page that one TMA box covers: 2^box_log2; a box lies in its stage as [128-byte column][token].
// `joined`: a map with the columns as a dimension of their own brings all of a box's at once.
template <typename T, bool EIGHT, int DP, int NT>
__global__ void __launch_bounds__(Layout<EIGHT, DP, NT>::kThreads, Layout<EIGHT, DP, NT>::kBlocks)
    token_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Attend a, const int box_log2, const int joined) {
  using L = Layout<EIGHT, DP, NT>;
  using H = typename std::conditional<EIGHT, __half, T>::type;  // of the products
  // whether the weights go in as two parts: e4m3 values times fp16 weights are far within a bf16 result's rounding
  constexpr bool kParts = !(EIGHT && ElemTraits<T>::kDtype == KSMM_BF16);
  constexpr int G = L::kStep / 16;  // groups of 16 tokens of a step
  constexpr float kRaise = ElemTraits<H>::kDtype == KSMM_F16 ? 15.f : 0.f;
  extern __shared__ __align__(1024) char smem[];
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  int* flags = reinterpret_cast<int*>(smem + L::kFlagsAt);
  volatile int* abort_flag = flags + L::kStages;
  const uint32_t full = base + L::kBarsAt, empty = full + 8 * L::kStages, segment_full = empty + 8 * L::kStages, segment_empty = segment_full + 8;
  Segment* const segment = reinterpret_cast<Segment*>(smem + L::kSegmentAt);
  if (base % 1024) {  // (without static shared memory it starts there; swizzled tiles need it)
    if (tid == 0) atomicCAS(a.status, 0, kWaits + 3);
    return;
  }
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, L::kConsumers);
    }
    mbar_init(segment_full, 1);
    mbar_init(segment_empty, L::kConsumers);
    fence_mbar_init();
  }
  for (int i = tid; i < L::kRows * L::kQRow / 4; i += L::kThreads) reinterpret_cast<uint32_t*>(smem + L::kQAt)[i] = 0;
  if (warp == L::kConsumers && lane == 0) {
    prefetch_tensormap(&maps.keys);
    prefetch_tensormap(&maps.values);
  }
  touch_parameters(a);
  grid_dep_wait();
  grid_dep_launch();
  clear_rest<T>(a);
  __syncthreads();
  const Pool& p = a.pool;
  const int box = 1 << box_log2, box_bytes = box * 128;
  Turn<L::kStages> turn;
  uint32_t segments = 0;  // so far

  if (warp == L::kConsumers) {
    // ---------------- producer: the warp walks the loop, tables 32 boxes ahead, one lane issues ----------------
    const int boxes = L::kTokens >> box_log2;
    const uint32_t bytes = static_cast<uint32_t>(box_bytes) * L::kBoxes * 2 + (EIGHT ? 2 * box * 4 : 0);
    const bool one = elect_one();
    uint32_t issued = 0;
    bool alive = true;
    Walker walker;
    bool more = walker.start(a);
    while (alive) {
      Segment g;
      g.s = -1;
      if (more) walker.next(a, &g);
      more = more && g.s >= 0;
      const int32_t* table = p.table + g.s * p.table_stride;
      int row_ahead = 0, page_ahead = -1, batch = 0;
      bool wanted = false;  // (whether a box is the sequence's; an entry outside the pool says nothing of it, whatever its value)
      auto look = [&](int u) {
        // the pages of the next 32 boxes
        const int token = u * L::kTokens + (lane << box_log2), nth = token / p.page_size;
        wanted = token < g.hi && token + box > g.lo;
        page_ahead = wanted ? table[nth] : -1;
        row_ahead = token - nth * p.page_size;
      };
      if (more) look(g.from);
      // hand it on, with its rows of q
      alive = __all_sync(0xffffffffu, mbar_wait<20>(segment_empty, (segments & 1) ^ 1, abort_flag, a.status, kWaits));
      if (!alive) break;
      if (more) {
        const int rows = min(L::kRows, g.n * a.group - g.tile * L::kRows);
        const int row = g.tile * L::kRows + min(lane, rows - 1), t = row / a.group;
        const int64_t row_at = (g.start + t) * a.q_token + (g.head * a.group + row - t * a.group) * a.q_head;
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
          const T* from = reinterpret_cast<const T*>(a.q) + __shfl_sync(0xffffffffu, row_at, r);
#pragma unroll
          for (int d = 0; d < DP; d += 64) {
            const int at = d + 2 * lane;
            if (at < p.dim) *reinterpret_cast<uint32_t*>(smem + L::kQAt + r * L::kQRow + at * 2) = *reinterpret_cast<const uint32_t*>(from + at);
          }
        }
      }
      if (lane == 0) *segment = g;
      __syncwarp();
      if (lane == 0) mbar_arrive(segment_full);
      ++segments;
      if (!more) break;
      for (int u = g.from; u < g.to; ++u) {
        if (batch == 0) {
          if (u > g.from) look(u);
          if (page_ahead >= p.pages) page_ahead = -1;
        }
        const bool of_unit = lane >= batch && lane < batch + boxes;
        const uint32_t missing = __ballot_sync(0xffffffffu, of_unit && wanted && page_ahead < 0) >> batch;
        const uint32_t load = __ballot_sync(0xffffffffu, of_unit && page_ahead >= 0) >> batch;
        const int st = turn.stage;
        alive = __all_sync(0xffffffffu, mbar_wait<0>(empty + 8 * st, turn.parity ^ 1, abort_flag, a.status, kWaits));
        if (!alive) break;
        const uint32_t bar = full + 8 * st;
        if (one) {
          flags[st] = static_cast<int>(missing);
          if (load) mbar_expect_tx(bar, __popc(load) * bytes);
          else mbar_arrive(bar);
        }
        // (same values in all lanes: addresses in uniform registers.  A lane for each box took 170 cycles per copy)
        for (int b = 0; b < boxes; ++b) {
          const int page = __shfl_sync(0xffffffffu, page_ahead, batch + b), row = __shfl_sync(0xffffffffu, row_ahead, batch + b);
          if (page < 0 || !one) continue;
          const uint32_t to = base + st * L::kStageBytes + b * box_bytes * L::kBoxes;
          if (joined) {
            tma_load_5d(to, &maps.keys, bar, 0, row, 0, g.head, page);
            tma_load_5d(to + L::kOperand, &maps.values, bar, 0, row, 0, g.head, page);
          } else {
#pragma unroll
            for (int k = 0; k < L::kBoxes; ++k) {
              tma_load_4d(to + k * box_bytes, &maps.keys, bar, k * (EIGHT ? 128 : 64), row, g.head, page);
              tma_load_4d(to + L::kOperand + k * box_bytes, &maps.values, bar, k * (EIGHT ? 128 : 64), row, g.head, page);
            }
          }
          if (EIGHT) {
            const uint32_t at = base + L::kScalesAt + st * L::kScales + b * box * 4;
            bulk_load(at, p.scales[0] + page * p.spage[0] + g.head * p.shead[0] + row, box * 4, bar);
            bulk_load(at + L::kTokens * 4, p.scales[1] + page * p.spage[1] + g.head * p.shead[1] + row, box * 4, bar);
          }
        }
        __syncwarp();
        ++issued;
        turn.next();
        batch += boxes;
        if (batch == 32) batch = 0;
      }
    }
    if (!alive) {
      // the copies in flight end before the block does
      int zero = 0;
      for (uint32_t i = issued > L::kStages ? issued - L::kStages : 0; i < issued; ++i)
        mbar_wait<100>(full + 8 * (i % L::kStages), i / L::kStages & 1, &zero, a.status, kWaits + 1);
    }
    return;
  }

  // ---------------- consumers ----------------
  const int gq = lane / 4, q4 = lane % 4;
  bool alive = true;
  bool slot_used[2] = {false, false};
  const int run = warp % L::kRuns, half = warp / L::kRuns;
  float* merge = reinterpret_cast<float*>(smem + L::kMergeAt + half * L::kMerge);
  float* stats = reinterpret_cast<float*>(smem + L::kStatsAt) + half * L::kRuns * 2 * L::kRows;
  // lane's token and chunk in the loads of four matrices: keys: tokens 0-7 | 8-15 | 0-7 | 8-15, chunks c, c, c + 1, c + 1;
  // values, transposed: tokens 0-7 | 0-7 | 8-15 | 8-15, chunks c, c + 1, c, c + 1
  const int k_row = (lane / 8 % 2) * 8 + lane % 8, k_chunk = lane / 16;
  const int v_row = (lane / 16) * 8 + lane % 8, v_chunk = lane / 8 % 2;
  // where the groups of 16 tokens lie in a stage
  uint32_t group_at[G];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int t = run * L::kStep + i * 16, b = t >> box_log2;
    group_at[i] = b * box_bytes * L::kBoxes + (t - (b << box_log2)) * 128;
  }
  while (true) {
    alive = alive && __all_sync(0xffffffffu, mbar_wait<0>(segment_full, segments & 1, abort_flag, a.status, kWaits + 2));
    // (one that gave up takes all with it: nobody is left at a barrier.  And the last segment's merges have been read)
    if (any_of<L::kConsumers * 32>(!alive)) {
      alive = false;
      break;
    }
    ++segments;
    const Segment g = *segment;
    if (g.s < 0) break;
    const int rows = min(L::kRows, g.n * a.group - g.tile * L::kRows);
    // A lane's columns of a product are the rows 2 q4 and 2 q4 + 1 of each eight, its rows the tokens gq and gq + 8.
    uint32_t qf[DP / 16][NT][2];
    float m[NT][2], sum[NT][2], row_scale[NT][2];
    int position[NT][2];
    float o[L::kCols / 16][NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // (8-bit chunks: elements 4 q4 + 2 e and the next instead of 2 q4 + 8 e)
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const char* at = smem + L::kQAt + (gq + 8 * t) * L::kQRow + c * 32;
        if constexpr (EIGHT) {
          const uint2 v = *reinterpret_cast<const uint2*>(at + 8 * q4);
          qf[c][t][0] = v.x;
          qf[c][t][1] = v.y;
        } else {
          qf[c][t][0] = *reinterpret_cast<const uint32_t*>(at + 4 * q4);
          qf[c][t][1] = *reinterpret_cast<const uint32_t*>(at + 4 * q4 + 16);
        }
      }
      float up = 1.f;  // of row gq
      if constexpr (EIGHT && ElemTraits<T>::kDtype == KSMM_BF16) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 v = unpack<T>(qf[c][t][e]);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e, e the largest element's exponent; subnormal rows are taken as 0, rows with infinities as they are
        const int e = static_cast<int>(__float_as_uint(top) >> 23);
        const float down = e == 0 || e >= 253 ? (e == 255 ? 1.f : e ? 0x1p-126f : 0.f) : __uint_as_float((254 - e) << 23);
        up = e == 0 || e >= 253 ? (e == 255 ? 1.f : e ? 0x1p126f : 0.f) : __uint_as_float(e << 23);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const float2 v = unpack<T>(qf[c][t][e2]);
            qf[c][t][e2] = pack<H>(v.x * down, v.y * down);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * t + 2 * q4 + e;
        position[t][e] = r < rows ? g.length - g.n + (g.tile * L::kRows + r) / a.group : INT_MAX;  // (a row that is not there masks nothing)
        m[t][e] = kNone;
        sum[t][e] = 0.f;
        row_scale[t][e] = a.scale;
        if constexpr (EIGHT && ElemTraits<T>::kDtype == KSMM_BF16) row_scale[t][e] *= __shfl_sync(0xffffffffu, up, (2 * q4 + e) * 4);
      }
    }
#pragma unroll
    for (int c = 0; c < L::kCols / 16; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][t][e] = 0.f;

    __syncwarp();
    if (lane == 0) mbar_arrive(segment_empty);
    // tokens from `clear` to below `sure` are seen by every row
    const int sure = g.first_position + 1;
    const int64_t clear = a.window ? static_cast<int64_t>(g.hi) - a.window : 0;
#pragma unroll 1
    for (int u = g.from; u < g.to; ++u) {
      const int st = turn.stage;
      alive = alive && __all_sync(0xffffffffu, mbar_wait<0>(full + 8 * st, turn.parity, abort_flag, a.status, kWaits + 2));
      const int token = u * L::kTokens + run * L::kStep;  // the warp's first
      if (alive && token < g.hi && token + L::kStep > g.lo) {
        const uint32_t ks = base + st * L::kStageBytes, vs = ks + L::kOperand;
        const int missing = flags[st];
        // ---- scores ----
        float s[G][NT][4];
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][t][e] = 0.f;
        if constexpr (!EIGHT) {
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
              uint32_t k[4];
              ldmatrix4(k, ks + group_at[i] + c / 4 * box_bytes + k_row * 128 + (((c % 4 * 2 + k_chunk) ^ (k_row & 7)) << 4));
#pragma unroll
              for (int t = 0; t < NT; ++t) mma<H>(s[i][t], k, qf[c][t][0], qf[c][t][1]);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < DP / 16; c += 2) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
              uint32_t b[4];  // tokens 0-7 and 8-15 of chunk c, then of c + 1
              ldmatrix4(b, ks + group_at[i] + c / 8 * box_bytes + k_row * 128 + (((c % 8 + k_chunk) ^ (k_row & 7)) << 4));
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t k[4] = {e4m3_to_half2(b[2 * e]), e4m3_to_half2(b[2 * e + 1]), e4m3_to_half2(b[2 * e] >> 16),
                                       e4m3_to_half2(b[2 * e + 1] >> 16)};
#pragma unroll
                for (int t = 0; t < NT; ++t) mma<H>(s[i][t], k, qf[c + e][t][0], qf[c + e][t][1]);
              }
            }
          }
        }
        float value_scale[G][2];  // of the lane's tokens
        if constexpr (EIGHT) {
          const float* sc = reinterpret_cast<const float*>(smem + L::kScalesAt + st * L::kScales) + run * L::kStep + gq;
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float key_scale = sc[16 * i + 8 * h];
              value_scale[i][h] = sc[L::kTokens + 16 * i + 8 * h];
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) s[i][t][2 * h + e] *= row_scale[t][e] * key_scale;
            }
        } else {
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[i][t][e] *= row_scale[t][e % 2];
        }
        const bool edge = token + L::kStep > sure || token < clear || token < g.lo || missing;
        uint32_t keep[2 * G];  // 16-bit pairs of tokens 2 q4, 2 q4 + 1 of each eight: whether they are the sequence's and there
        if (edge) {
#pragma unroll
          for (int i = 0; i < 2 * G; ++i) {
            const bool gone = missing >> ((run * L::kStep + i * 8) >> box_log2) & 1;
            keep[i] = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = token + 8 * i + 2 * q4 + e;
              if (j < g.hi && j >= g.lo && !gone) keep[i] |= e ? 0xffff0000u : 0xffffu;
            }
            const int j = token + 8 * i + gq;  // the lane's own of these eight
            const bool in = j < g.hi && j >= g.lo;
            if (EIGHT && (!in || gone)) value_scale[i / 2][i % 2] = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& x = s[i / 2][t][i % 2 * 2 + e];
                const bool sees = in && j <= position[t][e] && (!a.window || j > position[t][e] - a.window);
                x = sees ? (gone ? __int_as_float(0x7fffffff) : x) : -INFINITY;
              }
          }
        }
        // ---- running maximum and sum ----
        float value_size[G][2];  // log2 of the values' scales
        if constexpr (EIGHT) {
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) value_size[i][h] = fmaxf(log2_fast(fabsf(value_scale[i][h])), -80.f);
        }
        auto sized = [&](int i, int t, int e) {
          if constexpr (EIGHT) return s[i][t][e] + value_size[i][e / 2];
          else return s[i][t][e];
        };
        float scale_o[NT][2];
        bool grown = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(sized(0, t, e), sized(0, t, 2 + e));
#pragma unroll
            for (int i = 1; i < G; ++i) top = fmaxf(top, fmaxf(sized(i, t, e), sized(i, t, 2 + e)));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) - kRaise, m[t][e]);
            scale_o[t][e] = exp2_fast(m[t][e] - top);
            m[t][e] = top;
            sum[t][e] *= scale_o[t][e];
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                s[i][t][2 * h + e] = exp2_fast(s[i][t][2 * h + e] - top);
                sum[t][e] += s[i][t][2 * h + e];
              }
          }
        if constexpr (EIGHT) {
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[i][t][e] *= value_scale[i][e / 2];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) grown = grown || scale_o[t][0] != 1.f || scale_o[t][1] != 1.f;
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int c = 0; c < L::kCols / 16; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[c][t][e] *= scale_o[t][e % 2];
        }
        // ---- values ----
#pragma unroll
        for (int i = 0; i < G; ++i) {
          uint32_t hi[NT][2], part[NT][2];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x = s[i][t][2 * h], y = s[i][t][2 * h + 1];
              const uint32_t w = pack<H>(x, y);
              hi[t][h] = transpose8(w);
              if (kParts) {
                const float2 r = unpack<H>(w);
                part[t][h] = transpose8(pack<H>(x - r.x, y - r.y));
              }
            }
          const uint32_t at = vs + group_at[i] + half * (L::kBoxes / L::kHalves) * box_bytes + v_row * 128;
          if constexpr (!EIGHT) {
#pragma unroll
            for (int c = 0; c < L::kCols / 16; ++c) {
              uint32_t b[4];
              ldmatrix4_trans(b, at + c / 4 * box_bytes + (((c % 4 * 2 + v_chunk) ^ (v_row & 7)) << 4));
              if (edge) {
                b[0] &= keep[2 * i];
                b[1] &= keep[2 * i];
                b[2] &= keep[2 * i + 1];
                b[3] &= keep[2 * i + 1];
              }
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                mma<H>(o[c][t], b, hi[t][0], hi[t][1]);
                mma<H>(o[c][t], b, part[t][0], part[t][1]);
              }
            }
          } else {
            // a chunk of 16 elements: the even ones are the first eight rows of the product, the odd ones the others
#pragma unroll
            for (int c = 0; c < L::kCols / 16; c += 2) {
              uint32_t b[4];  // tokens 0-7 of chunks c and c + 1, then tokens 8-15
              ldmatrix4_trans(b, at + c / 8 * box_bytes + (((c % 8 + v_chunk) ^ (v_row & 7)) << 4));
              if (edge) {
                b[0] &= keep[2 * i];
                b[1] &= keep[2 * i];
                b[2] &= keep[2 * i + 1];
                b[3] &= keep[2 * i + 1];
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t v[4] = {e4m3_to_half2(__byte_perm(b[e], 0, 0x0020)), e4m3_to_half2(__byte_perm(b[e], 0, 0x0031)),
                                       e4m3_to_half2(__byte_perm(b[2 + e], 0, 0x0020)), e4m3_to_half2(__byte_perm(b[2 + e], 0, 0x0031))};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  mma<H>(o[c + e][t], v, hi[t][0], hi[t][1]);
                  if (kParts) mma<H>(o[c + e][t], v, part[t][0], part[t][1]);
                }
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * st);
      turn.next();
    }

    // ---- the four runs' results, in pieces of the columns that the buffer holds for all rows: every warp gives, then every
    // thread joins some pairs of neighbours and writes them ----
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2) sum[t][e] += __shfl_xor_sync(0xffffffffu, sum[t][e], x);
        if (gq == 0) {
          const int r = 8 * t + 2 * q4 + e;
          stats[run * 2 * L::kRows + r] = m[t][e];
          stats[(run * 2 + 1) * L::kRows + r] = !alive || g.bad ? __int_as_float(0x7fffffff) : sum[t][e];
        }
      }
    if (g.slot) {
      slot_used[g.slot - 1] = true;
      if (tid == 0) a.slots[2 * blockIdx.x + g.slot - 1] = g.item;
    }
    float* to_part = a.partial + (2 * static_cast<int64_t>(blockIdx.x) + g.slot - 1) * L::kRows * (p.dim + 2);
    // CAP: rows that fit, a power of two
    auto join = [&](auto cap) {
      constexpr int CAP = decltype(cap)::value, W = L::kMerge / 4 / 4 / CAP, kPieces = L::kCols / W;  // columns of a piece
      // (a store's rows, two apart, are moved by eight columns against each other: other banks)
      auto place = [&](int of_run, int r, int col) { return merge + (of_run * CAP + r) * W + (col ^ (r / 2 % 4) * 8 % W); };
#pragma unroll
      for (int piece = 0; piece < kPieces; ++piece) {
        if (piece) bar_sync_named(1, L::kConsumers * 32);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * t + 2 * q4 + e;
            if (8 * t >= CAP || r >= CAP) continue;
#pragma unroll
            for (int c = piece * (W / 16); c < (piece + 1) * (W / 16); ++c) {
              const int col = c * 16 - piece * W;
              if constexpr (EIGHT) {
                *reinterpret_cast<float2*>(place(run, r, col + 2 * gq)) = make_float2(o[c][t][e], o[c][t][2 + e]);
              } else {
                *place(run, r, col + gq) = o[c][t][e];
                *place(run, r, col + 8 + gq) = o[c][t][2 + e];
              }
            }
          }
        bar_sync_named(1, L::kConsumers * 32);
        for (int e = run * 32 + lane; e < rows * (W / 2); e += L::kRuns * 32) {
          const int r = e / (W / 2), col = e % (W / 2) * 2, d = half * L::kCols + piece * W + col;
          float top = stats[r];
#pragma unroll
          for (int k = 1; k < L::kRuns; ++k) top = fmaxf(top, stats[2 * k * L::kRows + r]);
          float total = 0.f, x = 0.f, y = 0.f;
#pragma unroll
          for (int k = 0; k < L::kRuns; ++k) {
            const float f = exp2_fast(stats[2 * k * L::kRows + r] - top);
            total = fmaf(stats[(2 * k + 1) * L::kRows + r], f, total);
            const float2 v = *reinterpret_cast<const float2*>(place(k, r, col));
            x = fmaf(v.x, f, x);
            y = fmaf(v.y, f, y);
          }
          if (d >= p.dim) continue;
          if (g.slot) {
            *reinterpret_cast<float2*>(to_part + r * p.dim + d) = make_float2(x, y);
            if (d == 0) {
              to_part[L::kRows * p.dim + r] = top;
              to_part[L::kRows * (p.dim + 1) + r] = total;
            }
          } else {
            const int row = g.tile * L::kRows + r, t = row / a.group;
            const float back = total == 0.f ? 0.f : 1.f / total;
            T* to = reinterpret_cast<T*>(a.out) + (g.start + t) * a.out_token + (g.head * a.group + row - t * a.group) * a.out_head;
            *reinterpret_cast<uint32_t*>(to + d) = pack<T>(x * back, y * back);
          }
        }
      }
    };
    if (rows <= 4) join(std::integral_constant<int, 4>());
    else if (NT == 1 || rows <= 8) join(std::integral_constant<int, 8>());
    else if constexpr (NT == 2) join(std::integral_constant<int, 16>());
  }
  if (!alive && a.split && tid < 2) slot_used[tid] = false;
  if (a.split && tid < 2 && !slot_used[tid]) a.slots[2 * blockIdx.x + tid] = -1;
}

template <typename T, bool EIGHT, int DP, int NT>
int launch_one(const Maps& maps, const Attend& a, int box, int joined, unsigned grid, cudaStream_t stream) {
  using L = Layout<EIGHT, DP, NT>;
  auto kern = token_kernel<T, EIGHT, DP, NT>;
  static std::atomic<uint64_t> ready{0};  // a bit per device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(ready.load(std::memory_order_acquire) & bit)) {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (err == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  }
  if (err == cudaSuccess) err = launch_pdl(kern, grid, L::kThreads, L::kBytes, stream, maps, a, 31 - __builtin_clz(box), joined);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "attention token kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

template <typename T, bool EIGHT, int DP, int NT>
int launch_maps(const Attend& a, int cache_dtype, unsigned grid, cudaStream_t stream) {
  using L = Layout<EIGHT, DP, NT>;
  const Pool& p = a.pool;
  int box = L::kTokens;
  while (p.page_size % box) box /= 2;
  constexpr uint64_t kColumn = EIGHT ? 128 : 64;  // elements of 128 bytes
  const bool joined = L::kBoxes > 1 && p.dim % kColumn == 0;
  Maps maps;
  for (int i = 0; i < 2; ++i) {
    const uint64_t dim = p.dim, rows = p.page_size, heads = p.kv_heads, pages = p.pages, token = p.token[i], head = p.head[i], page = p.page[i];
    const uint64_t dims4[4] = {dim, rows, heads, pages}, strides4[4] = {1, token, head, page};
    const uint64_t dims5[5] = {kColumn, rows, dim / kColumn, heads, pages}, strides5[5] = {1, token, kColumn, head, page};
    const uint32_t size[5] = {static_cast<uint32_t>(kColumn), static_cast<uint32_t>(box), joined ? L::kBoxes : 1u, 1, 1};
    const int st = encode_map(i ? &maps.values : &maps.keys, cache_dtype, joined ? 5 : 4, p.data[i], joined ? dims5 : dims4,
                              joined ? strides5 : strides4, size);
    if (st != KSMM_OK) return st;
  }
  return launch_one<T, EIGHT, DP, NT>(maps, a, box, joined, grid, stream);
}

template <typename T, bool EIGHT>
int launch_dim(const Attend& a, int cache_dtype, unsigned grid, cudaStream_t stream) {
  const int dp = padded_dim(a.pool.dim);
  if constexpr (!EIGHT) {
    if (a.tile_rows == 16) {
      if (dp == 64) return launch_maps<T, false, 64, 2>(a, cache_dtype, grid, stream);
      return launch_maps<T, false, 128, 2>(a, cache_dtype, grid, stream);
    }
  }
  if (dp == 64) return launch_maps<T, EIGHT, 64, 1>(a, cache_dtype, grid, stream);
  if (dp == 128) return launch_maps<T, EIGHT, 128, 1>(a, cache_dtype, grid, stream);
  return launch_maps<T, EIGHT, 256, 1>(a, cache_dtype, grid, stream);
}

}  // namespace

int launch_token(const Attend& a, int dtype, int cache_dtype, unsigned grid, cudaStream_t stream) {
  const bool eight = cache_dtype == KSMM_F8E4M3;
  if (dtype == KSMM_F16)
    return eight ? launch_dim<__half, true>(a, cache_dtype, grid, stream) : launch_dim<__half, false>(a, cache_dtype, grid, stream);
  return eight ? launch_dim<__nv_bfloat16, true>(a, cache_dtype, grid, stream) : launch_dim<__nv_bfloat16, false>(a, cache_dtype, grid, stream);
}

}  // namespace cache
}  // namespace ksmm
