// Attention of many new tokens (prompts) over a paged cache in 16 or 8 bits, on tcgen05.
//
// An item is one key head and a tile of up to 128 rows: a row is (token, head of the group), all heads that share the key head
// side by side, so that keys and values are read once for them.  Per tile of keys: S = Q K^T into tensor memory, a thread per row
// turns its S into weights (running maximum, exponentials, sum in fp32) and writes them back as 16-bit pairs, O += P V takes them
// from tensor memory as its A operand.  P lies over S.
//
// Four warps of rows, one that issues TMA loads, one that issues MMAs; two blocks on an SM (four for up to 64 columns), each with its
// part of the tensor memory: while the rows of one work, the tensor cores run another's products, and one's start and end (6 us,
// as much as five tiles) pass under the others' work.  32 prompts of 1000 tokens, 12 heads of 64: 186 us with one block of two row
// tiles, 181 with two blocks, 154 with four (now 151).  A prompt of 8192 tokens, 32/8 heads of 128: 507 to 515 us, 1070 TFLOP/s or more, as
// a replayed graph; call after call 585 to 595, where the power limit holds the clock down.
// What bounds it: the chain of a tile (products, scores to registers, maximum, exponentials, weights back, products), 3700 cycles for two
// blocks, of which the products are 2050.  No unit is full: heads of 64 issue in 42 % of the cycles and keep the tensor pipe busy for
// 17 %; a quarter of the exponentials as polynomials made it slower (650 us).
//
// K is K-major as it lies in the pages, V is the MN-major operand (its tokens are the contraction), so neither is turned.  O stays in
// tensor memory; it is rescaled only when a row's maximum has grown by more than 2^kLag since the last time, and the sum is exact to
// fp32 either way.  Weights are rounded once to 16 bits, a choice: the sum is that of the unrounded ones, the errors are
// independent and together as large as the result's own rounding (1.3 to 1.4 times the error of fp32 weights, against 64 bits), and a
// second part would double the second product.  fp16 numbers are subnormal below 2^-14 and end at 2^-24, where the sum would still
// count what the product lost: a key that takes nearly all of a row's weight, and has small values, leaves the result to thousands of
// weights down there.  So fp16 weights are raised by 2^kRaise, to 2^15 with the lag, and lose digits from 25 octaves below a row's
// largest on, not from 14 (the sum has the same factor).  A lag of 2 octaves and two more of range took 156 us for 32 prompts of
// 1000 tokens, 12 heads of 64, where 4 take 151 and 8 150.
#include <atomic>
#include <climits>

#include "cache.cuh"
#include "tc_epilogue.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace ksmm {
namespace cache {
namespace {

using namespace tc;

template <int DP, bool EIGHT>
struct Prompt {
  // Blocks on an SM, as tensor memory has room for their S and O; the more the better: a tile is a chain (products, loads, maximum,
  // exponentials, stores) whose parts leave each unit idle most of the time.
  static constexpr int kBlocks = DP == 64 ? (EIGHT ? 2 : 4) : DP == 128 ? 2 : 1;
  static constexpr int kKeys = DP == 128 && !EIGHT ? 128 : 64;  // tokens of a tile of keys (8 bits: the widening warps need registers)
  static constexpr int kBoxes = DP / 64;                       // 128-byte columns of a row
  static constexpr int kQ = 128 * DP * 2;
  static constexpr int kOperand = kKeys * DP * 2;              // a tile of keys or values
  // (one of each for 128 columns: the next keys are loaded while the rows work, the next values while they work again)
  static constexpr int kStages = DP == 128 || EIGHT ? 1 : 2;
  static constexpr int kRingAt = kQ;
  static constexpr int kBarsAt = kRingAt + 2 * kStages * kOperand;
  // q | k full, k empty, v full, v empty | s, p, o | a load of its own | scales
  static constexpr int kScaleSlots = EIGHT ? 4 : 0;
  static constexpr int kBars = 1 + 4 * kStages + 3 + 1 + kScaleSlots;
  static constexpr int kFlagsAt = kBarsAt + 8 * kBars;         // abort, tensor memory's address
  static constexpr int kSegmentAt = (kFlagsAt + 8 + 7) / 8 * 8;
  static constexpr int kScalesAt = (kSegmentAt + static_cast<int>(sizeof(Segment)) + 15) / 16 * 16;  // [slot][keys, values][token]
  static constexpr int kCodesAt = kScalesAt + kScaleSlots * 2 * kKeys * 4;  // two tiles' [keys, values]
  static constexpr int kCodes = EIGHT ? kKeys * DP : 0;
  static constexpr int kBytes = kCodesAt + 4 * kCodes;
  static constexpr int kConverters = !EIGHT ? 0 : DP == 256 ? 8 : 4;  // warps that widen, the producer's among them
  static constexpr int kThreads = 128 + 64 + (EIGHT ? 32 * (kConverters - 1) : 0);
  static constexpr int kOAt = kKeys;                           // columns of tensor memory: S, then O
  static constexpr int kColumns = DP == 64 ? 128 : DP == 128 ? 256 : 512;  // (an allocation is a power of two)
  static_assert(kOAt + DP <= kColumns && kBlocks * kColumns <= 512, "tensor memory");
  // log2 of how much a maximum may grow before O is rescaled, and of what fp16 weights are raised by (8 bits: up to twice as
  // much, with a part of a value's scale)
  template <typename T> static constexpr bool kHalfs = ElemTraits<T>::kDtype == KSMM_F16;
  template <typename T> static constexpr float kLag = kHalfs<T> ? 4.f : 8.f;
  template <typename T> static constexpr float kRaise = !kHalfs<T> ? 0.f : EIGHT ? 10.f : 11.f;
  static_assert(kBlocks * (kBytes + 1024) <= 228 * 1024, "the blocks of an SM fit its shared memory");
};

struct PromptMaps {
  CUtensorMap q, keys, values;
};

struct PromptArgs {
  Attend a;
  int tile_tokens;  // of a row tile: its rows are tile_tokens * group
  int box;          // tokens of a page that a TMA box covers
  uint32_t idesc_s, idesc_o;
};

// A from tensor memory: 128 rows, 16 k in 8 columns of pairs
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int N>
__device__ __forceinline__ void store_weights(uint32_t at, const uint32_t (&w)[N]) {
  if constexpr (N == 32) {
    tmem_st32(at, w);
  } else {
    static_assert(N == 16, "half of a tile of 64 keys");
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]), "r"(w[11]),
        "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
        : "memory");
  }
}

constexpr int kPromptWaits = kWaits + 4;

// e4m3 pairs as the model's type, exactly: fp16 holds them, times a power of two where `by` is not one
template <typename T, bool SCALED>
__device__ __forceinline__ uint32_t widen(uint32_t codes, uint32_t by) {
  const uint32_t h = e4m3_to_half2(codes);
  if constexpr (ElemTraits<T>::kDtype == KSMM_F16) {
    if constexpr (!SCALED) return h;
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&by));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack2(f.x, f.y, ElemTraits<T>::kDtype);
  }
}

// The widening warps of an 8-bit cache.  Each thread copies its pieces of two tiles ahead into shared memory and widens them itself
// into the operands' tiles.  What one warp does one after the other is the longest part of a tile (without it 8192 tokens of 32/8
// heads of 128 would take 800 us): loads into registers, which every arrival at a barrier waits for, 1566 us; copies 1483; addresses
// worked out once per box of a page 1196, a row's place in it once per thread 1116; half of the warps for keys, half for values 1842
// (twice the pieces in a row).  More warps leave the rows too few registers with two blocks on an SM; heads of 256, one block, have
// eight (689 -> 499 us with 8/1 heads), and heads of 64 four (282 against 297 us with two warps and three blocks, 32 prompts of 1000).
// A key's scale multiplies its scores and a value's scale its weights, in fp32 and for the rows to do: K
// and V hold the codes as they are.  With fp16, whose weights have no room for any scale, V takes the power of two that lies in
// [2^-24, 2^15] (below, a value vanishes in fp16 results) and the weights the rest, below 2 for scales that fp16 holds: a code times
// its scale's power of two is no more than the element itself, which does not pass 65504.
// A tile's scales are in one of four slots: V's tile, waited for below, is free only when the rows have left the tile before.
template <typename T, int DP>
__device__ __forceinline__ bool convert(const Pool& p, const Segment& g, char* smem, int first, int count, int box, int thread,
                                        uint32_t k_full, uint32_t alone, volatile int* abort_flag, int* status) {
  using C = Prompt<DP, true>;
  constexpr int kPer = DP / 16;  // 16 codes a piece; a row's are in one warp
  constexpr int kStep = 32 * C::kConverters / kPer, kPieces = C::kKeys / kStep;
  constexpr bool kHalf = ElemTraits<T>::kDtype == KSMM_F16;
  const int piece = thread % kPer, row = thread / kPer, lane = thread % 32;
  const bool inside = piece * 16 < p.dim;
  const int box_log2 = __ffs(box) - 1, boxes = C::kKeys >> box_log2, batch = 32 / boxes;
  const int32_t* table = p.table + g.s * p.table_stride;
  const uint32_t base = smem_u32(smem);
  float* const scales = reinterpret_cast<float*>(smem + C::kScalesAt);
  // Where a lane's box starts, for the tiles of a batch; before the pool: not there.
  int64_t ahead[2] = {-1, -1}, scales_ahead[2] = {0, 0};
  // (a row's place in its box is that of its thread's first row plus a part that all threads share)
  const int64_t in_box = row & (box - 1);
  const int64_t codes_in_box[2] = {in_box * p.token[0] + piece * 16, in_box * p.token[1] + piece * 16};
  const uint32_t codes_at = base + C::kCodesAt + row * DP + piece * 16;
  const uint32_t scale_at = base + C::kScalesAt + (piece * C::kKeys + row) * 4;
  auto get = [&](int j) {
    if (j < count) {
      if (j % batch == 0) {
        const int token = (first + j) * C::kKeys + (lane << box_log2);
        const int column = token / p.page_size;
        const int slot = token - column * p.page_size;
        const int page = token < g.hi && token + box > g.lo ? table[column] : -1;
#pragma unroll
        for (int of = 0; of < 2; ++of) {
          ahead[of] = page < 0 || page >= p.pages ? -1 : page * p.page[of] + g.head * p.head[of] + slot * p.token[of];
          scales_ahead[of] = page * p.spage[of] + g.head * p.shead[of] + slot;  // (a box's scales lie side by side: the host's check)
        }
      }
      int64_t at[2], scale = 0;
      const int token = (first + j) * C::kKeys + row;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        if (i == 0 || boxes > 1) {
          const int from = j % batch * boxes + ((row + i * kStep) >> box_log2);
          const int64_t key = __shfl_sync(0xffffffffu, scales_ahead[0], from), value = __shfl_sync(0xffffffffu, scales_ahead[1], from);
          at[0] = __shfl_sync(0xffffffffu, ahead[0], from);
          at[1] = __shfl_sync(0xffffffffu, ahead[1], from);
          scale = piece ? value : key;
        }
        const int64_t slot = (i * kStep) & (box - 1);
        const bool there = at[0] >= 0 && token + i * kStep >= g.lo && token + i * kStep < g.hi;
#pragma unroll
        for (int of = 0; of < 2; ++of)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(codes_at + (j % 2 * 2 + of) * C::kCodes + i * kStep * DP),
                       "l"(p.data[of] + (there && inside ? at[of] + codes_in_box[of] + slot * p.token[of] : 0)), "r"(there && inside ? 16 : 0)
                       : "memory");
        if (piece < 2)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(scale_at + (j % 4 * 2 * C::kKeys + i * kStep) * 4),
                       "l"(p.scales[piece] + (there ? scale + in_box + slot : 0)), "r"(there ? 4 : 0)
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int unit = piece % 4 * 2, turn = piece / 4 & 1;  // (the second box's odd half first: other banks than the first box's)
  char* const to = smem + piece / 4 * (C::kKeys * 128) + row * 128;
  char* const one = to + ((unit + turn ^ row & 7) << 4);  // (kStep is a multiple of 8)
  char* const other = to + ((unit + 1 - turn ^ row & 7) << 4);
  static_assert(kStep % 8 == 0 && (kStep & (kStep - 1)) == 0, "a thread's pieces are swizzled alike, boxes hold steps or steps boxes");
  auto put = [&](int at, int of, int j, const uint32_t (&by)[kPieces]) {
    uint4 in[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      in[i] = *reinterpret_cast<const uint4*>(smem + (codes_at - base) + (j % 2 * 2 + of) * C::kCodes + i * kStep * DP);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t codes[4] = {in[i].x, in[i].y, in[i].z, in[i].w};
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t pair = codes[e / 2] >> (e % 2 * 16);
        w[e] = of ? widen<T, true>(pair, by[i]) : widen<T, false>(pair, 0);
      }
      const uint4 lo = make_uint4(w[0], w[1], w[2], w[3]), hi = make_uint4(w[4], w[5], w[6], w[7]);
      *reinterpret_cast<uint4*>(one + at + i * kStep * 128) = turn ? hi : lo;
      *reinterpret_cast<uint4*>(other + at + i * kStep * 128) = turn ? lo : hi;
    }
    fence_proxy_async();
    __syncwarp();
  };
  get(0);
  get(1);
  bool alive = true;
  for (int j = 0; j < count; ++j) {
    const int kt = C::kRingAt, vt = kt + C::kOperand;
    const uint32_t parity = (j & 1) ^ 1;
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    uint32_t by[kPieces] = {};
    if constexpr (kHalf) {
      float rest[kPieces];
      float* const v = scales + (j % 4 * 2 + 1) * C::kKeys + row;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const float f = v[i * kStep];
        const int e = min(max((__float_as_int(f) >> 23 & 255) - 127, -24), 15);
        by[i] = (e >= -14 ? e + 15 << 10 : 1 << (e + 24)) * 0x10001u;
        rest[i] = f * __int_as_float(127 - e << 23);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if (piece == 0) v[i * kStep] = rest[i];
      __syncwarp();
    }
    if (lane == 0) mbar_arrive(alone + 8 * (1 + j % 4));
    alive = __all_sync(0xffffffffu, mbar_wait<20>(k_full + 8, parity, abort_flag, status, kPromptWaits + 1));
    if (!alive) break;
    put(kt, 0, j, by);
    if (lane == 0) mbar_arrive(k_full);
    alive = __all_sync(0xffffffffu, mbar_wait<20>(k_full + 24, parity, abort_flag, status, kPromptWaits + 1));
    if (!alive) break;
    put(vt, 1, j, by);
    if (lane == 0) mbar_arrive(k_full + 16);
    get(j + 2);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  return alive;
}

template <typename T, int DP, bool EIGHT>
__global__ void __launch_bounds__(Prompt<DP, EIGHT>::kThreads, Prompt<DP, EIGHT>::kBlocks)
    prompt_kernel(const __grid_constant__ PromptMaps maps, const __grid_constant__ PromptArgs args) {
  using C = Prompt<DP, EIGHT>;
  extern __shared__ __align__(1024) char smem[];
  const Attend& a = args.a;
  const Pool& p = a.pool;
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  constexpr int kProducer = 4, kIssuer = 5;
  volatile int* abort_flag = reinterpret_cast<int*>(smem + C::kFlagsAt);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kFlagsAt + 4);
  const uint32_t q_full = base + C::kBarsAt;
  auto k_full = [&](int i) { return q_full + 8 * (1 + i); };
  auto k_empty = [&](int i) { return q_full + 8 * (1 + C::kStages + i); };
  auto v_full = [&](int i) { return q_full + 8 * (1 + 2 * C::kStages + i); };
  auto v_empty = [&](int i) { return q_full + 8 * (1 + 3 * C::kStages + i); };
  const uint32_t s_full = q_full + 8 * (1 + 4 * C::kStages), p_full = s_full + 8, o_full = p_full + 8;
  const uint32_t alone = o_full + 8;
  auto scales_full = [&](int i) { return alone + 8 * (1 + i); };
  if (base % 1024) {  // (without static shared memory it starts there; swizzled tiles need it)
    if (tid == 0) atomicCAS(a.status, 0, kPromptWaits);
    return;
  }
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < C::kBars; ++i) {
      const uint32_t bar = q_full + 8 * i;
      const bool converted = EIGHT && ((bar >= k_full(0) && bar < k_empty(0)) || (bar >= v_full(0) && bar < v_empty(0)) || bar > alone);
      mbar_init(bar, converted ? C::kConverters : bar == p_full ? 4 : 1);
    }
    fence_mbar_init();
  }
  if (warp == kProducer && lane == 0) {
    prefetch_tensormap(&maps.q);
    if constexpr (!EIGHT) {
      prefetch_tensormap(&maps.keys);
      prefetch_tensormap(&maps.values);
    }
  }
  touch_parameters(args);
  grid_dep_wait();
  grid_dep_launch();
  clear_rest<T>(a);
  Segment* segment = reinterpret_cast<Segment*>(smem + C::kSegmentAt);
  if (warp == 0) {
    Walker walker;
    Segment next;
    next.s = -1;
    if (walker.start(a)) walker.next(a, &next);
    if (lane == 0) *segment = next;
  }
  if (warp == kIssuer) {
    tmem_alloc(smem_u32(tmem_slot), C::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Segment g = *segment;
  if (g.s < 0) {
    if (warp == kIssuer) tmem_dealloc(tmem, C::kColumns);
    return;
  }

  // tiles of keys: [first, first + count)
  const int first = g.lo / C::kKeys, token0 = g.tile * args.tile_tokens;
  const int count = max((g.hi + C::kKeys - 1) / C::kKeys - first, 0);

  if (warp < kProducer) {
    // ---------------- a thread per row ----------------
    const int r = tid;
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t s_at = tmem + lanes, o_at = s_at + C::kOAt;
    const int token = token0 + r / a.group;
    const bool live = r < args.tile_tokens * a.group && token < g.n;
    const int position = g.length - g.n + token;
    const int sure = g.first_position + 1;  // keys below are seen by all rows
    const int64_t clear = a.window ? static_cast<int64_t>(sure) - 1 + args.tile_tokens - a.window : 0;  // so are keys from here on
    const int boxes = C::kKeys / args.box;
    float top = kNone, sum = 0.f;
    bool alive = true;
    // whether lane i's box of the next tile is a page that is not there
    auto missing_box = [&](int j) {
      const int at = (first + j) * C::kKeys + lane * args.box;
      if (lane >= boxes || at >= g.hi || at + args.box <= g.lo) return false;
      const int page = p.table[g.s * p.table_stride + at / p.page_size];
      return page < 0 || page >= p.pages;
    };
    bool missing_next = count > 0 && missing_box(0);
    for (int j = 0; j < count; ++j) {
      const uint32_t missing = __ballot_sync(0xffffffffu, missing_next);
      if (j + 1 < count) missing_next = missing_box(j + 1);
      if constexpr (EIGHT)
        alive = __all_sync(0xffffffffu, mbar_wait<0>(scales_full(j % 4), j / 4 & 1, abort_flag, a.status, kPromptWaits + 4));
      alive = alive && __all_sync(0xffffffffu, mbar_wait<0>(s_full, j & 1, abort_flag, a.status, kPromptWaits + 4));
      if (!alive) break;
      tc_fence_after();
      const float* scales = reinterpret_cast<const float*>(smem + C::kScalesAt) + j % 4 * (2 * C::kKeys);
      // In halves of the columns: the second is kept while the maximum is found and turned into weights first, the first is read
      // again (registers for a whole row at once do not go round with two blocks).
      constexpr int kHalf = C::kKeys / 2;
      const int key = (first + j) * C::kKeys;
      const bool edge = key + C::kKeys > sure || key < clear || key < g.lo || missing;
      float s[kHalf];
      auto load = [&](int half) {
#pragma unroll
        for (int c = 0; c < kHalf; c += 32) tmem_ld32(s_at + half * kHalf + c, reinterpret_cast<uint32_t*>(s) + c);
        tmem_ld_wait();
        if constexpr (EIGHT) {
#pragma unroll
          for (int c = 0; c < kHalf; c += 4) {
            const float4 k = *reinterpret_cast<const float4*>(scales + half * kHalf + c);
            unpack_f2(mul_f2(pack_f2(s[c], s[c + 1]), pack_f2(k.x, k.y)), s[c], s[c + 1]);
            unpack_f2(mul_f2(pack_f2(s[c + 2], s[c + 3]), pack_f2(k.z, k.w)), s[c + 2], s[c + 3]);
          }
        }
        if (!edge) return;
        if (missing) {
#pragma unroll
          for (int c = 0; c < kHalf; c += 16)
            if (missing >> ((half * kHalf + c) / args.box) & 1) {
#pragma unroll
              for (int e = 0; e < 16; ++e) s[c + e] = __int_as_float(0x7fffffff);
            }
        }
        const int64_t oldest = a.window ? position - a.window + 1 - key : 0;
        const int to = min(position + 1, g.hi) - key - half * kHalf;
        const int from = static_cast<int>(oldest < 0 ? 0 : oldest < C::kKeys ? oldest : C::kKeys) - half * kHalf;
#pragma unroll
        for (int c = 0; c < kHalf; ++c)
          if (c >= to || c < from) s[c] = -INFINITY;
      };
      float high[4] = {top, kNone, kNone, kNone};
      auto highest = [&]() {
#pragma unroll
        for (int c = 0; c < kHalf; c += 2) high[c / 2 % 4] = fmaxf(fmaxf(high[c / 2 % 4], s[c]), s[c + 1]);  // (of three: one instruction)
      };
      load(0);
      highest();
      load(1);
      highest();
      const float now = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
      const bool grown = (now - top) * a.scale > C::template kLag<T>;
      if (j == 0) {
        top = now;
      } else if (__any_sync(0xffffffffu, grown)) {
        const float f = grown ? exp2_fast((top - now) * a.scale) : 1.f;
        if (grown) top = now;
        sum *= f;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_at + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st32(o_at + c, o);
        }
      }
      const float shift = (top == kNone ? 0.f : -top * a.scale) + C::template kRaise<T>;
      const uint64_t scale2 = pack_f2(a.scale, a.scale), shift2 = pack_f2(shift, shift);
      uint64_t sums[2] = {0, 0};  // pairs
      uint32_t w[kHalf / 2];
      auto weights = [&](int half) {
#pragma unroll
        for (int e = 0; e < kHalf / 2; ++e) {
          float x, y;
          unpack_f2(fma_f2(pack_f2(s[2 * e], s[2 * e + 1]), scale2, shift2), x, y);
          x = exp2_fast(x);
          y = exp2_fast(y);
          sums[e % 2] = add_f2(sums[e % 2], pack_f2(x, y));
          if constexpr (EIGHT) {
            const float2 v = *reinterpret_cast<const float2*>(scales + C::kKeys + half * kHalf + 2 * e);
            unpack_f2(mul_f2(pack_f2(x, y), pack_f2(v.x, v.y)), x, y);
          }
          w[e] = pack2(x, y, ElemTraits<T>::kDtype);
        }
      };
      // (P's second half lies over S's first, which is read again before it is written)
      uint32_t second[kHalf / 2];
      weights(1);
#pragma unroll
      for (int e = 0; e < kHalf / 2; ++e) second[e] = w[e];
      load(0);
      weights(0);
      store_weights<kHalf / 2>(s_at, w);
      store_weights<kHalf / 2>(s_at + kHalf / 2, second);
      {
        float x, y;
        unpack_f2(add_f2(sums[0], sums[1]), x, y);
        sum += x + y;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (count > 0 && alive)
      alive = __all_sync(0xffffffffu, mbar_wait<20>(o_full, 0, abort_flag, a.status, kPromptWaits + 4));
    tc_fence_after();
    T* to = reinterpret_cast<T*>(a.out) + static_cast<int64_t>(g.start + token) * a.out_token +
            static_cast<int64_t>(g.head * a.group + r % a.group) * a.out_head;
    if (g.bad || !alive) sum = __int_as_float(0x7fffffff);
    const float f = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
    for (int c = 0; c < DP; c += 32) {
      uint32_t o[32];
      if (count > 0 && alive) {
        tmem_ld32(o_at + c, o);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0u;
      }
      if (!live) continue;
#pragma unroll
      for (int e = 0; e < 32; e += 8) {
        if (c + e >= p.dim) break;
        uint4 v;
        v.x = pack2(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f, ElemTraits<T>::kDtype);
        v.y = pack2(__uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f, ElemTraits<T>::kDtype);
        v.z = pack2(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f, ElemTraits<T>::kDtype);
        v.w = pack2(__uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f, ElemTraits<T>::kDtype);
        *reinterpret_cast<uint4*>(to + c + e) = v;
      }
    }
    tc_fence_before();
  } else {
    if (EIGHT && warp != kIssuer) {
      // ---------------- 8-bit keys and values into the tiles' 16 bits ----------------
      if (count > 0 && warp == kProducer && lane == 0) {
        mbar_expect_tx(q_full, static_cast<uint32_t>(args.tile_tokens * a.group) * DP * 2);
#pragma unroll
        for (int b = 0; b < C::kBoxes; ++b) tma_load_3d(base + b * 128 * 128, &maps.q, q_full, b * 64, g.head * a.group, g.start + token0);
      }
      if constexpr (EIGHT) {
        const bool alive = convert<T, DP>(p, g, smem, first, count, args.box, (warp == kProducer ? 0 : warp - kIssuer) * 32 + lane, k_full(0), alone,
                                          abort_flag, a.status);
        if (!alive && count > 0 && warp == kProducer) {
          int zero = 0;
          mbar_wait<100>(q_full, 0, &zero, a.status, kPromptWaits + 2);  // (its copy ends before the block does)
        }
      }
    } else if (warp == kProducer) {
      // ---------------- TMA: a lane for each box of a tile, tables 32 boxes ahead ----------------
      const int boxes = C::kKeys / args.box;
      const uint32_t bytes = static_cast<uint32_t>(args.box) * DP * 2;
      const int32_t* table = p.table + g.s * p.table_stride;
      if (count > 0 && lane == 0) {
        mbar_expect_tx(q_full, static_cast<uint32_t>(args.tile_tokens * a.group) * DP * 2);
#pragma unroll
        for (int b = 0; b < C::kBoxes; ++b) tma_load_3d(base + b * 128 * 128, &maps.q, q_full, b * 64, g.head * a.group, g.start + token0);
      }
      int page_ahead = -2, ahead = 0;
      int loaded_k = 0, loaded_v = 0, lone = 0;
      bool alive = true;
      for (int j = 0; j < count && alive; ++j) {
        const int in_batch = j % (32 / boxes);
        if (in_batch == 0) {
          const int token = (first + j) * C::kKeys + lane * args.box;
          ahead = token / p.page_size;
          const bool there = token < g.hi && token + args.box > g.lo;
          page_ahead = there ? table[ahead] : -2;
          if (page_ahead < 0 || page_ahead >= p.pages) page_ahead = -2;
          ahead = token - ahead * p.page_size;
        }
        const int from = in_batch * boxes + lane;
        const int page = __shfl_sync(0xffffffffu, page_ahead, from & 31), row = __shfl_sync(0xffffffffu, ahead, from & 31);
        const bool get = lane < boxes && page >= 0;
        const uint32_t gets = __ballot_sync(0xffffffffu, get);
        const uint32_t load = __popc(gets);
        const int tile_token = (first + j) * C::kKeys;
        const int st = j % C::kStages;
        const uint32_t parity = (j / C::kStages & 1) ^ 1;
        alive = __all_sync(0xffffffffu, mbar_wait<20>(k_empty(st), parity, abort_flag, a.status, kPromptWaits + 1));
        if (!alive) break;
        if (lane == 0) {
          if (load) mbar_expect_tx(k_full(st), load * bytes);
          else mbar_arrive(k_full(st));
        }
        ++loaded_k;
        __syncwarp();
        const uint32_t kt = base + C::kRingAt + st * C::kOperand, vt = kt + C::kStages * C::kOperand;
        if (get) {
#pragma unroll
          for (int b = 0; b < C::kBoxes; ++b)
            tma_load_4d(kt + b * C::kKeys * 128 + lane * args.box * 128, &maps.keys, k_full(st), b * 64, row, g.head, page);
        }
        __syncwarp();
        alive = __all_sync(0xffffffffu, mbar_wait<20>(v_empty(st), parity, abort_flag, a.status, kPromptWaits + 1));
        if (!alive) break;
        // values that no row may meet are zeros, whatever lies in the page behind the sequence or in the stage from before
        const bool ragged = load < boxes || tile_token < g.lo || tile_token + C::kKeys > g.hi;
        const uint32_t bar = ragged ? alone : v_full(st);
        if (lane == 0 && load) mbar_expect_tx(bar, load * bytes);
        __syncwarp();
        if (get) {
#pragma unroll
          for (int b = 0; b < C::kBoxes; ++b)
            tma_load_4d(vt + b * C::kKeys * 128 + lane * args.box * 128, &maps.values, bar, b * 64, row, g.head, page);
        }
        __syncwarp();
        if (!ragged) {
          ++loaded_v;
          continue;
        }
        if (load) {
          alive = __all_sync(0xffffffffu, mbar_wait<20>(alone, lone & 1, abort_flag, a.status, kPromptWaits + 2));
          if (!alive) break;
          ++lone;
        }
        for (int i = lane; i < C::kKeys * C::kBoxes * 8; i += 32) {
          const int r = i / 8 % C::kKeys, token = tile_token + r;
          const bool keep = token >= g.lo && token < g.hi && (gets >> (r / args.box) & 1);
          if (!keep) *reinterpret_cast<uint4*>(smem + (vt - base) + i * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full(st));
        ++loaded_v;
      }
      if (!alive) {
        // the copies in flight end before the block does (one of its own: `alone`; waits that give up already did)
        int zero = 0;
        for (int j = loaded_k > C::kStages ? loaded_k - C::kStages : 0; j < loaded_k; ++j)
          mbar_wait<100>(k_full(j % C::kStages), j / C::kStages & 1, &zero, a.status, kPromptWaits + 2);
        for (int j = loaded_v > C::kStages ? loaded_v - C::kStages : 0; j < loaded_v; ++j)
          mbar_wait<100>(v_full(j % C::kStages), j / C::kStages & 1, &zero, a.status, kPromptWaits + 2);
        if (count > 0) mbar_wait<100>(q_full, 0, &zero, a.status, kPromptWaits + 2);
      }
    } else if (warp == kIssuer) {
      // ---------------- MMAs: the warp walks the loop, one lane issues ----------------
      constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const bool one = elect_one();
      bool alive = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        alive = alive && __all_sync(0xffffffffu, mbar_wait<0>(bar, parity, abort_flag, a.status, kPromptWaits + 3));
        return alive;
      };
      auto commit = [&](uint32_t bar) {
        if (one) umma_commit(bar);
      };
      auto scores = [&](int st) {
        if (one) {
          const uint32_t q = base >> 4 | 1u << 16, k = (base + C::kRingAt + st * C::kOperand) >> 4 | 1u << 16;
#pragma unroll
          for (int i = 0; i < DP / 16; ++i) {
            const uint64_t qd = static_cast<uint64_t>(kDescHi) << 32 | (q + i / 4 * (128 * 128 >> 4) + i % 4 * 2);
            const uint64_t kd = static_cast<uint64_t>(kDescHi) << 32 | (k + i / 4 * (C::kKeys * 128 >> 4) + i % 4 * 2);
            umma<2>(tmem, qd, kd, args.idesc_s, i != 0);
          }
        }
        commit(s_full);
      };
      auto outputs = [&](int st, bool more) {
        if (one) {
          const uint32_t v = (base + C::kRingAt + (C::kStages + st) * C::kOperand) >> 4 | static_cast<uint32_t>(C::kKeys * 128 >> 4) << 16;
#pragma unroll
          for (int i = 0; i < C::kKeys / 16; ++i) {
            const uint64_t vd = static_cast<uint64_t>(kDescHi) << 32 | (v + i * (16 * 128 >> 4));
            umma_ts(tmem + C::kOAt, tmem + i * 8, vd, args.idesc_o, more || i != 0);
          }
        }
      };
      if (count > 0 && wait(q_full, 0) && wait(k_full(0), 0)) {
        tc_fence_after();
        scores(0);
        commit(k_empty(0));
        for (int j = 0; j < count; ++j) {
          const int st = j % C::kStages, next = (j + 1) % C::kStages;
          if (!wait(v_full(st), j / C::kStages & 1) || !wait(p_full, j & 1)) break;
          tc_fence_after();
          outputs(st, j > 0);
          commit(v_empty(st));
          if (j + 1 == count) {
            commit(o_full);
          } else {
            if (!wait(k_full(next), (j + 1) / C::kStages & 1)) break;
            tc_fence_after();
            scores(next);  // (over P, which the products before have read: they run in order)
            commit(k_empty(next));
          }
        }
      }
      if (!alive) {
        // MMAs in flight end before tensor memory is given back
        int zero = 0;
        commit(alone);
        mbar_wait<100>(alone, 0, &zero, a.status, kPromptWaits + 3);
      }
    }
  }
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kColumns);
  }
}

template <typename T, int DP, bool EIGHT>
int launch_one(const PromptMaps& maps, const PromptArgs& args, unsigned grid, cudaStream_t stream) {
  using C = Prompt<DP, EIGHT>;
  auto kern = prompt_kernel<T, DP, EIGHT>;
  static std::atomic<uint64_t> ready{0};  // a bit per device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(ready.load(std::memory_order_acquire) & bit)) {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (err == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  }
  if (err == cudaSuccess) err = launch_pdl(kern, grid, C::kThreads, C::kBytes, stream, maps, args);
  if (err != cudaSuccess) return set_error(KSMM_ERR_CUDA, "attention prompt kernel: %s", cudaGetErrorString(err));
  count_launch();
  return KSMM_OK;
}

template <typename T, bool EIGHT>
int launch_dim(const PromptMaps& maps, const PromptArgs& args, unsigned grid, cudaStream_t stream) {
  if (args.a.pool.dim <= 64) return launch_one<T, 64, EIGHT>(maps, args, grid, stream);
  if (args.a.pool.dim <= 128) return launch_one<T, 128, EIGHT>(maps, args, grid, stream);
  return launch_one<T, 256, EIGHT>(maps, args, grid, stream);
}

}  // namespace

int launch_prompt(const Attend& a, int dtype, bool eight, unsigned grid, cudaStream_t stream) {
  const Pool& p = a.pool;
  PromptArgs args = {};
  args.a = a;
  args.tile_tokens = 128 / a.group;
  const int keys = p.dim > 64 && p.dim <= 128 && !eight ? Prompt<128, false>::kKeys : 64;
  args.box = keys;
  while (p.page_size % args.box) args.box /= 2;
  const uint32_t fmt = dtype == KSMM_F16 ? 0u : 1u;
  const uint32_t common = 1u << 4 | fmt << 7 | fmt << 10 | 128u >> 4 << 24;
  const uint32_t dp = p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256;
  args.idesc_s = common | static_cast<uint32_t>(keys >> 3) << 17;
  args.idesc_o = common | 1u << 16 | dp >> 3 << 17;
  PromptMaps maps = {};
  for (int i = 0; i < 2 && !eight; ++i) {
    const uint64_t dims[4] = {static_cast<uint64_t>(p.dim), static_cast<uint64_t>(p.page_size), static_cast<uint64_t>(p.kv_heads),
                              static_cast<uint64_t>(p.pages)};
    const uint64_t strides[4] = {1, static_cast<uint64_t>(p.token[i]), static_cast<uint64_t>(p.head[i]), static_cast<uint64_t>(p.page[i])};
    const uint32_t size[4] = {64, static_cast<uint32_t>(args.box), 1, 1};
    const int st = encode_map(i ? &maps.values : &maps.keys, dtype, 4, p.data[i], dims, strides, size);
    if (st != KSMM_OK) return st;
  }
  const uint64_t dims[3] = {static_cast<uint64_t>(p.dim), static_cast<uint64_t>(a.heads), static_cast<uint64_t>(p.tokens)};
  const uint64_t strides[3] = {1, static_cast<uint64_t>(a.q_head), static_cast<uint64_t>(a.q_token)};
  const uint32_t size[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(args.tile_tokens)};
  const int st = encode_map(&maps.q, dtype, 3, a.q, dims, strides, size);
  if (st != KSMM_OK) return st;
  if (eight) return dtype == KSMM_F16 ? launch_dim<__half, true>(maps, args, grid, stream) : launch_dim<__nv_bfloat16, true>(maps, args, grid, stream);
  return dtype == KSMM_F16 ? launch_dim<__half, false>(maps, args, grid, stream) : launch_dim<__nv_bfloat16, false>(maps, args, grid, stream);
}

}  // namespace cache
}  // namespace ksmm
